// What the kernels of the attention over the 4-bit cache share (kv4_attn.cu, kv4_prompt.cu).
#pragma once
#include "kv4.cuh"

namespace moe {

// Division of a number below 2^31 by a run-time constant without a divide: (umulhi(n, mul) + n) >> shift with
// shift = ceil(log2 d) and mul = floor(2^32 (2^shift - d) / d) + 1 (Granlund-Montgomery).
struct GroupDiv {
    uint32_t mul, shift, d;
};
inline GroupDiv make_group_div(uint32_t d) {
    GroupDiv g{0, 0, d};
    while ((1ull << g.shift) < d) ++g.shift;
    g.mul = (uint32_t)((((1ull << g.shift) - d) << 32) / d) + 1u;
    return g;
}

struct AttnArgs {
    Kv4View cache;
    Kv4Seqs seqs;
    const void* q;
    const void* gate;        // null: none
    void* out;
    int64_t qt, qh, gt, gh;  // element strides
    int vec_q, vec_gate;     // rows readable 16 bytes at a time
    int heads, group;        // query heads; query heads per KV head
    GroupDiv by_group, by_page;  // divisions of rows by heads that share a KV head, of positions by a page's
    float scale_log2;        // scale * log2(e)
    int window;              // 0: none
    int lo_rows, hi_rows;    // sequences with lo_rows <= rows < hi_rows (rows x query heads per KV head) are this launch's
    int run;                 // blocks of a tile that one copy brings (they lie in one page)
    int image_seqs;          // prompts: sequences the expanded tiles have room for
    unsigned* wide;          // prompts: [sequence] == call where its values are too unequal for f16 tiles
    unsigned call;
    int wide_too;            // those sequences are this launch's too
    int whole;               // one sequence: its units are dealt whole, nothing to join
    float* part;             // work area of the call
};

int kv4_reserve(moe_engine* e, size_t bytes);
// Prompts of bf16 rows on the fifth-generation tensor cores: sequences of at least kPromptRows rows x query heads per KV
// head; whether the call has such and its work area is not too large
constexpr int kPromptRows = 128;
template <int D>
bool kv4_prompt_fits(const moe_engine* e, const AttnArgs& a);
template <int D>
int launch_kv4_prompt(moe_engine* e, AttnArgs& call);  // sets wide and call

#ifdef __CUDACC__
// A sequence as a launch sees it: without rows where they are another launch's.
__device__ __forceinline__ Kv4Seq attn_seq(const AttnArgs& a, int b, unsigned int* err) {
    Kv4Seq s = kv4_seq(a.seqs, b, err);
    const long long rows = (long long)s.q_len * a.group;
    if ((rows < a.lo_rows || rows >= a.hi_rows) && !(a.wide_too && a.wide[b] == a.call)) s.q_len = 0;
    return s;
}
// First position of the window that ends at position p; a row before the first position (p < 0) sees none, and its p is not
// taken further down, where p - window would pass 32 bits.
__device__ __forceinline__ int window_from(const AttnArgs& a, int p) { return a.window > 0 ? max(max(p, 0) - a.window + 1, 0) : 0; }
// First position that a row of a sequence sees; pages that end before it may be gone and are not looked up.
__device__ __forceinline__ int first_seen(const AttnArgs& a, int len, int q_len) { return window_from(a, len - q_len); }
// Row tile `at` in the line of all sequences' row tiles (of `rows` rows): its sequence (n_seqs: none), its index there and the
// number of sequences with rows before that one.  Called by all threads of a CTA of n_threads (a multiple of 32);
// red: one word per warp and two more, in shared memory.
struct RowTile {
    int b, rt, rts, before;
};
__device__ __forceinline__ RowTile locate_row_tile(const AttnArgs& a, long long at, int rows, int n_threads, long long* red, unsigned int* err) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = n_threads >> 5;
    constexpr long long kOne = 1ll << 44;  // sequences counted above the row tiles
    long long carry = 0;
    for (int b0 = 0; b0 < a.seqs.n_seqs; b0 += n_threads) {
        long long mine = 0;
        if (b0 + tid < a.seqs.n_seqs) {
            const Kv4Seq s = attn_seq(a, b0 + tid, err);
            mine = ((long long)s.q_len * a.group + rows - 1) / rows;
        }
        const long long own = mine > 0 ? mine + kOne : 0;
        long long inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        __syncthreads();
        if (lane == 31) red[warp] = inc;
        __syncthreads();
        long long before = carry, sum = 0;
        for (int w = 0; w < nw; ++w) {
            if (w < warp) before += red[w];
            sum += red[w];
        }
        before += inc - own;
        const long long lo = before & (kOne - 1);
        if (mine > 0 && at >= lo && at < lo + mine) {
            red[nw] = (long long)(b0 + tid) << 32 | (at - lo);
            red[nw + 1] = (before >> 44) << 32 | mine;
        }
        carry += sum;
        if (at < (carry & (kOne - 1))) {
            __syncthreads();
            return RowTile{(int)(red[nw] >> 32), (int)(red[nw] & 0xFFFFFFFFll), (int)(red[nw + 1] & 0xFFFFFFFFll), (int)(red[nw + 1] >> 32)};
        }
    }
    return RowTile{a.seqs.n_seqs, 0, 0, 0};
}
__device__ __forceinline__ int over_group(int n, const GroupDiv& g) { return (int)((__umulhi((uint32_t)n, g.mul) + (uint32_t)n) >> g.shift); }
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));  // without ftz the compiler adds three instructions for results below 2^-126
    return r;
}
// sigmoid(g), as t / (1 + t) or 1 / (1 + t) with t = exp(-|g|), which never overflows; the quotient to 2 ulp.  f32 rows: t to 2 ulp,
// all of it below 2^-20; bf16 rows: t to 2 + 1.2 |g| ulp, a 2^-14th where |g| reaches 87.
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
    const float t = sizeof(T) == 4 ? expf(-fabsf(g)) : __expf(-fabsf(g));
    return __fdividef(g < 0.0f ? t : 1.0f, 1.0f + t);
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// (a & m) | c as one instruction (written out: with two constants the compiler makes two of it)
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t m, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(m), "r"(c));
    return d;
}
// four nibble pairs of a word as f16 pairs of n - 8: word bits {0-3, 16-19}, {4-7, 20-23}, {8-11, 24-27}, {12-15, 28-31}.
// 0x6400 | n is the f16 number 1024 + n, 0x6400 | n << 4 is 1024 + 16 n; both subtractions are exact.
__device__ __forceinline__ void nibbles_h2(uint32_t w, uint32_t (&o)[4]) {
    const __half2 m1032 = bits_h2(0xE408E408u), sixteenth = bits_h2(0x2C002C00u), m72 = bits_h2(0xD480D480u);  // -1032, 1 / 16, -72
    const uint32_t w8 = w >> 8;
    o[0] = h2_bits(__hadd2(bits_h2(and_or(w, 0x000F000Fu, 0x64006400u)), m1032));
    o[1] = h2_bits(__hfma2(bits_h2(and_or(w, 0x00F000F0u, 0x64006400u)), sixteenth, m72));
    o[2] = h2_bits(__hadd2(bits_h2(and_or(w8, 0x000F000Fu, 0x64006400u)), m1032));
    o[3] = h2_bits(__hfma2(bits_h2(and_or(w8, 0x00F000F0u, 0x64006400u)), sixteenth, m72));
}
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
#endif

}  // namespace moe

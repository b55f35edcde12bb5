// The paged 4-bit KV cache: page format, batch description and the device helpers its kernels share.
//
// A page holds page_size positions of one layer: per KV head page_size / 16 blocks, a block 16 positions of that head,
// 18 * head_dim bytes:
//   K nibbles   8 * D bytes   K pairs   D bytes   V nibbles   8 * D bytes   V pairs   D bytes
// Every 64 elements of a key or value share one (scale, bias) pair, both bf16, value = nibble * scale + bias: the codec
// of the 4-bit weights (moe_pack_int4_*), bit for bit but for groups of equal values, whose scale is 0 here.  A
// pair is one 32-bit word (scale low), stored [group][position].
//
// The nibbles lie in the order in which a warp feeds them to mma.m16n8k16, so that one 16-byte load per
// lane (512 contiguous bytes per warp, no bank conflicts, no shuffles) covers two 64-element groups of 8 keys, or one
// group of the values of 16 positions:
//   K: position t of the block sits in row (t % 2) * 8 + t / 2; the row's 64-byte segment of two groups is
//      [c 4][group 2][j 2] words, word = elements 16 c + 8 j .. + 7 of the group, element i in bits 4 i (head_dim 64: one
//      group, 32-byte rows);
//   V: [group][n 8][c 4][x 4] words, word = elements 8 n + 2 x (low nibbles) and + 1 (high) of positions 4 c .. 4 c + 3,
//      one byte per position, so that appending a position writes whole bytes.
// The contraction index of an MMA may be permuted freely as long as both operands agree; the queries (and the softmax
// weights) are laid out to match.
#pragma once
#include <cuda_fp16.h>
#include "stage.cuh"

namespace moe {

constexpr int kKv4Block = 16;  // positions per block

__host__ __device__ constexpr int kv4_block_bytes(int d) { return 18 * d; }

struct Kv4View {               // moe_kv4_cache_t as the kernels take it
    uint8_t* pages;
    int64_t num_pages;
    int page_size, kv_heads;
};
struct Kv4Seqs {               // moe_kv4_batch_t as the kernels take it
    const int32_t* q_start;
    const int32_t* seq_lens;
    const int32_t* page_table;
    int n_seqs, n_tokens, max_pages, max_seq_len, max_q_len;
};

int check_kv4(const moe_kv4_cache_t* c, const moe_kv4_batch_t* b);
Kv4View kv4_view(const moe_kv4_cache_t* c);
Kv4Seqs kv4_seqs(const moe_kv4_batch_t* b);

// device error codes (engine error word); mapped to messages in engine.cu
constexpr unsigned kErrKv4Page = 12u;    // page table entry outside the cache
constexpr unsigned kErrRopePos = 13u;    // position outside the rotary table
constexpr unsigned kErrKv4Batch = 14u;   // q_start / seq_lens disagree with the batch's host-side bounds

#ifdef __CUDACC__
// One sequence of the batch, its bounds checked: a sequence that breaks them is reported and worked on as if empty.
struct Kv4Seq {
    int row0, q_len, len;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Seqs& s, int b, unsigned int* err) {
    Kv4Seq r;
    r.row0 = s.q_start[b];
    r.q_len = s.q_start[b + 1] - r.row0;
    r.len = s.seq_lens[b];
    if (r.row0 < 0 || r.q_len < 0 || r.q_len > s.max_q_len || r.len < 0 || r.len > s.max_seq_len ||
        (long long)r.row0 + r.q_len > s.n_tokens) {
        atomicExch(err, kErrKv4Batch);
        r.row0 = r.q_len = r.len = 0;
    }
    return r;
}
// Block of a position; null (reported) when the page table does not lead into the cache.
__device__ __forceinline__ uint8_t* kv4_block(const Kv4View& c, const Kv4Seqs& s, int b, int h, int pos, int block_bytes, unsigned int* err) {
    const int pg = pos / c.page_size;
    const int32_t id = pg < s.max_pages ? s.page_table[(size_t)b * s.max_pages + pg] : -1;
    if (id < 0 || id >= c.num_pages) {
        atomicExch(err, kErrKv4Page);
        return nullptr;
    }
    const int blocks = c.page_size / kKv4Block;
    return c.pages + (((size_t)id * c.kv_heads + h) * blocks + (pos - pg * c.page_size) / kKv4Block) * block_bytes;
}

__device__ __forceinline__ float ld_act(const float* p) { return *p; }
__device__ __forceinline__ float ld_act(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st_act(float* p, float v) { *p = v; }
__device__ __forceinline__ void st_act(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// eight elements at p (16-byte aligned when vec) as f32
__device__ __forceinline__ void ld_act8(const float* p, bool vec, float (&v)[8]) {
    if (vec) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
}
__device__ __forceinline__ void ld_act8(const __nv_bfloat16* p, bool vec, float (&v)[8]) {
    if (vec) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void st_act8(float* p, bool vec, const float (&v)[8]) {
    if (vec) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = v[i];
    }
}
__device__ __forceinline__ void st_act8(__nv_bfloat16* p, bool vec, const float (&v)[8]) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(v[i]);
    }
}
#endif

}  // namespace moe

// Attention of many rows (prompts, chunks of prompts) over the 4-bit cache, bf16 rows, on tcgen05.
//
// With hundreds of rows per position the products dominate (4 D flops per row, head and position) and every position is
// read by many row tiles, so the positions the call sees are first expanded, once, into f16 tiles of 128 positions that
// lie in memory exactly as the MMAs want them in shared memory (K-major, 128-byte swizzle): a tile then arrives by plain
// bulk copies.  f16 keeps 11 bits down to 2^-14.  Keys of a tile are scaled by a power of two, values by one per tile or, where
// positions differ by more than 2^5 or a group of 64 lies below 2^-12 of the tile's largest, by one per position, which the
// weights carry: so only what a row sees decides how its weights are scaled (8,192 rows in a short run: 500 us, with every tile of
// the second kind 840).  A sequence with a key group below 2^-12 of its tile's largest key or a value group below 2^-12 of its position's
// largest (zeros aside) is left to the kernel of few rows, which has no such limits (6.2 ms).
//
// Attention kernel: a CTA owns 128 rows (of the query heads that share a KV head) and walks its positions.  One thread
// copies, one issues MMAs, eight warps hold a row per pair of threads (half a tile's positions, then half of O, each):
//   S = Q K^T (128 x 128, two buffers in tensor memory)  ->  w = exp2(S f - m)  ->  f16 P in shared memory  ->  O += P V
// O stays in tensor memory; it is rescaled only when a row's maximum has grown by more than 2^8 (the weights of a row
// share one reference, so the result does not depend on when).  QK of the next tile runs under the softmax of this one.
//
// A tile of heads of 256 takes some 2,800 cycles; its MMAs need 2,370 (N = 128: 84 cycles for K = 16), its exponentials 1,030.
// 8,192 rows of 16 heads over two KV heads: 560 us, 0.98 PFLOP/s; four warps with a row per thread: 752 us.
#include <math.h>

#include "kv4_attn.cuh"
#include "umma.cuh"

namespace moe {

constexpr int kPtTile = 128;                 // positions of a tile, rows of a CTA
// ints per tile: exponent of K; twice that of V, and 1 if every position has an exponent of its own; four words of "value is
// NaN" bits; the positions' exponents (f32) from the eighth on
constexpr int kPtMeta = 8 + kPtTile;
// exponents of tiles and positions, and the power of two that a row's sum of weights is held in: weights reach 2^15 2^100 where the
// values are all zero, 2^24 of them 2^139
constexpr int kPtLow = -100, kPtHigh = 114, kPtSum = -12;
constexpr float kSpan = 1.0f / 4096, kEven = 1.0f / 32;

template <int D>
struct PtCfg {
    static constexpr int G = D / 64;
    static constexpr int IMG = D * kPtTile * 2;                    // one f16 image of a tile
    static constexpr int OFF_K = IMG, OFF_V = 2 * IMG, OFF_P = 3 * IMG;
    static constexpr int P_BYTES = kPtTile * kPtTile * 2;
    static constexpr int OFF_TOP = OFF_P + P_BYTES;                // [2][2][128] f32: maxima of a row's two threads
    static constexpr int OFF_BAR = OFF_TOP + 2048;
    // never so little that two CTAs would share an SM (tensor memory holds one)
    static constexpr int SMEM = OFF_BAR + 128 > 118 * 1024 ? OFF_BAR + 128 : 118 * 1024;
    static constexpr int COL_S = D;                                // tensor memory: O, then two score buffers
    static constexpr int COLS = 512;
};

// Tiles of a sequence that its rows see: the first one's index and their number.
__device__ __forceinline__ void pt_range(const AttnArgs& a, const Kv4Seq& s, int& t0, int& n) {
    t0 = first_seen(a, s.len, s.q_len) / kPtTile;
    n = s.q_len > 0 ? (s.len + kPtTile - 1) / kPtTile - t0 : 0;
}

// two values n s + b, given n - 8 and b + 8 s, rounded to f16 once
__device__ __forceinline__ uint32_t value_pair(uint32_t n8, float s0, float b0, float s1, float b1) {
    const float2 f = __half22float2(bits_h2(n8));
    return h2_bits(__floats2half2_rn(fmaf(f.x, s0, b0), fmaf(f.y, s1, b1)));
}

// One CTA expands K or V of one tile of one head.  image: [(sequence, head, tile)][K, V][IMG bytes], the sequences that have
// rows here counted; meta alike, kPtMeta ints.
template <int D>
__global__ void __launch_bounds__(256) kv4_expand_kernel(AttnArgs a, int tiles_per_seq, uint8_t* image, int* meta, unsigned int* err) {
    using C = PtCfg<D>;
    constexpr int G = C::G;
    extern __shared__ __align__(1024) uint8_t ex_sm[];
    __shared__ uint8_t* blocks[8];
    __shared__ float mag[G * kPtTile], down[kPtTile], red[16];
    __shared__ unsigned int nan_bits[4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool is_v = blockIdx.x & 1;
    const int ti = blockIdx.x >> 1, h = blockIdx.y, b = blockIdx.z;
    const Kv4Seq s = attn_seq(a, b, err);
    int tile0, n;
    pt_range(a, s, tile0, n);
    if (ti >= n || ti >= tiles_per_seq) return;  // (a sequence without rows here has no tiles)
    int before = 0;                              // sequences with rows before this one
    for (int b0 = 0; b0 < b; b0 += 256) before += __syncthreads_count(b0 + tid < b && attn_seq(a, b0 + tid, err).q_len > 0);
    if (before >= a.image_seqs) {                // sequences that share rows: each is in bounds, together they are more than n_tokens
        if (tid == 0) atomicExch(err, kErrKv4Batch);
        return;
    }
    const int p0 = (tile0 + ti) * kPtTile;
    if (tid < 8)
        blocks[tid] = p0 + tid * 16 < s.len && p0 + tid * 16 + 16 > first_seen(a, s.len, s.q_len) ? kv4_block(a.cache, a.seqs, b, h, p0 + tid * 16, kv4_block_bytes(D), err) : nullptr;
    if (tid < 4) nan_bits[tid] = 0;
    __syncthreads();
    // the largest |value| that each group of each position holds
    for (int i = tid; i < G * kPtTile; i += 256) {
        const int t = i % kPtTile, g = i / kPtTile;
        const uint8_t* blk = blocks[t >> 4];
        float v = 0.0f;
        if (blk && p0 + t < s.len) {
            const uint32_t pw = *reinterpret_cast<const uint32_t*>(blk + (is_v ? 17 * D : 8 * D) + g * 64 + (t & 15) * 4);
            const float sc = __uint_as_float(pw << 16), bi = __uint_as_float(pw & 0xFFFF0000u);
            v = fmaxf(fabsf(bi), fabsf(fmaf(15.0f, sc, bi)));
            if (!(v < INFINITY && fabsf(sc) < INFINITY && fabsf(bi) < INFINITY)) {
                v = 0.0f;
                atomicOr(nan_bits + (t >> 5), 1u << (t & 31));
            }
        }
        mag[i] = v;
    }
    __syncthreads();
    // of a position: the largest, and the smallest that is not 0
    float top = 0.0f, least = INFINITY;
    if (tid < kPtTile) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float v = mag[g * kPtTile + tid];
            top = fmaxf(top, v);
            if (v > 0.0f) least = fminf(least, v);
        }
    }
    float mx = top, mn = least;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane == 0) {
        red[warp] = mx;
        red[8 + warp] = mn;
    }
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    mn = fminf(fminf(red[8], red[9]), fminf(red[10], red[11]));
    const bool here = tid < kPtTile && p0 + tid < s.len && blocks[(tid & (kPtTile - 1)) >> 4];
    if (is_v ? here && least < top * kSpan : tid == 0 && mn < mx * kSpan) a.wide[b] = a.call;
    const bool uneven = __syncthreads_or(is_v && here && (top < mx * kEven || least < mx * kSpan));
    // scaled into [1, 2) (from 2^115 on into up to 2^14); what is all zero lifts nothing
    auto exponent = [](float m) { return min(max((int)(__float_as_uint(m) >> 23) - 127, kPtLow), kPtHigh); };
    const int e = exponent(mx);
    if (tid < kPtTile) down[tid] = pow2f(-(uneven ? exponent(top) : e));
    __syncthreads();
    const size_t at = ((size_t)before * a.cache.kv_heads + h) * tiles_per_seq + ti;
    if (tid == 0) meta[at * kPtMeta + (is_v ? 1 : 0)] = is_v ? 2 * e + (uneven ? 1 : 0) : e;
    if (is_v && tid < 4) meta[at * kPtMeta + 2 + tid] = (int)nan_bits[tid];
    if (uneven && tid < kPtTile) reinterpret_cast<float*>(meta)[at * kPtMeta + 8 + tid] = (float)exponent(top);

    if (!is_v) {
        // a word = 8 elements of a position, f16 order 0 4 1 5 2 6 3 7 (the queries' too): one 16-byte chunk of the row
        for (int i = tid; i < kPtTile * (D / 8); i += 256) {
            const int c8 = i % (D / 8), t = i / (D / 8), g = c8 >> 3;
            const uint8_t* blk = blocks[t >> 4];
            uint32_t o[4] = {0, 0, 0, 0};
            if (blk && p0 + t < s.len) {
                constexpr int U = D >= 128 ? 2 : 1;
                const int tt = t & 15, cc = (c8 >> 1) & 3, j = c8 & 1;
                const uint32_t w = *reinterpret_cast<const uint32_t*>(blk + (g / U) * (512 * U) + ((tt & 1) * 8 + (tt >> 1)) * (32 * U) + cc * (8 * U) + (g % U) * 8 + j * 4);
                const uint32_t pw = *reinterpret_cast<const uint32_t*>(blk + 8 * D + g * 64 + tt * 4);
                const float sc = __uint_as_float(pw << 16) * down[t], mid = fmaf(8.0f, __uint_as_float(pw << 16), __uint_as_float(pw & 0xFFFF0000u)) * down[t];
                uint32_t nb[4];
                nibbles_h2(w, nb);
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = value_pair(nb[k], sc, mid, sc, mid);
            }
            *reinterpret_cast<uint4*>(ex_sm + g * (kPtTile * 128) + umma::sw128_offset(t, c8 & 7)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    } else {
        // rows are elements, 8 positions to a 16-byte chunk in the order 0 2 1 3 4 6 5 7 (the weights' too)
        for (int i = tid; i < (kPtTile / 8) * (D / 8); i += 256) {
            const int ch = i % (kPtTile / 8), n8 = i / (kPtTile / 8), g = n8 >> 3;  // chunk of positions, 8 elements
            const uint8_t* blk = blocks[ch >> 1];
            uint32_t o[8][4];
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[d][k] = 0;
            if (blk) {
                const int t = (ch & 1) * 8;
#pragma unroll
                for (int qd = 0; qd < 2; ++qd) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(blk + 9 * D + g * 512 + (n8 & 7) * 64 + ((t >> 2) + qd) * 16);
                    const uint4 p4 = *reinterpret_cast<const uint4*>(blk + 17 * D + g * 64 + (t + 4 * qd) * 4);
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w}, pw[4] = {p4.x, p4.y, p4.z, p4.w};
                    float sc[4], bi[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float s0 = __uint_as_float(pw[k] << 16), b0 = __uint_as_float(pw[k] & 0xFFFF0000u);
                        const bool in = p0 + ch * 8 + qd * 4 + k < s.len && fabsf(s0) < INFINITY && fabsf(b0) < INFINITY;  // NaN: marked above
                        const float d = down[ch * 8 + qd * 4 + k];
                        sc[k] = in ? s0 * d : 0.0f;
                        bi[k] = in ? fmaf(8.0f, s0, b0) * d : 0.0f;
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t nb[4];
                        nibbles_h2(w[x], nb);
                        o[2 * x][2 * qd] = value_pair(nb[0], sc[0], bi[0], sc[2], bi[2]);
                        o[2 * x + 1][2 * qd] = value_pair(nb[1], sc[0], bi[0], sc[2], bi[2]);
                        o[2 * x][2 * qd + 1] = value_pair(nb[2], sc[1], bi[1], sc[3], bi[3]);
                        o[2 * x + 1][2 * qd + 1] = value_pair(nb[3], sc[1], bi[1], sc[3], bi[3]);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < 8; ++d)
                *reinterpret_cast<uint4*>(ex_sm + (ch >> 3) * (D * 128) + umma::sw128_offset(n8 * 8 + d, ch & 7)) = make_uint4(o[d][0], o[d][1], o[d][2], o[d][3]);
        }
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(image + (at * 2 + (is_v ? 1 : 0)) * C::IMG);
    for (int i = tid; i < C::IMG / 16; i += 256) dst[i] = reinterpret_cast<const uint4*>(ex_sm)[i];
}

// Instruction descriptor for kind::f16 with f16 A and B (format 0), f32 D; the other fields as in umma::make_idesc_bf16.
__device__ __forceinline__ uint32_t make_idesc_f16(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const float (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]),
        "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]),
        "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
        : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// A wait ran out: reported; copies and MMAs in flight get some 10 ms to end before the CTA's memory is given back.
__device__ __noinline__ void give_up(unsigned int* err) {
    atomicExch(err, 1u);
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitCycles / 100) {}
}

template <int D>
__global__ void __launch_bounds__(320) kv4_prompt_kernel(AttnArgs a, int tiles_per_seq, const uint8_t* image, const int* meta, unsigned int* err) {
    using C = PtCfg<D>;
    extern __shared__ __align__(1024) uint8_t sm[];  // all of the CTA's shared memory: no static part moves it off its alignment
    if (smem_u32(sm) & 1023u) {
        if (threadIdx.x == 0) atomicExch(err, 2u);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t *k_full = bars, *v_full = bars + 1, *k_free = bars + 2, *pv_done = bars + 3, *s_full = bars + 4 /* 2 */, *p_ready = bars + 6, *q_ready = bars + 7;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 8);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);  // a row thread's wait ran out
    const int tid = threadIdx.x, warp = tid >> 5;

    // which rows: units are counted in row tiles, the last rows of a sequence (which see most) first
    const int h = blockIdx.x % a.cache.kv_heads;
    const RowTile where = locate_row_tile(a, blockIdx.x / a.cache.kv_heads, kPtTile, 320, reinterpret_cast<long long*>(sm + C::OFF_TOP), err);
    const int b = where.b;
    if (b >= a.seqs.n_seqs) return;
    if (where.before >= a.image_seqs) {  // as above: nothing was expanded for it
        if (tid == 0) atomicExch(err, kErrKv4Batch);
        return;
    }
    if (a.wide[b] == a.call) return;     // the kernel of few rows takes it
    const Kv4Seq s = kv4_seq(a.seqs, b, err);
    const int rt = where.rts - 1 - where.rt, rows_all = s.q_len * a.group, pos_base = s.len - s.q_len;
    int seq_t0, seq_n;
    pt_range(a, s, seq_t0, seq_n);
    const int j_first = rt * kPtTile / a.group, j_last = min((rt * kPtTile + kPtTile - 1) / a.group, s.q_len - 1);
    const int p_last = pos_base + j_last;  // may be negative: rows without a position
    const int t_begin = window_from(a, pos_base + j_first) / kPtTile;
    const int n_tiles = p_last >= 0 ? min(p_last / kPtTile + 1, seq_t0 + min(seq_n, tiles_per_seq)) - t_begin : 0;
    const size_t img0 = ((size_t)where.before * a.cache.kv_heads + h) * tiles_per_seq + (t_begin - seq_t0);

    if (tid == 0) {
        mbar_init(k_full, 1);
        mbar_init(v_full, 1);
        mbar_init(k_free, 1);
        mbar_init(pv_done, 1);
        mbar_init(s_full, 1);
        mbar_init(s_full + 1, 1);
        mbar_init(p_ready, 256);
        mbar_init(q_ready, 256);
        mbar_fence_init();
        *gave_up = 0;
    }
    if (warp == 9) umma::tmem_alloc(tmem_slot, C::COLS);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 8) {
        // ── copies ──
        if ((tid & 31) == 0) {
            auto load = [&](int i, int v) {
                uint64_t* bar = v ? v_full : k_full;
                uint8_t* dst = sm + (v ? C::OFF_V : C::OFF_K);
                const uint8_t* src = image + ((img0 + i) * 2 + v) * C::IMG;
                mbar_expect_tx(bar, C::IMG);
#pragma unroll
                for (int p = 0; p < C::IMG; p += 16384) bulk_g2s(dst + p, src + p, C::IMG < 16384 ? C::IMG : 16384, bar);
            };
            if (n_tiles > 0) {
                load(0, 0);
                load(0, 1);
            }
            if (n_tiles > 1 && (ok = mbar_wait(k_free, 0))) load(1, 0);
            for (int i = 0; i + 1 < n_tiles && ok; ++i) {
                if (i + 2 < n_tiles) {
                    if (!(ok = mbar_wait(k_free, (i + 1) & 1))) break;
                    load(i + 2, 0);
                }
                if (!(ok = mbar_wait(pv_done, i & 1))) break;
                load(i + 1, 1);
            }
            if (!ok) give_up(err);
        }
    } else if (warp == 9) {
        // ── MMAs ──
        if ((tid & 31) == 0 && n_tiles > 0) {
            const uint32_t id_qk = make_idesc_f16(128, kPtTile), id_pv = make_idesc_f16(128, D);
            auto qk = [&](int i) {
                umma::fence_after_sync();
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k >> 2) * (kPtTile * 128) + (k & 3) * 32;
                    umma::mma_bf16(tmem + C::COL_S + (i & 1) * kPtTile, umma::make_desc_sw128_kmajor(smem_u32(sm + off)),
                                   umma::make_desc_sw128_kmajor(smem_u32(sm + C::OFF_K + off)), id_qk, k > 0);
                }
                umma::commit(s_full + (i & 1));
                umma::commit(k_free);
            };
            ok = mbar_wait(q_ready, 0) && mbar_wait(k_full, 0);
            if (ok) qk(0);
            for (int i = 0; i < n_tiles && ok; ++i) {
                if (i + 1 < n_tiles) {
                    if (!(ok = mbar_wait(k_full, (i + 1) & 1))) break;
                    qk(i + 1);
                }
                if (!(ok = mbar_wait(p_ready, i & 1) && mbar_wait(v_full, i & 1))) break;
                umma::fence_after_sync();
#pragma unroll
                for (int k = 0; k < kPtTile / 16; ++k)
                    umma::mma_bf16(tmem, umma::make_desc_sw128_kmajor(smem_u32(sm + C::OFF_P + (k >> 2) * (kPtTile * 128) + (k & 3) * 32)),
                                   umma::make_desc_sw128_kmajor(smem_u32(sm + C::OFF_V + (k >> 2) * (D * 128) + (k & 3) * 32)), id_pv, (i > 0 || k > 0));
                umma::commit(pv_done);
            }
            if (!ok) give_up(err);
        }
    } else {
        // ── two threads per row: positions 64 half .. 64 half + 63 of a tile, elements half * D / 2 .. of O ──
        const int row = tid & 127, half = tid >> 7, rr = rt * kPtTile + row;
        const bool valid = rr < rows_all;
        const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);  // lanes 32 * (warp % 4) of tensor memory (bits 16-31)
        float* tops = reinterpret_cast<float*>(sm + C::OFF_TOP);         // [2 tiles][2 halves][128 rows]
        // rows whole, 16 bytes a lane: D / 8 lanes to a row, so 256 / D rows to a warp's load, and 16 rows to a warp
        constexpr int LPR = D / 8, RPL = 32 / LPR, NL = 16 / RPL;
        const int lane = tid & 31, sub = lane / LPR, lc = lane % LPR;
        auto row_of = [&](int i) { return warp * 16 + i * RPL + sub; };
        auto load_rows = [&](const uint16_t* base, int64_t ts, int64_t hs, bool vec, uint4 (&raw)[NL]) {
            base += (int64_t)s.row0 * ts + (int64_t)(h * a.group) * hs + 8 * lc;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int rw = min(rt * kPtTile + row_of(i), rows_all - 1);  // rows behind the last: a copy, not written
                const int jj = over_group(rw, a.by_group);
                const uint16_t* e = base + jj * ts + (rw - jj * a.group) * hs;
                if (vec) raw[i] = *reinterpret_cast<const uint4*>(e);
                else raw[i] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
            }
        };
        int e_k = 0, e_v = 0;  // of the tile at hand, requested a tile ahead
        if (n_tiles > 0) {
            e_k = meta[img0 * kPtMeta];
            e_v = meta[img0 * kPtMeta + 1];
        }
        {
            uint4 raw[NL];
            load_rows((const uint16_t*)a.q, a.qt, a.qh, a.vec_q, raw);
            const float mag = fabsf(a.scale_log2);
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                uint32_t mb = 0;  // the largest magnitude, as bf16 bits
#pragma unroll
                for (int k = 0; k < 4; ++k) mb = max(mb, max(w[k] & 0x7FFFu, (w[k] >> 16) & 0x7FFFu));
#pragma unroll
                for (int o = 1; o < LPR; o <<= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
                // scaled by a power of two into [2^14, 2^15); a negative scale turns the queries' sign, a scale of 0 makes them 0
                const int e = min(max((int)(mb >> 7) - 127, -110), 127);
                float up = pow2f(min(14 - e, 127));
                if (a.scale_log2 < 0.0f) up = -up;
                if (mag == 0.0f) up = 0.0f;
                const int rw = row_of(i);
                if (lc == 0) tops[rw] = (mag == 0.0f ? 1.0f : mag) * pow2f(max(e - 14, -126));
                float v[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[2 * k] = __uint_as_float(w[k] << 16) * up;
                    v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u) * up;
                }
                *reinterpret_cast<uint4*>(sm + (lc >> 3) * (kPtTile * 128) + umma::sw128_offset(rw, lc & 7)) =
                    make_uint4(h2_bits(__floats2half2_rn(v[0], v[4])), h2_bits(__floats2half2_rn(v[1], v[5])), h2_bits(__floats2half2_rn(v[2], v[6])),
                               h2_bits(__floats2half2_rn(v[3], v[7])));
            }
            umma::fence_smem_to_async();
            mbar_arrive(q_ready);
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float f_row = tops[row];
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the place is used for the tiles' maxima next
        const int j = valid ? over_group(rr, a.by_group) : 0;
        const int see_hi = valid ? pos_base + j : 0x7FFFFFFF;
        const int see_lo = valid ? window_from(a, see_hi) : 0;
        float m_ref = -INFINITY, l = 0.0f;
        for (int i = 0; i < n_tiles; ++i) {
            const int t0 = (t_begin + i) * kPtTile + 64 * half;  // this thread's positions
            const int* mt = meta + (img0 + i) * kPtMeta;
            const int ek = e_k, ev = e_v >> 1;
            const bool uneven = e_v & 1;
            const uint32_t nb[2] = {(uint32_t)mt[2 + 2 * half], (uint32_t)mt[3 + 2 * half]};
            if (i + 1 < n_tiles) {
                e_k = mt[kPtMeta];
                e_v = mt[kPtMeta + 1];
            }
            ok = mbar_wait(s_full + (i & 1), (i >> 1) & 1) && ok;
            umma::fence_after_sync();
            float v[2][32];
            const uint32_t sc = lane_base + C::COL_S + (i & 1) * kPtTile + 64 * half;
            umma::ld_32x32(sc, v[0]);
            umma::ld_32x32(sc + 32, v[1]);
            if (t0 + 63 > see_hi || t0 < see_lo) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const int t = t0 + 32 * q + k;
                        if (t > see_hi || t < see_lo) v[q][k] = -INFINITY;
                    }
            }
            // weights are exp2(S f + e - m): the tile's values are held divided by 2^e
            float f = fmaxf(f_row * pow2f(ek), 1.2e-38f), e_top = (float)ev;
            float2 e_own = make_float2(0.0f, 0.0f);  // of positions 2 lane, 2 lane + 1 of the 64
            auto e_of = [&](int k) { return __shfl_sync(0xffffffffu, (k & 1) ? e_own.y : e_own.x, k >> 1); };
            if (uneven) {  // an exponent per position
                e_own = reinterpret_cast<const float2*>(mt + 8 + 64 * half)[lane];
#pragma unroll
                for (int k = 0; k < 64; ++k) v[k >> 5][k & 31] = fmaf(v[k >> 5][k & 31], f, e_of(k));
                f = 1.0f;
                e_top = 0.0f;
            }
            float mx[4] = {v[0][0], v[0][1], v[1][0], v[1][1]};
#pragma unroll
            for (int k = 2; k < 32; k += 2) {
                mx[0] = fmaxf(mx[0], v[0][k]);
                mx[1] = fmaxf(mx[1], v[0][k + 1]);
                mx[2] = fmaxf(mx[2], v[1][k]);
                mx[3] = fmaxf(mx[3], v[1][k + 1]);
            }
            float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), f, e_top);
            tops[((i & 1) * 2 + half) * 128 + row] = top;
            if (!ok) *gave_up = 1;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float other = tops[((i & 1) * 2 + (half ^ 1)) * 128 + row];
            if (*gave_up) {
                ok = false;
                break;
            }
            top = fmaxf(top, other);  // (NaN where a row's scores all are: the weights then carry it)
            if (fabsf(top) > 65536.0f && top > -INFINITY) {  // scores whose own rounding exp2 would show: rounded first, like top
#pragma unroll
                for (int k = 0; k < 64; ++k) v[k >> 5][k & 31] = fmaf(v[k >> 5][k & 31], f, e_top);
                f = 1.0f;
                e_top = 0.0f;
            }
            // weights of 2^7 to 2^15 at the largest: the top of f16's range, so that the smallest keep most bits
            const bool grow = top > m_ref + 15.0f || (m_ref == -INFINITY && top > -INFINITY);
            float fix = 1.0f;
            if (grow) {
                fix = exp2_approx(m_ref - (top - 7.0f));  // 0 from -infinity
                m_ref = top - 7.0f;
                l *= fix;
            }
            const float off = e_top - (m_ref == -INFINITY ? 0.0f : m_ref);
            float l_uneven = 0.0f;
            if (uneven) {
#pragma unroll
                for (int k = 0; k < 64; ++k) l_uneven += exp2_approx(v[k >> 5][k & 31] + off - e_of(k) + (float)kPtSum);
            }
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            uint32_t w[32];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                float x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[k] = exp2_approx(fmaf(v[c >> 2][(c & 3) * 8 + k], f, off));
                    sum[k & 3] += x[k];
                }
                w[4 * c] = h2_bits(__floats2half2_rn(x[0], x[2]));
                w[4 * c + 1] = h2_bits(__floats2half2_rn(x[1], x[3]));
                w[4 * c + 2] = h2_bits(__floats2half2_rn(x[4], x[6]));
                w[4 * c + 3] = h2_bits(__floats2half2_rn(x[5], x[7]));
            }
            if (i > 0) {
                // the product before this one has read its weights, and O may be touched
                ok = mbar_wait(pv_done, (i - 1) & 1);
                if (__any_sync(0xffffffffu, grow)) {
                    umma::fence_after_sync();
#pragma unroll 1
                    for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
                        float o[32];
                        umma::ld_32x32(lane_base + c, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] *= fix;
                        tmem_st_32x32(lane_base + c, o);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(sm + C::OFF_P + half * (kPtTile * 128) + umma::sw128_offset(row, c)) =
                    make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
            umma::fence_smem_to_async();
            umma::fence_before_sync();
            mbar_arrive(p_ready);
            l = uneven ? l + l_uneven : fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), pow2f(kPtSum - ev), l);
            if (nb[0] | nb[1]) {  // values that are NaN: held as 0; rows that see one become NaN
                for (int t = 0; t < 64; ++t)
                    if ((nb[t >> 5] >> (t & 31) & 1u) && t0 + t <= see_hi && t0 + t >= see_lo) l = NAN;
            }
        }
        pdl_trigger();
        // the gates of the rows this warp will write, all requested before the last product is waited for
        uint4 graw[NL];
        if (a.gate) {
            load_rows((const uint16_t*)a.gate, a.gt, a.gh, a.vec_gate, graw);
        }
        if (ok && n_tiles > 0) ok = mbar_wait(pv_done, (n_tiles - 1) & 1);
        umma::fence_after_sync();
        tops[half * 128 + row] = l;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        l += tops[(half ^ 1) * 128 + row];
        const float inv = l == 0.0f ? 0.0f : pow2f(kPtSum) / l;
        // through shared memory (where K and V were: every product has been waited for), so that rows are written whole
        float* stage = reinterpret_cast<float*>(sm + C::OFF_K);
#pragma unroll 1
        for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            float o[32];
            if (n_tiles > 0) {
                umma::ld_32x32(lane_base + c, o);
            } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                *reinterpret_cast<float4*>(stage + row * D + (((c >> 2) + k) ^ (row & 7)) * 4) =
                    make_float4(o[4 * k] * inv, o[4 * k + 1] * inv, o[4 * k + 2] * inv, o[4 * k + 3] * inv);
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ok) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int rw = row_of(i), rr2 = rt * kPtTile + rw;
                if (rr2 >= rows_all) continue;
                const int jj = over_group(rr2, a.by_group);
                const float4 y0 = *reinterpret_cast<const float4*>(stage + rw * D + ((2 * lc) ^ (rw & 7)) * 4);
                const float4 y1 = *reinterpret_cast<const float4*>(stage + rw * D + ((2 * lc + 1) ^ (rw & 7)) * 4);
                float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
                if (a.gate) {
                    const uint32_t w[4] = {graw[i].x, graw[i].y, graw[i].z, graw[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        y[2 * k] *= sigmoid<__nv_bfloat16>(__uint_as_float(w[k] << 16));
                        y[2 * k + 1] *= sigmoid<__nv_bfloat16>(__uint_as_float(w[k] & 0xFFFF0000u));
                    }
                }
                st_act8((__nv_bfloat16*)a.out + ((int64_t)(s.row0 + jj) * a.heads + h * a.group + rr2 - jj * a.group) * D + 8 * lc, true, y);
            }
        }
        if (!ok && tid == 0) atomicExch(err, 1u);
    }
    umma::fence_before_sync();
    __syncthreads();
    if (warp == 9) umma::tmem_dealloc(tmem, C::COLS);
}

// ─── host side ──────────────────────────────────────────────────────────────
static int pt_tiles_per_seq(const AttnArgs& a) {
    const int64_t all = ((int64_t)a.seqs.max_seq_len + kPtTile - 1) / kPtTile;
    if (a.window <= 0) return (int)all;
    const int64_t seen = ((int64_t)a.window + a.seqs.max_q_len + kPtTile - 1) / kPtTile + 1;
    return (int)(seen < all ? seen : all);
}
static int64_t pt_max_seqs(const AttnArgs& a) {  // sequences that can have kPromptRows rows
    const int64_t n = (int64_t)a.seqs.n_tokens * a.group / kPromptRows;
    return a.seqs.n_seqs == 1 ? 1 : n < a.seqs.n_seqs ? n : a.seqs.n_seqs;
}
template <int D>
static size_t pt_image_bytes(const AttnArgs& a) {
    return (size_t)pt_max_seqs(a) * a.cache.kv_heads * pt_tiles_per_seq(a) * 2 * PtCfg<D>::IMG;
}

// Images of at most 4 GB: a call that could need more (many sequences of unknown lengths) takes the kernel that needs none.
template <int D>
bool kv4_prompt_fits(const moe_engine* e, const AttnArgs& a) {
    // (counted in tiles first, 2^17 of which are 4 GB at least: 65,535 sequences x 65,535 heads x 2^24 tiles pass 64 bits in bytes)
    return (int64_t)a.seqs.max_q_len * a.group >= kPromptRows && a.cache.kv_heads <= 65535 && a.seqs.n_seqs <= 65535 &&
           pt_max_seqs(a) * a.cache.kv_heads * pt_tiles_per_seq(a) <= 1 << 17 && pt_image_bytes<D>(a) <= (size_t)4 << 30;
}

template <int D>
int launch_kv4_prompt(moe_engine* e, AttnArgs& call) {
    using C = PtCfg<D>;
    Kv4State& st = e->kv4;
    if (!st.wide) {
        const cudaError_t rc = cudaMalloc(&st.wide, 65536 * sizeof(unsigned));
        if (rc != cudaSuccess) {
            cudaGetLastError();
            st.wide = nullptr;
            return cuda_fail(rc, "kv4_attention: work area", __FILE__, __LINE__);
        }
        st.calls = 0xFFFFFFFFu;
    }
    if (++st.calls == 0) {  // the first, or all numbers used: none is anybody's
        MOE_CUDA(cudaMemsetAsync(st.wide, 0, 65536 * sizeof(unsigned), e->stream));
        st.calls = 1;
    }
    call.wide = st.wide;
    call.call = st.calls;
    AttnArgs a = call;
    const int tiles = pt_tiles_per_seq(a);
    const size_t image = pt_image_bytes<D>(a), meta = (size_t)pt_max_seqs(a) * a.cache.kv_heads * tiles * kPtMeta * 4;
    a.lo_rows = a.seqs.n_seqs == 1 ? 1 : kPromptRows;
    a.hi_rows = 0x7FFFFFFF;
    a.image_seqs = (int)pt_max_seqs(a);
    int rc = kv4_reserve(e, image + meta);
    if (rc) return rc;
    uint8_t* img = reinterpret_cast<uint8_t*>(e->kv4.work);
    int* mt = reinterpret_cast<int*>(img + image);
    unsigned int* err = e->dec_sync + 2;
    int& set = e->kv4.occupancy[48 + D / 64];
    if (!set) {
        MOE_CUDA(cudaFuncSetAttribute(kv4_expand_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::IMG));
        MOE_CUDA(cudaFuncSetAttribute(kv4_prompt_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        set = 1;
    }
    const int64_t q_rows = (int64_t)a.seqs.max_q_len * a.group;
    int64_t units = (int64_t)a.seqs.n_tokens * a.group / kPtTile + a.seqs.n_seqs, per = (q_rows + kPtTile - 1) / kPtTile * a.seqs.n_seqs;
    units = (per < units ? per : units) * a.cache.kv_heads;
    MOE_REQUIRE(units < 0x7FFFFFFF, "kv4_attention: too many rows for one call");
    if (tiles > 0) {
        kv4_expand_kernel<D><<<dim3(2 * tiles, a.cache.kv_heads, a.seqs.n_seqs), 256, C::IMG, e->stream>>>(a, tiles, img, mt, err);
        e->launches++;
    }
    kv4_prompt_kernel<D><<<(unsigned)units, 320, C::SMEM, e->stream>>>(a, tiles, img, mt, err);
    e->launches++;
    MOE_CUDA(cudaGetLastError());
    return MOE_OK;
}

template bool kv4_prompt_fits<64>(const moe_engine*, const AttnArgs&);
template bool kv4_prompt_fits<128>(const moe_engine*, const AttnArgs&);
template bool kv4_prompt_fits<256>(const moe_engine*, const AttnArgs&);
template int launch_kv4_prompt<64>(moe_engine*, AttnArgs&);
template int launch_kv4_prompt<128>(moe_engine*, AttnArgs&);
template int launch_kv4_prompt<256>(moe_engine*, AttnArgs&);

}  // namespace moe

// Attention over the paged 4-bit KV cache (page format: kv4.cuh), for single tokens, a few tokens and prompts.
//
//   o[j, h] = sum_t softmax_t(scale q[j, h] . k_t) v_t   over the positions t that row j sees.
//
// The nibbles go to the tensor cores as they are: n - 8 is exact in f16, so with k_t = s n + b (per 64 elements, group g)
//   q . k_t = sum_g  s[t, g] (q_g . (n - 8)) + (b + 8 s)[t, g] sum(q_g)
//   o_g     = sum_t (p_t s[t, g]) (n - 8)    + sum_t p_t (b + 8 s)[t, g]
// which leaves one scale per score and group instead of one per element, and no rounding of keys or values.  Queries and
// weights are f16 operands scaled by powers of two; for f32 rows they are split into a high and a low f16 term that share
// an MMA as rows r and r + 8 (22 bits; the eight query heads of a KV head fill the tile), for bf16 rows one term is
// exact (queries) or four bits finer than the result's type (weights).  Sums and the softmax are f32.
//
// A work unit is (sequence, KV head, row tile): `rows` query rows of the heads that share a KV head against its positions,
// 64 * TB at a time.  A producer warp brings the tiles' blocks in with bulk copies (one per 16 positions, so pages may end
// anywhere), four warps compute: in the score pass each warp owns a quarter of the tile's positions and keeps a running
// maximum and sum of its own, in the value pass it owns a group of 64 elements (and, for heads of less than four groups, a
// part of the positions); the weights cross in shared memory, one barrier per tile.
// Few rows (decode, verification): the tiles of all units are dealt evenly to as many CTAs as fit the GPU, in one line, so
// sequences of any lengths balance; units that cross CTAs leave partial sums that a second kernel joins.  Many rows
// (prompts): one CTA per unit over the positions its rows see, nothing to join.
#include <math.h>

#include "kv4_attn.cuh"

namespace moe {

template <int D_, bool F32_, int MT_, int TB_, bool SPLIT_>
struct AttnCfg {
    static constexpr int D = D_, MT = MT_, TB = TB_;
    static constexpr bool F32 = F32_, SPLIT = SPLIT_;
    static constexpr int G = D / 64;               // scale groups of a head
    static constexpr int RH = F32 ? 1 : 2;         // query rows a lane holds per MMA tile
    static constexpr int ROWS = 8 * RH * MT;       // query rows of a unit
    static constexpr int NB = 4 * TB;              // blocks of a tile
    static constexpr int TILE = NB * kKv4Block;    // positions of a tile
    static constexpr int TP = 4 / G;               // warps that share a group in the value pass
    static constexpr int PB = NB / TP;             // blocks a warp takes in the value pass
    static constexpr int BLK = kv4_block_bytes(D);
    static constexpr int STAGE = NB * BLK;
    static constexpr int STAGES = MT >= 4 ? 2 : 3;
    static constexpr int KS = D / 16;              // MMA steps over a head
    static constexpr int OFF_Q = STAGES * STAGE;
    static constexpr int OFF_P = OFF_Q + KS * MT * 512;
    static constexpr int P_BYTES = NB * ROWS * 64;                  // one buffer of weights
    static constexpr int RED_BYTES = (TP - 1) * ROWS * D * 4;       // partial sums of the value pass meet in the same place
    static constexpr int P_TOTAL = 2 * P_BYTES > RED_BYTES ? 2 * P_BYTES : RED_BYTES;
    static constexpr int OFF_M = OFF_P + P_TOTAL;                   // [2][NB][ROWS] running maxima that go with the weights
    static constexpr int OFF_QS = OFF_M + 2 * NB * ROWS * 4;        // [G][ROWS] sums of the queries' groups
    static constexpr int OFF_RF = OFF_QS + G * ROWS * 4;            // [ROWS] factor that makes a score of the MMA's sum
    static constexpr int OFF_ML = OFF_RF + ROWS * 4;                // [2][4][ROWS] maxima and sums of the warps
    static constexpr int OFF_BAR = (OFF_ML + 8 * ROWS * 4 + 15) / 16 * 16;
    static constexpr int SMEM = OFF_BAR + 2 * STAGES * 8 + 64;
};

// A unit of work and the tiles of it that exist.
struct AttnUnit {
    int b, h, rt;        // sequence, KV head, row tile
    int row0, q_len, len;
    int t_lo, n_tiles;   // first position (multiple of the tile) and tiles
};

// Row tiles of a sequence and tiles of each (SPLIT: every row tile of a sequence counts the same positions).
template <class C>
__device__ __forceinline__ void attn_seq_tiles(const AttnArgs& a, const Kv4Seq& s, int& rts, int& lo, int& tiles) {
    rts = (int)(((int64_t)s.q_len * a.group + C::ROWS - 1) / C::ROWS);
    const int first = max(s.len - s.q_len, 0);
    lo = a.window > 0 ? max(first - a.window + 1, 0) / C::TILE * C::TILE : 0;
    tiles = max((s.len - lo + C::TILE - 1) / C::TILE, 1);  // a sequence without positions still has rows to write
}

// The tiles of the batch in one line, dealt to min(CTAs, tiles) CTAs: those of this CTA, and the sequence they begin in with
// the number of tiles before it.  Called by the whole CTA.
struct AttnPlan {
    long long begin, end, prefix;
    int b;
};
template <class C>
__device__ AttnPlan attn_scan(const AttnArgs& a, int nthreads, long long (&red)[8], unsigned int* err) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = nthreads >> 5;
    AttnPlan p{0, 0, 0, a.seqs.n_seqs};
    auto cost = [&](int b) -> long long {
        if (b >= a.seqs.n_seqs) return 0;
        const Kv4Seq s = kv4_seq(a.seqs, b, err);
        int rts, lo, tiles;
        attn_seq_tiles<C>(a, s, rts, lo, tiles);
        return (long long)rts * tiles * a.cache.kv_heads;
    };
    long long mine = 0;
    for (int b = tid; b < a.seqs.n_seqs; b += nthreads) mine += cost(b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();
    if (lane == 0) red[warp] = mine;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < nw; ++w) total += red[w];
    const long long parts = min((long long)gridDim.x, total);
    if (blockIdx.x >= parts) return p;
    p.begin = total * blockIdx.x / parts;
    p.end = total * (blockIdx.x + 1) / parts;
    const long long at = p.begin;
    long long carry = 0;
    for (int b0 = 0; b0 < a.seqs.n_seqs; b0 += nthreads) {
        const long long c = cost(b0 + tid);
        long long inc = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long n = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += n;
        }
        __syncthreads();
        if (lane == 31) red[warp] = inc;
        __syncthreads();
        long long before = carry, sum = 0;
        for (int w = 0; w < nw; ++w) {
            if (w < warp) before += red[w];
            sum += red[w];
        }
        const long long lo = before + inc - c, hi = before + inc;
        const bool here = at >= lo && at < hi;
        __syncthreads();
        if (here) {
            red[0] = b0 + tid;
            red[1] = lo;
        }
        __syncthreads();
        if (at < carry + sum) {
            p.b = (int)red[0];
            p.prefix = red[1];
            return p;
        }
        carry += sum;
    }
    return p;
}

// ─── small device pieces ────────────────────────────────────────────────────
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <class C, typename T>
__global__ void __launch_bounds__(160) kv4_attn_kernel(AttnArgs a, unsigned int* err) {
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ long long red[8];
    constexpr int D = C::D, G = C::G, MT = C::MT, RH = C::RH, ROWS = C::ROWS, NB = C::NB, TILE = C::TILE;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t* empty = full + C::STAGES;
    int* abort_flag = reinterpret_cast<int*>(empty + C::STAGES);
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 4);
        }
        mbar_fence_init();
        *abort_flag = 0;
    }
    pdl_trigger();

    // this CTA's tiles [w_begin, w_end) of the line of all tiles (SPLIT), or one unit
    long long w_begin = 0, w_end = 0, w_at = 0;
    AttnUnit u{};
    {
        AttnPlan p;
        if constexpr (C::SPLIT) {
            p = attn_scan<C>(a, 160, red, err);
            w_begin = p.begin;
            w_end = p.end;
            if (w_begin >= w_end) return;
            const Kv4Seq s = kv4_seq(a.seqs, p.b, err);
            int rts;
            attn_seq_tiles<C>(a, s, rts, u.t_lo, u.n_tiles);
            u.b = p.b; u.row0 = s.row0; u.q_len = s.q_len; u.len = s.len;
            const long long in = w_begin - p.prefix;
            const int unit = (int)(in / u.n_tiles);
            u.h = unit / rts;
            u.rt = unit - u.h * rts;
            w_at = p.prefix + (long long)unit * u.n_tiles;  // first tile of the unit
        } else {
            // one unit per CTA, the units of a sequence's last rows (the longest) first; units are counted in row tiles
            const int h = blockIdx.x % a.cache.kv_heads;
            long long at = blockIdx.x / a.cache.kv_heads;
            int b = 0;
            Kv4Seq s{0, 0, 0};
            int rts = 0;
            for (; b < a.seqs.n_seqs; ++b) {
                s = kv4_seq(a.seqs, b, err);
                rts = (int)(((int64_t)s.q_len * a.group + ROWS - 1) / ROWS);
                if (at < rts) break;
                at -= rts;
            }
            if (b >= a.seqs.n_seqs) return;
            u.b = b; u.h = h; u.rt = rts - 1 - (int)at;
            u.row0 = s.row0; u.q_len = s.q_len; u.len = s.len;
            const int j0 = u.rt * ROWS / a.group, j1 = min((u.rt * ROWS + ROWS - 1) / a.group, s.q_len - 1);
            const int p0 = s.len - s.q_len + j0, p1 = s.len - s.q_len + j1;
            u.t_lo = a.window > 0 ? max(p0 - a.window + 1, 0) / TILE * TILE : 0;
            u.n_tiles = max((p1 + 1 - u.t_lo + TILE - 1) / TILE, 1);
            w_begin = 0; w_end = u.n_tiles; w_at = 0;
        }
    }
    __syncthreads();

    // steps to the unit behind u
    auto next_unit = [&](AttnUnit& n, long long& at) {
        at += n.n_tiles;
        int rts, lo, tiles;
        Kv4Seq s{n.row0, n.q_len, n.len};
        attn_seq_tiles<C>(a, s, rts, lo, tiles);
        if (++n.rt < rts) return;
        n.rt = 0;
        if (++n.h < a.cache.kv_heads) return;
        n.h = 0;
        do {
            if (++n.b >= a.seqs.n_seqs) return;
            s = kv4_seq(a.seqs, n.b, err);
        } while (s.q_len == 0);
        n.row0 = s.row0; n.q_len = s.q_len; n.len = s.len;
        attn_seq_tiles<C>(a, s, rts, n.t_lo, n.n_tiles);
    };

    if (warp == 4) {
        // ── producer ──
        AttnUnit n = u;
        long long at = w_at;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (long long w = w_begin; w < w_end && ok; ++w) {
            if (w >= at + n.n_tiles) next_unit(n, at);
            const int pos = n.t_lo + (int)(w - at) * TILE + lane * kKv4Block;
            const uint8_t* src = nullptr;
            if (lane < NB && pos < n.len) src = kv4_block(a.cache, a.seqs, n.b, n.h, pos, C::BLK, err);
            ok = mbar_wait(empty + stage, phase ^ 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const unsigned have = __ballot_sync(0xffffffffu, src != nullptr);
            if (lane == 0) mbar_expect_tx(full + stage, __popc(have) * C::BLK);
            __syncwarp();
            if (src) bulk_g2s(sm + stage * C::STAGE + lane * C::BLK, src, C::BLK, full + stage);
            if (++stage == C::STAGES) {
                stage = 0;
                phase ^= 1;
            }
        }
        if (!ok && lane == 0) atomicExch(err, 1u);
        return;
    }

    // ── the four computing warps ──
    const int r = lane >> 2, c = lane & 3;
    const int g_own = warp % G, tp = warp / G;  // value pass: group, part of the positions
    const T* qp = (const T*)a.q;
    const T* gatep = (const T*)a.gate;
    T* outp = (T*)a.out;
    float* q_sum = reinterpret_cast<float*>(sm + C::OFF_QS);
    float* row_f = reinterpret_cast<float*>(sm + C::OFF_RF);
    float* m_buf = reinterpret_cast<float*>(sm + C::OFF_M);
    float* ml = reinterpret_cast<float*>(sm + C::OFF_ML);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (long long w = w_begin; w < w_end && ok;) {
        if (w >= w_at + u.n_tiles) next_unit(u, w_at);
        const long long w_stop = min(w_end, w_at + u.n_tiles);
        const int rows_all = u.q_len * a.group;
        const int pos_base = u.len - u.q_len;

        // queries of the unit as MMA operands: a warp takes a row at a time; scaled by a power of two so that the largest
        // element lies in [2^14, 2^15)
        for (int row = warp; row < ROWS; row += 4) {
            const int rr = u.rt * ROWS + row;
            const bool valid = rr < rows_all;
            const int j = valid ? rr / a.group : 0, hq = u.h * a.group + (valid ? rr % a.group : 0);
            float x[D / 32];
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {  // lane: elements (i * 32 + lane)
                x[i] = valid ? ld_act(qp + (int64_t)(u.row0 + j) * a.qt + (int64_t)hq * a.qh + i * 32 + lane) : 0.0f;
                mx = max(mx, fabsf(x[i]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            int e = (int)(__float_as_uint(mx) >> 23) - 127;  // mx in [2^e, 2^(e + 1))
            e = max(e, -110);
            const float up = pow2f(14 - e > 127 ? 127 : 14 - e);
            if (lane == 0) row_f[row] = a.scale_log2 * pow2f(max(e - 14, -126));
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const float v = x[i] * up;
                const __half hi = __float2half_rn(v);
                const __half lo = __float2half_rn(v - __half2float(hi));
                // sums over 64 elements: i even / odd halves of a group
                float sum = C::F32 ? v : __half2float(hi);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == 0) {
                    if (i & 1) q_sum[(i >> 1) * ROWS + row] += sum;
                    else q_sum[(i >> 1) * ROWS + row] = sum;
                }
                // element d of the head -> (step, register, half) of the A operand
                const int d = i * 32 + lane, g = d >> 6, cc = (d >> 4) & 3, jj = (d >> 3) & 1, k8 = d & 7;
                const int ks = g * 4 + jj * 2 + ((k8 >> 1) & 1);
                const int reg = (k8 & 1) * 2, half = k8 >> 2;  // elements (0,4): a0, (1,5): a2; (2,6), (3,7): next step
                const int mt = row / (8 * RH), rin = row % (8 * RH);
                uint8_t* dst = sm + C::OFF_Q + (ks * MT + mt) * 512 + ((rin & 7) * 4 + cc) * 16 + half * 2;
                if (C::F32) {
                    *reinterpret_cast<__half*>(dst + reg * 4) = hi;
                    *reinterpret_cast<__half*>(dst + (reg + 1) * 4) = lo;
                } else {
                    *reinterpret_cast<__half*>(dst + (reg + (rin >> 3)) * 4) = hi;
                }
            }
        }
        compute_barrier();

        float m_run[MT][RH], l_run[MT][RH], rf[MT][RH];
        int see_hi[MT][RH], see_lo[MT][RH];  // positions the row sees: see_lo <= t <= see_hi
        int all_hi = 0x7FFFFFFF, all_lo = -1;
        float o[MT][8][4], o_bias[MT][RH], m_val[MT][RH];
        int e_run = 0;                       // exponent field of the value scales' reference
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int h = 0; h < RH; ++h) {
                m_run[mt][h] = m_val[mt][h] = -INFINITY;
                l_run[mt][h] = o_bias[mt][h] = 0.0f;
                const int row = mt * 8 * RH + h * 8 + r, rr = u.rt * ROWS + row;
                rf[mt][h] = row_f[row];
                // rows behind the last are computed unmasked and not written
                see_hi[mt][h] = rr < rows_all ? pos_base + rr / a.group : 0x7FFFFFFF;
                see_lo[mt][h] = a.window > 0 && rr < rows_all ? see_hi[mt][h] - a.window + 1 : 0;
                all_hi = min(all_hi, see_hi[mt][h]);
                all_lo = max(all_lo, see_lo[mt][h]);
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.0f;
        }
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) {
            all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, s));
            all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, s));
        }

        int buf = 0;
        for (; w < w_stop; ++w, buf ^= 1) {
            const int t0 = u.t_lo + (int)(w - w_at) * TILE;
            ok = mbar_wait(full + stage, phase);
            if (!ok) *abort_flag = 1;
            const uint8_t* st = sm + stage * C::STAGE;
            // ── scores ──
#pragma unroll 1
            for (int tb = 0; tb < C::TB; ++tb) {
                const int blk = warp * C::TB + tb;
                const uint8_t* kb = st + blk * C::BLK;
                const int pos0 = t0 + blk * kKv4Block + 4 * c;  // this lane's positions pos0 .. pos0 + 3
                float s[MT][RH][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < RH; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[mt][h][i] = 0.0f;
                constexpr int U = G >= 2 ? 2 : 1;
#pragma unroll
                for (int it = 0; it < G / U; ++it) {
                    uint32_t kw[2][2 * U];  // key tile, word of (group, j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if constexpr (U == 2) {
                            const uint4 q = *reinterpret_cast<const uint4*>(kb + it * 1024 + i * 512 + lane * 16);
                            kw[i][0] = q.x; kw[i][1] = q.y; kw[i][2] = q.z; kw[i][3] = q.w;
                        } else {
                            const uint2 q = *reinterpret_cast<const uint2*>(kb + i * 256 + lane * 8);
                            kw[i][0] = q.x; kw[i][1] = q.y;
                        }
                    }
#pragma unroll
                    for (int uu = 0; uu < U; ++uu) {
                        const int g = it * U + uu;
                        float acc[MT][2][4];
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int k = 0; k < 4; ++k) acc[mt][i][k] = 0.0f;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            uint32_t nb[2][4];
                            nibbles_h2(kw[0][uu * 2 + j], nb[0]);
                            nibbles_h2(kw[1][uu * 2 + j], nb[1]);
#pragma unroll
                            for (int v = 0; v < 2; ++v)
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) {
                                    const uint4 af = *reinterpret_cast<const uint4*>(sm + C::OFF_Q + ((g * 4 + j * 2 + v) * MT + mt) * 512 + lane * 16);
                                    mma_f16(acc[mt][0], af, nb[0][2 * v], nb[0][2 * v + 1]);
                                    mma_f16(acc[mt][1], af, nb[1][2 * v], nb[1][2 * v + 1]);
                                }
                        }
                        const uint4 pr = *reinterpret_cast<const uint4*>(kb + 8 * D + g * 64 + c * 16);
                        const uint32_t pw[4] = {pr.x, pr.y, pr.z, pr.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {  // position pos0 + k: key tile k % 2, column 2 c + k / 2
                            const float sc = __uint_as_float(pw[k] << 16), bi = fmaf(8.0f, sc, __uint_as_float(pw[k] & 0xFFFF0000u));
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                                for (int h = 0; h < RH; ++h) {
                                    const float qs = q_sum[g * ROWS + mt * 8 * RH + h * 8 + r];
                                    const float d = C::F32 ? acc[mt][k & 1][k >> 1] + acc[mt][k & 1][2 + (k >> 1)] : acc[mt][k & 1][2 * h + (k >> 1)];
                                    s[mt][h][k] = fmaf(sc, d, fmaf(bi, qs, s[mt][h][k]));
                                }
                        }
                    }
                }
                const bool whole = t0 + TILE - 1 <= all_hi && t0 >= all_lo;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < RH; ++h) {
                        const int row = mt * 8 * RH + h * 8 + r;
                        float mx = -INFINITY;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float x = s[mt][h][k] * rf[mt][h];
                            if (!whole && (pos0 + k > see_hi[mt][h] || pos0 + k < see_lo[mt][h])) x = -INFINITY;
                            s[mt][h][k] = x;
                            mx = fmaxf(mx, x);
                        }
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const float m_new = fmaxf(m_run[mt][h], mx);
                        const float m_ref = m_new == -INFINITY ? 0.0f : m_new;
                        float4 p;
                        p.x = exp2_approx(s[mt][h][0] - m_ref);
                        p.y = exp2_approx(s[mt][h][1] - m_ref);
                        p.z = exp2_approx(s[mt][h][2] - m_ref);
                        p.w = exp2_approx(s[mt][h][3] - m_ref);
                        l_run[mt][h] = fmaf(l_run[mt][h], exp2_approx(m_run[mt][h] - m_ref), (p.x + p.y) + (p.z + p.w));
                        m_run[mt][h] = m_new;
                        *reinterpret_cast<float4*>(sm + C::OFF_P + buf * C::P_BYTES + (blk * ROWS + row) * 64 + c * 16) = p;
                        if (c == 0) m_buf[(buf * NB + blk) * ROWS + row] = m_new;
                    }
            }
            compute_barrier();
            if (*(volatile int*)abort_flag) ok = false;
            // ── values ──
            // the largest scale this warp meets in the tile, positions past the sequence's end left out
            const bool tail = t0 + TILE > u.len;
            uint32_t e_max = 0;
#pragma unroll
            for (int pb = 0; pb < C::PB; ++pb) {
                const int blk = tp * C::PB + pb;
                const uint4 pr = *reinterpret_cast<const uint4*>(st + blk * C::BLK + 17 * D + g_own * 64 + c * 16);
                const uint32_t pw[4] = {pr.x, pr.y, pr.z, pr.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (!tail || t0 + blk * kKv4Block + 4 * c + k < u.len) e_max = max(e_max, (pw[k] >> 7) & 0xFFu);
            }
            e_max = max(e_max, __shfl_xor_sync(0xffffffffu, e_max, 1));
            e_max = max(e_max, __shfl_xor_sync(0xffffffffu, e_max, 2));
            // a group that was stored as NaN must not reach rows that do not see it (weight 0), nor set the reference
            const bool weird = e_max == 0xFFu;
            if (weird) {
                e_max = 0;
                for (int pb = 0; pb < C::PB; ++pb) {
                    const int blk = tp * C::PB + pb;
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t pw = *reinterpret_cast<const uint32_t*>(st + blk * C::BLK + 17 * D + g_own * 64 + c * 16 + k * 4);
                        const uint32_t ex = (pw >> 7) & 0xFFu;
                        if (ex != 0xFFu && (!tail || t0 + blk * kKv4Block + 4 * c + k < u.len)) e_max = max(e_max, ex);
                    }
                }
                e_max = max(e_max, __shfl_xor_sync(0xffffffffu, e_max, 1));
                e_max = max(e_max, __shfl_xor_sync(0xffffffffu, e_max, 2));
            }
            if ((int)e_max > e_run) {
                const int e_new = max((int)e_max, 20);
                const float f = e_run == 0 ? 0.0f : pow2f(max(e_run - e_new, -126));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[mt][n][i] *= f;
                e_run = e_new;
            }
            const float s_up = pow2f(127 - max(e_run, 20) + 14);
            float f_blk[MT][RH][C::PB];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < RH; ++h) {
                    const int row = mt * 8 * RH + h * 8 + r;
                    float m_new = m_val[mt][h];
#pragma unroll
                    for (int pb = 0; pb < C::PB; ++pb) {
                        f_blk[mt][h][pb] = m_buf[(buf * NB + tp * C::PB + pb) * ROWS + row];
                        m_new = fmaxf(m_new, f_blk[mt][h][pb]);
                    }
                    const float m_ref = m_new == -INFINITY ? 0.0f : m_new;
#pragma unroll
                    for (int pb = 0; pb < C::PB; ++pb) f_blk[mt][h][pb] = exp2_approx(f_blk[mt][h][pb] - m_ref);
                    if (m_new != m_val[mt][h]) {
                        const float f = exp2_approx(m_val[mt][h] - m_ref);
                        o_bias[mt][h] *= f;
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            if (C::F32) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[mt][n][i] *= f;
                            } else {
                                o[mt][n][2 * h] *= f;
                                o[mt][n][2 * h + 1] *= f;
                            }
                        }
                        m_val[mt][h] = m_new;
                    }
                }
#pragma unroll 1
            for (int pb = 0; pb < C::PB; ++pb) {
                const int blk = tp * C::PB + pb;
                const uint8_t* vb = st + blk * C::BLK + 9 * D;
                const uint4 vw = *reinterpret_cast<const uint4*>(vb + g_own * 512 + lane * 16);
                const uint4 pr = *reinterpret_cast<const uint4*>(vb + 8 * D + g_own * 64 + c * 16);
                const uint32_t pw[4] = {pr.x, pr.y, pr.z, pr.w};
                float sc[4], bi[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = !tail || t0 + blk * kKv4Block + 4 * c + k < u.len;
                    const float s0 = in ? __uint_as_float(pw[k] << 16) : 0.0f;
                    bi[k] = in ? fmaf(8.0f, s0, __uint_as_float(pw[k] & 0xFFFF0000u)) : 0.0f;
                    sc[k] = s0 * s_up;
                }
                uint32_t nb[4][4];  // word x: {b0 of tile 2x, b0 of 2x + 1, b1 of 2x, b1 of 2x + 1}
                nibbles_h2(vw.x, nb[0]);
                nibbles_h2(vw.y, nb[1]);
                nibbles_h2(vw.z, nb[2]);
                nibbles_h2(vw.w, nb[3]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    uint32_t af[4];
#pragma unroll
                    for (int h = 0; h < RH; ++h) {
                        const int row = mt * 8 * RH + h * 8 + r;
                        float4 p = *reinterpret_cast<const float4*>(sm + C::OFF_P + buf * C::P_BYTES + (blk * ROWS + row) * 64 + c * 16);
                        float f = f_blk[mt][h][0];  // f_blk[mt][h][pb] without indexing registers by a variable
#pragma unroll
                        for (int k = 1; k < C::PB; ++k) f = pb == k ? f_blk[mt][h][k] : f;
                        p.x *= f; p.y *= f; p.z *= f; p.w *= f;
                        if (!weird) {
                            o_bias[mt][h] += fmaf(p.x, bi[0], p.y * bi[1]) + fmaf(p.z, bi[2], p.w * bi[3]);
                            p.x *= sc[0]; p.y *= sc[1]; p.z *= sc[2]; p.w *= sc[3];
                        } else {
                            o_bias[mt][h] += (p.x == 0.0f ? 0.0f : p.x * bi[0]) + (p.y == 0.0f ? 0.0f : p.y * bi[1]) +
                                             (p.z == 0.0f ? 0.0f : p.z * bi[2]) + (p.w == 0.0f ? 0.0f : p.w * bi[3]);
                            p.x = p.x == 0.0f ? 0.0f : p.x * sc[0];
                            p.y = p.y == 0.0f ? 0.0f : p.y * sc[1];
                            p.z = p.z == 0.0f ? 0.0f : p.z * sc[2];
                            p.w = p.w == 0.0f ? 0.0f : p.w * sc[3];
                        }
                        const __half2 h02 = __floats2half2_rn(p.x, p.z), h13 = __floats2half2_rn(p.y, p.w);
                        if (C::F32) {
                            const float2 b02 = __half22float2(h02), b13 = __half22float2(h13);
                            af[0] = h2_bits(h02);
                            af[2] = h2_bits(h13);
                            af[1] = h2_bits(__floats2half2_rn(p.x - b02.x, p.z - b02.y));
                            af[3] = h2_bits(__floats2half2_rn(p.y - b13.x, p.w - b13.y));
                        } else {
                            af[h] = h2_bits(h02);
                            af[2 + h] = h2_bits(h13);
                        }
                    }
                    const uint4 av = make_uint4(af[0], af[1], af[2], af[3]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        mma_f16(o[mt][2 * x], av, nb[x][0], nb[x][2]);
                        mma_f16(o[mt][2 * x + 1], av, nb[x][1], nb[x][3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + stage);
            if (++stage == C::STAGES) {
                stage = 0;
                phase ^= 1;
            }
            if (!ok) break;
        }
        if (!ok) break;

        // ── the unit's end: maxima and sums of the warps, sums of the value pass ──
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < RH; ++h) {
                const int row = mt * 8 * RH + h * 8 + r;
                float l = l_run[mt][h], ob = o_bias[mt][h];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                ob += __shfl_xor_sync(0xffffffffu, ob, 1);
                ob += __shfl_xor_sync(0xffffffffu, ob, 2);
                o_bias[mt][h] = ob;
                if (c == 0) {
                    ml[warp * ROWS + row] = m_run[mt][h];
                    ml[(4 + warp) * ROWS + row] = l;
                }
            }
        compute_barrier();
        const bool whole_unit = w_at >= w_begin && w_at + u.n_tiles <= w_end;
        const float unscale_a = pow2f(max(min(max(e_run, 20) - 127 - 14, 127), -126));
        float* slot = nullptr;
        if (C::SPLIT && !whole_unit) slot = a.part + (size_t)(2 * blockIdx.x + (w_at <= w_begin ? 0 : 1)) * ROWS * (D + 2);
        float* red_o = reinterpret_cast<float*>(sm + C::OFF_P);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < RH; ++h) {
                const int row = mt * 8 * RH + h * 8 + r;
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) m = fmaxf(m, ml[i * ROWS + row]);
                const float m_ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int i = 0; i < 4; ++i) l = fmaf(ml[(4 + i) * ROWS + row], exp2_approx(ml[i * ROWS + row] - m_ref), l);
                const float f = exp2_approx(m_val[mt][h] - m_ref);
                const float fo = f * unscale_a, fb = f * o_bias[mt][h];
                // 16 elements of the row: 64 g + 16 c + (0..7) in column 0 of the MMA tiles, + 8 in column 1
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const float x0 = C::F32 ? o[mt][n][0] + o[mt][n][2] : o[mt][n][2 * h];
                    const float x1 = C::F32 ? o[mt][n][1] + o[mt][n][3] : o[mt][n][2 * h + 1];
                    o[mt][n][C::F32 ? 0 : 2 * h] = fmaf(x0, fo, fb);
                    o[mt][n][C::F32 ? 1 : 2 * h + 1] = fmaf(x1, fo, fb);
                }
                l_run[mt][h] = l;
                m_run[mt][h] = m;
                if (C::TP > 1 && tp > 0) {
                    float* d = red_o + ((size_t)(tp - 1) * ROWS + row) * D + 64 * g_own + 16 * c;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        d[n] = o[mt][n][C::F32 ? 0 : 2 * h];
                        d[8 + n] = o[mt][n][C::F32 ? 1 : 2 * h + 1];
                    }
                }
            }
        if (C::TP > 1) compute_barrier();
        if (tp == 0) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < RH; ++h) {
                    const int row = mt * 8 * RH + h * 8 + r, rr = u.rt * ROWS + row;
                    float y[16];
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        y[n] = o[mt][n][C::F32 ? 0 : 2 * h];
                        y[8 + n] = o[mt][n][C::F32 ? 1 : 2 * h + 1];
                    }
                    if (C::TP > 1) {
#pragma unroll
                        for (int t = 0; t < C::TP - 1; ++t) {
                            const float* d = red_o + ((size_t)t * ROWS + row) * D + 64 * g_own + 16 * c;
#pragma unroll
                            for (int n = 0; n < 16; ++n) y[n] += d[n];
                        }
                    }
                    const int d0 = 64 * g_own + 16 * c;
                    if (slot) {
                        float4* dst = reinterpret_cast<float4*>(slot + (size_t)row * D + d0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                        if (g_own == 0 && c == 0) {
                            slot[(size_t)ROWS * D + row] = m_run[mt][h];
                            slot[(size_t)ROWS * (D + 1) + row] = l_run[mt][h];
                        }
                    } else if (rr < rows_all) {
                        const int j = rr / a.group, hq = u.h * a.group + rr % a.group;
                        const float inv = l_run[mt][h] == 0.0f ? 0.0f : 1.0f / l_run[mt][h];
                        T* dst = outp + ((int64_t)(u.row0 + j) * a.heads + hq) * D + d0;
                        const T* gp = gatep ? gatep + (int64_t)(u.row0 + j) * a.gt + (int64_t)hq * a.gh + d0 : nullptr;
#pragma unroll
                        for (int n = 0; n < 16; ++n) {
                            y[n] *= inv;
                            if (gp) y[n] /= 1.0f + expf(-ld_act(gp + n));
                        }
                        float y0[8], y1[8];
#pragma unroll
                        for (int n = 0; n < 8; ++n) { y0[n] = y[n]; y1[n] = y[8 + n]; }
                        st_act8(dst, true, y0);
                        st_act8(dst + 8, true, y1);
                    }
                }
        }
        compute_barrier();  // the weights' place and the row tables are free again
    }
}

// Joins the partial results of units that were split over CTAs: one CTA per row of such a unit.
template <class C, typename T>
__global__ void __launch_bounds__(256) kv4_attn_join_kernel(AttnArgs a, int splits, unsigned int* err) {
    pdl_wait();
    constexpr int D = C::D, ROWS = C::ROWS, COLS = D / 4, PARTS = 256 / COLS;
    __shared__ long long red[8];
    __shared__ float4 sums[256];
    __shared__ float ls[256];
    // grid: x = row of the tile, y = row tile, z = (sequence, KV head)
    const int row = blockIdx.x, rt = blockIdx.y, b = blockIdx.z / a.cache.kv_heads, h = blockIdx.z % a.cache.kv_heads;
    const Kv4Seq s = kv4_seq(a.seqs, b, err);
    const int rr = rt * ROWS + row;
    if (rr >= s.q_len * a.group) return;
    int rts, lo, tiles;
    attn_seq_tiles<C>(a, s, rts, lo, tiles);
    // tiles before this unit: those of the sequences before b, then of the units before this one
    const int tid = threadIdx.x;
    long long mine = 0, before = 0, total = 0;
    for (int i = tid; i < a.seqs.n_seqs; i += 256) {
        const Kv4Seq si = kv4_seq(a.seqs, i, err);
        int r2, l2, t2;
        attn_seq_tiles<C>(a, si, r2, l2, t2);
        const long long cst = (long long)r2 * t2 * a.cache.kv_heads;
        mine += cst;
        if (i < b) before += cst;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mine += __shfl_xor_sync(0xffffffffu, mine, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if ((tid & 31) == 0) red[tid >> 5] = mine;
    __syncthreads();
    for (int w = 0; w < 8; ++w) total += red[w];
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = before;
    __syncthreads();
    before = 0;
    for (int w = 0; w < 8; ++w) before += red[w];
    const long long at = before + (long long)(h * rts + rt) * tiles, n = min((long long)splits, total);
    const int i0 = (int)(((at + 1) * n - 1) / total), i1 = (int)(((at + tiles) * n - 1) / total);
    if (i0 == i1) return;  // the unit was written whole
    // slot of CTA i's part of this unit: its first unit has the even one
    auto slot_of = [&](int i) { return (size_t)(2 * i + (i > i0 || total * i / n >= at ? 0 : 1)) * ROWS * (D + 2); };
    const int col = tid % COLS, part = tid / COLS;
    float m = -INFINITY;
    for (int i = i0 + part; i <= i1; i += PARTS) m = fmaxf(m, a.part[slot_of(i) + (size_t)ROWS * D + row]);
    ls[tid] = m;
    __syncthreads();
    m = -INFINITY;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) m = fmaxf(m, ls[p * COLS]);
    __syncthreads();
    const float m_ref = m == -INFINITY ? 0.0f : m;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (int i = i0 + part; i <= i1; i += PARTS) {
        const float* sp = a.part + slot_of(i);
        const float f = exp2_approx(sp[(size_t)ROWS * D + row] - m_ref);
        const float4 v = reinterpret_cast<const float4*>(sp + (size_t)row * D)[col];
        l = fmaf(sp[(size_t)ROWS * (D + 1) + row], f, l);
        acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    }
    sums[tid] = acc;
    ls[tid] = l;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int p = 1; p < PARTS; ++p) {
        const float4 v = sums[p * COLS + col];
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
        l += ls[p * COLS + col];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int j = rr / a.group, hq = h * a.group + rr % a.group;
    float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    if (a.gate) {
        const T* gp = (const T*)a.gate + (int64_t)(s.row0 + j) * a.gt + (int64_t)hq * a.gh + 4 * col;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] /= 1.0f + expf(-ld_act(gp + i));
    }
    T* dst = (T*)a.out + ((int64_t)(s.row0 + j) * a.heads + hq) * D + 4 * col;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
}

// ─── host side ──────────────────────────────────────────────────────────────
void kv4_destroy(moe_engine* e) {
    if (e->kv4.work) cudaFree(e->kv4.work);
    e->kv4 = Kv4State{};
}

int kv4_reserve(moe_engine* e, size_t bytes) {
    if (bytes <= e->kv4.work_bytes) return MOE_OK;
    MOE_CUDA(cudaStreamSynchronize(e->stream));
    if (e->kv4.work) cudaFree(e->kv4.work);
    e->kv4.work = nullptr;
    e->kv4.work_bytes = 0;
    MOE_CUDA(cudaMalloc(&e->kv4.work, bytes));
    e->kv4.work_bytes = bytes;
    return MOE_OK;
}

template <class C, typename T>
static int run_attn(moe_engine* e, AttnArgs a, int variant, int64_t units) {
    auto* kernel = kv4_attn_kernel<C, T>;
    int& occ = e->kv4.occupancy[variant];
    if (occ == 0) {
        MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        int n = 0;
        MOE_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 160, C::SMEM));
        MOE_REQUIRE(n > 0, "kv4_attention: the kernel does not fit this device");
        occ = n;
    }
    unsigned int* err = e->dec_sync + 2;
    if constexpr (!C::SPLIT) {
        MOE_REQUIRE(units < 0x7FFFFFFF, "kv4_attention: too many rows for one call");
        MOE_CUDA(launch_kernel(false, kernel, dim3((unsigned)units), dim3(160), C::SMEM, e->stream, a, err));
        e->launches++;
        return MOE_OK;
    } else {
        // no more CTAs than tiles there can be
        const int64_t row_tiles = ((int64_t)a.seqs.max_q_len * a.group + C::ROWS - 1) / C::ROWS;
        const int64_t most = units * ((a.seqs.max_seq_len + C::TILE - 1) / C::TILE + 1);
        int64_t grid = (int64_t)e->sm_count * occ;
        if (grid > most) grid = most;
        int rc = kv4_reserve(e, (size_t)grid * 2 * C::ROWS * (C::D + 2) * 4);
        if (rc) return rc;
        a.part = e->kv4.work;
        MOE_REQUIRE((int64_t)a.seqs.n_seqs * a.cache.kv_heads <= 65535 && row_tiles <= 65535, "kv4_attention: too many sequences for one call");
        MOE_CUDA(launch_kernel(false, kernel, dim3((unsigned)grid), dim3(160), C::SMEM, e->stream, a, err));
        MOE_CUDA(launch_kernel(true, kv4_attn_join_kernel<C, T>, dim3(C::ROWS, (unsigned)row_tiles, (unsigned)(a.seqs.n_seqs * a.cache.kv_heads)),
                               dim3(256), 0, e->stream, a, (int)grid, err));
        e->launches += 2;
        return MOE_OK;
    }
}

// Rows of the tile: as few MMA tiles as hold a sequence's rows, up to four.  Units of their own (no splitting) once they
// fill the GPU twice over.
template <int D, typename T>
static int launch_attn(moe_engine* e, const AttnArgs& a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int R1 = F32 ? 8 : 16, V0 = (D == 64 ? 0 : D == 128 ? 8 : 16) + (F32 ? 4 : 0);
    const int64_t q_rows = (int64_t)a.seqs.max_q_len * a.group, n = a.seqs.n_seqs;
    auto units = [&](int rows) {  // at most: whole tiles of all rows, and one that is not full for every sequence
        const int64_t per_seq = (q_rows + rows - 1) / rows;
        const int64_t all = (int64_t)a.seqs.n_tokens * a.group / rows + n;
        return (all < per_seq * n ? all : per_seq * n) * a.cache.kv_heads;
    };
    constexpr int TB = 4 / (D / 64);
    if constexpr (!F32) {
        if (kv4_prompt_fits<D>(e, a)) return launch_kv4_prompt<D>(e, a);
    }
    if (q_rows > 2 * R1 && units(4 * R1) >= 2 * e->sm_count) return run_attn<AttnCfg<D, F32, 4, 1, false>, T>(e, a, V0 + 3, units(4 * R1));
    if (q_rows > 2 * R1) return run_attn<AttnCfg<D, F32, 4, 1, true>, T>(e, a, V0 + 2, units(4 * R1));
    if (q_rows > R1) return run_attn<AttnCfg<D, F32, 2, 1, true>, T>(e, a, V0 + 1, units(2 * R1));
    return run_attn<AttnCfg<D, F32, 1, TB, true>, T>(e, a, V0, units(R1));
}

int check_kv4(const moe_kv4_cache_t* c, const moe_kv4_batch_t* b);
Kv4View kv4_view(const moe_kv4_cache_t* c);
Kv4Seqs kv4_seqs(const moe_kv4_batch_t* b);

}  // namespace moe

using namespace moe;

extern "C" int moe_kv4_attention_dev(moe_engine_t* e, const moe_kv4_cache_t* cache, const moe_kv4_batch_t* batch, const void* q_dev,
                                     int64_t q_token_stride, int64_t q_head_stride, const void* gate_dev, int64_t gate_token_stride,
                                     int64_t gate_head_stride, void* out_dev, int32_t dtype, int32_t num_heads, float scale, int32_t window) {
    MOE_REQUIRE(e, "kv4_attention: null engine");
    int rc = check_kv4(cache, batch);
    if (rc) return rc;
    MOE_REQUIRE(dtype == MOE_DT_F32 || dtype == MOE_DT_BF16, "kv4_attention: queries are f32 or bf16 (got dtype %d)", dtype);
    MOE_REQUIRE(num_heads > 0 && num_heads % cache->num_kv_heads == 0, "kv4_attention: num_heads (%d) must be a positive multiple of num_kv_heads (%d)",
                num_heads, cache->num_kv_heads);
    MOE_REQUIRE(window >= 0, "kv4_attention: negative window");
    MOE_REQUIRE(isfinite(scale), "kv4_attention: the scale is not finite");
    MOE_REQUIRE((int64_t)batch->max_q_len * (num_heads / cache->num_kv_heads) < (1 << 30), "kv4_attention: too many rows in one sequence");
    if (batch->n_seqs == 0 || batch->n_tokens == 0 || batch->max_q_len == 0) return MOE_OK;
    MOE_REQUIRE(q_dev && out_dev, "kv4_attention: null argument");
    const uintptr_t amask = dtype == MOE_DT_F32 ? 3 : 1;
    MOE_REQUIRE((((uintptr_t)q_dev | (uintptr_t)gate_dev) & amask) == 0, "kv4_attention: misaligned pointer");
    MOE_REQUIRE(((uintptr_t)out_dev & 15) == 0, "kv4_attention: the output must be 16-byte aligned");
    MOE_REQUIRE(q_token_stride >= 0 && q_head_stride >= 0 && gate_token_stride >= 0 && gate_head_stride >= 0, "kv4_attention: negative stride");
    DeviceScope scope(e->device);
    MOE_CUDA(scope.status);
    AttnArgs a{};
    a.cache = kv4_view(cache);
    a.seqs = kv4_seqs(batch);
    a.q = q_dev; a.gate = gate_dev; a.out = out_dev;
    a.qt = q_token_stride; a.qh = q_head_stride; a.gt = gate_token_stride; a.gh = gate_head_stride;
    a.heads = num_heads;
    a.group = num_heads / cache->num_kv_heads;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.window = window;
    const bool f32 = dtype == MOE_DT_F32;
    switch (cache->head_dim) {
        case 64: return f32 ? launch_attn<64, float>(e, a) : launch_attn<64, __nv_bfloat16>(e, a);
        case 128: return f32 ? launch_attn<128, float>(e, a) : launch_attn<128, __nv_bfloat16>(e, a);
        default: return f32 ? launch_attn<256, float>(e, a) : launch_attn<256, __nv_bfloat16>(e, a);
    }
}

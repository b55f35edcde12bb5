// Attention over the paged 4-bit KV cache (page format: kv4.cuh), for single tokens, a few tokens and prompts.
//
//   o[j, h] = sum_t softmax_t(scale q[j, h] . k_t) v_t   over the positions t that row j sees.
//
// The nibbles go to the tensor cores as they are: as a bit pattern, n is the f16 subnormal n 2^-24, exactly.  With
// k_t = s n + b (per 64 elements, group g)
//   q . k_t = sum_g  s[t, g] (q_g . n) + b[t, g] sum(q_g)
//   o_g     = sum_t (w_t s[t, g]) n    + sum_t w_t b[t, g]
// (every other pair of values as b + 15 s - s (15 - n)), which leaves one scale per score and group instead of one per element,
// and no rounding of keys or values.  Keys and values are the A operand of mma.m16n8k16 (16 positions, 16 elements), eight
// query rows the columns: the eight query heads of a KV head fill it.  Queries and weights are f16 operands scaled by powers
// of two; for f32 rows they are split into a high and a low f16 term (22 bits) that two MMAs add into the same sums, for bf16
// rows one term is exact (queries) or three bits finer than the result's type (weights).  Sums and the softmax are f32.
//
// Weights are w = exp2(x - ref), one reference per row: it moves only when a score passes it, then to 2^8 above (so the largest
// weight, which counts most, is a power of two and loses nothing as an operand).  As operands the products w s are scaled by a power of two, one per row and group, that moves only when a
// product would leave f16's range: a group's bits depend on the products that the row sees in that group, not on other groups
// or on positions hidden from it.
//
// A work unit is (sequence, KV head, row tile): `rows` query rows of the heads that share a KV head against its positions,
// 64 * TB at a time.  The tiles' blocks come in by bulk copies (as many blocks at once as lie in one page, so pages may end
// anywhere).  Four warps: in the score pass each owns a quarter of the tile's positions, in the value pass a group of 64
// elements (and, for heads of less than four groups, a part of the positions); the weights cross in shared memory, one barrier
// per tile.
// Few rows (decode, verification): the tiles of all units are dealt evenly to as many CTAs as fit the GPU, in one line, so
// sequences of any lengths balance; units that cross CTAs leave partial sums that a second kernel joins.  Many rows
// (f32 prompts; bf16 ones have kv4_prompt.cu): one CTA per unit over the positions its rows see, nothing to join.
//
// Bound by issue slots and dependent instructions: about 860 instructions per 16 positions and head of 256, 54 % of the slots
// used at four CTAs per SM (barrier and MMA latency take the rest); 250,001 positions of two heads, f32, eight query heads each:
// 57.4 us, 2.5 TB/s (55.6 with one power of two per tile, for all groups and rows).
#include <math.h>

#include <type_traits>

#include "kv4_attn.cuh"
#include "umma.cuh"

namespace moe {

template <int D_, bool F32_, int NT_, int TB_, bool SPLIT_>
struct AttnCfg {
    static constexpr int D = D_, NT = NT_, TB = TB_;
    static constexpr bool F32 = F32_, SPLIT = SPLIT_;
    static constexpr int G = D / 64;               // scale groups of a head
    static constexpr int ROWS = 8 * NT;            // query rows of a unit
    static constexpr int NB = 4 * TB;              // blocks of a tile
    static constexpr int TILE = NB * kKv4Block;    // positions of a tile
    static constexpr int TP = 4 / G;               // warps that share a group in the value pass
    static constexpr int PB = NB / TP;             // blocks a warp takes in the value pass
    static constexpr int BLK = kv4_block_bytes(D);
    static constexpr int STAGE = NB * BLK;
    static constexpr int STAGES = 2;
    static constexpr int KS = D / 16;              // MMA steps over a head
    static constexpr int QW = F32 ? 16 : 8;        // bytes of a lane's query operand per step
    static constexpr int PS = 20;                  // floats from one row's weights of a block to the next (no bank conflicts)
    static constexpr int OFF_Q = STAGES * STAGE;
    static constexpr int OFF_P = OFF_Q + KS * NT * 32 * QW;
    static constexpr int P_BYTES = NB * ROWS * PS * 4;              // one buffer of weights
    static constexpr int RED_BYTES = (TP - 1) * ROWS * D * 4;       // partial sums of the value pass meet in the same place
    static constexpr int P_TOTAL = 2 * P_BYTES > RED_BYTES ? 2 * P_BYTES : RED_BYTES;
    static constexpr int OFF_M = OFF_P + P_TOTAL;                   // [2][4][ROWS] references the warps used for a tile
    static constexpr int OFF_FL = OFF_M + 8 * ROWS * 4;             // [2][4] whether a warp moved a row's reference
    static constexpr int OFF_QS = OFF_FL + 32;                      // [G][ROWS] sums of the queries' groups
    static constexpr int OFF_RF = OFF_QS + G * ROWS * 4;            // [ROWS] factor that makes a score of the MMA's sum
    static constexpr int OFF_L = OFF_RF + ROWS * 4;                 // [4][ROWS] sums of the warps' weights
    static constexpr int OFF_BAR = (OFF_L + 4 * ROWS * 4 + 15) / 16 * 16;
    static constexpr int SMEM = OFF_BAR + STAGES * 8 + 16;
};
constexpr float kRefAbove = 8.0f;    // a new reference lies this far above the row's largest score (weights stay at most 1)
constexpr float kProdTop = 32768.0f; // weight * scale * power of two: at most this,
constexpr int kProdSet = 7;          // and log2 of where a new power puts the largest

// A unit of work and the tiles of it that exist.
struct AttnUnit {
    int b, h, rt;        // sequence, KV head, row tile
    int row0, q_len, len;
    int t_lo, n_tiles;   // first position (multiple of the tile) and tiles
    int seen;            // first position that a row of the sequence sees
};

// What a unit costs beside its tiles (queries staged, result written), in tiles: counted where tiles are dealt to CTAs, or a
// CTA that got many short sequences would finish last (48 sequences of 100 to 16,000 positions, when a tile took a third
// longer: 110 us without, 76 with 3; later 58.2 us with 1, 57.4 with 2, 59.4 with 3).
constexpr int kUnitCost = 2;

// Row tiles of a sequence and tiles of each (SPLIT: every row tile of a sequence counts the same positions).
template <class C>
__device__ __forceinline__ void attn_seq_tiles(const AttnArgs& a, const Kv4Seq& s, int& rts, int& lo, int& tiles) {
    rts = (int)(((int64_t)s.q_len * a.group + C::ROWS - 1) / C::ROWS);
    lo = first_seen(a, s.len, s.q_len) / C::TILE * C::TILE;
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
        const Kv4Seq s = attn_seq(a, b, err);
        int rts, lo, tiles;
        attn_seq_tiles<C>(a, s, rts, lo, tiles);
        return (long long)rts * (tiles + kUnitCost) * a.cache.kv_heads;
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
    long long step = 1;  // the line is cut at its tiles
    if constexpr (!C::F32 && C::NT == 2) {  // (whole: prompts of bf16 rows, which have more than eight)
        if (a.whole && total > 0) {
            int rts, lo, tiles;
            attn_seq_tiles<C>(a, attn_seq(a, 0, err), rts, lo, tiles);
            step = tiles + kUnitCost;
        }
    }
    const long long steps = total / step, parts = min((long long)gridDim.x, steps);
    if (blockIdx.x >= parts) return p;
    p.begin = steps * blockIdx.x / parts * step;
    p.end = steps * (blockIdx.x + 1) / parts * step;
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
}
// The eight nibbles of a word as four pairs of f16 subnormals: the pattern n is n 2^-24, n << 4 is 16 n 2^-24, both exact.
// bf16 rows: where the nibbles lie, a mask per pair (words 1 and 3 count 16 times: the other operand or the sum makes up for
// it).  The tensor core aligns products by their exponents, and a subnormal's is that of 2^-14, so n << 4 keeps four more bits
// of a sum: kWide (f32 rows) moves all of them there.  Measured when chosen (250,001 positions, f32): 54.3 us and 6.5e-6 off
// where they lie, 57.3 us and 9.6e-7 wide, 57.5 us and 6.0e-7 with n - 8 made a normal number (two instructions more per pair);
// the ragged bf16 batch 61.1 us with n - 8, 57.4 where they lie.  kFlip: words 2 and 3 hold 15 - n.
constexpr float kSub = 16777216.0f;  // 2^24
template <bool kWide, bool kFlip = false>
__device__ __forceinline__ void nibbles_sub(uint32_t w, uint32_t (&o)[4]) {
    if constexpr (kWide) {
        const uint32_t wl = w << 4, wr = w >> 4, w8 = w >> 8;
        o[0] = wl & 0x00F000F0u;
        o[1] = w & 0x00F000F0u;
        o[2] = (kFlip ? ~wr : wr) & 0x00F000F0u;
        o[3] = (kFlip ? ~w8 : w8) & 0x00F000F0u;
        return;
    }
    const uint32_t w8 = w >> 8;
    o[0] = w & 0x000F000Fu;
    o[1] = w & 0x00F000F0u;
    o[2] = (kFlip ? ~w8 : w8) & 0x000F000Fu;
    o[3] = (kFlip ? ~w8 : w8) & 0x00F000F0u;
}
// the largest; NaN if one is
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ int exponent_of(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }  // of a positive number (-127 below 2^-126)
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <class C, typename T>
__global__ void __launch_bounds__(128) __maxnreg__(C::NT == 1 ? 128 : 168) kv4_attn_kernel(AttnArgs a, unsigned int* err) {
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ long long red[8];
    constexpr int D = C::D, G = C::G, NT = C::NT, ROWS = C::ROWS, NB = C::NB, TILE = C::TILE, TB = C::TB, PB = C::PB, PS = C::PS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    int* abort_flag = reinterpret_cast<int*>(full + C::STAGES);
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) mbar_init(full + i, 1);
        mbar_fence_init();
        *abort_flag = 0;
    }
    pdl_trigger();
    pdl_wait();  // (behind a prompt kernel: that one still reads the work area)

    // this CTA's tiles [w_begin, w_end) of the line of all tiles (SPLIT), or one unit
    long long w_begin = 0, w_end = 0, w_at = 0;
    AttnUnit u{};
    {
        AttnPlan p;
        if constexpr (C::SPLIT) {
            p = attn_scan<C>(a, 128, red, err);
            w_begin = p.begin;
            w_end = p.end;
            if (w_begin >= w_end) return;
            const Kv4Seq s = attn_seq(a, p.b, err);
            int rts;
            attn_seq_tiles<C>(a, s, rts, u.t_lo, u.n_tiles);
            u.b = p.b; u.row0 = s.row0; u.q_len = s.q_len; u.len = s.len; u.seen = first_seen(a, s.len, s.q_len);
            const long long in = w_begin - p.prefix;
            const int unit = (int)(in / (u.n_tiles + kUnitCost));
            u.h = unit / rts;
            u.rt = unit - u.h * rts;
            w_at = p.prefix + (long long)unit * (u.n_tiles + kUnitCost);  // where the unit begins: kUnitCost steps, then its tiles
        } else {
            // one unit per CTA, the units of a sequence's last rows (the longest) first; units are counted in row tiles
            const int h = blockIdx.x % a.cache.kv_heads;
            const RowTile where = locate_row_tile(a, blockIdx.x / a.cache.kv_heads, ROWS, 128, red, err);
            if (where.b >= a.seqs.n_seqs) return;
            const Kv4Seq s = attn_seq(a, where.b, err);
            u.b = where.b; u.h = h; u.rt = where.rts - 1 - where.rt;
            u.row0 = s.row0; u.q_len = s.q_len; u.len = s.len; u.seen = first_seen(a, s.len, s.q_len);
            const int j0 = u.rt * ROWS / a.group, j1 = min((u.rt * ROWS + ROWS - 1) / a.group, s.q_len - 1);
            const int p0 = s.len - s.q_len + j0, p1 = s.len - s.q_len + j1;
            u.t_lo = window_from(a, p0) / TILE * TILE;
            u.n_tiles = max((p1 + 1 - u.t_lo + TILE - 1) / TILE, 1);
            w_begin = 0; w_end = u.n_tiles + kUnitCost; w_at = 0;
        }
    }
    __syncthreads();

    // steps to the unit behind u
    auto next_unit = [&](AttnUnit& n, long long& at) {
        at += n.n_tiles + kUnitCost;
        int rts, lo, tiles;
        Kv4Seq s{n.row0, n.q_len, n.len};
        attn_seq_tiles<C>(a, s, rts, lo, tiles);
        if (++n.rt < rts) return;
        n.rt = 0;
        if (++n.h < a.cache.kv_heads) return;
        n.h = 0;
        do {
            if (++n.b >= a.seqs.n_seqs) return;
            s = attn_seq(a, n.b, err);
        } while (s.q_len == 0);
        n.row0 = s.row0; n.q_len = s.q_len; n.len = s.len; n.seen = first_seen(a, s.len, s.q_len);
        attn_seq_tiles<C>(a, s, rts, n.t_lo, n.n_tiles);
    };

    // The first warp also brings the tiles in, one ahead: a tile's place is free once all warps have met at the barrier of the
    // tile after it.  Blocks that lie in one page are one copy (a.run of them: a power of two that divides a page's blocks and
    // a tile's).  The pages are looked up another tile before, so that the table's latency is not waited for; the
    // others wait for this warp, so a position's page is found without a division (57.3 us with it on one long sequence, 55.9).
    int nx_page = 0, nx_block = -1;  // lane: page and first block of its run in the tile to copy next; block -1: none
    auto look_up = [&](const AttnUnit& n, int t) {
        nx_block = -1;
        const int pos = n.t_lo + t * TILE + lane * a.run * kKv4Block;
        if (lane * a.run < NB && pos < n.len && pos + a.run * kKv4Block > n.seen) {
            const int pg = over_group(pos, a.by_page);
            nx_block = (int)((unsigned)(pos - pg * a.cache.page_size) / kKv4Block);
            nx_page = -1;
            if (pg < a.seqs.max_pages) nx_page = a.seqs.page_table[(size_t)n.b * a.seqs.max_pages + pg];
        }
    };
    const unsigned page_blocks = (unsigned)a.cache.page_size / kKv4Block;  // a block's number fits 32 bits: 2^32 blocks are 4.9 TB
    auto copy_in = [&](int h, int st) {
        bool copy = nx_block >= 0;
        if (copy && (nx_page < 0 || nx_page >= a.cache.num_pages)) {
            atomicExch(err, kErrKv4Page);
            copy = false;
        }
        const unsigned have = __ballot_sync(0xffffffffu, copy);
        if (lane == 0) mbar_expect_tx(full + st, __popc(have) * a.run * C::BLK);
        __syncwarp();
        if (copy)
            bulk_g2s(sm + st * C::STAGE + lane * a.run * C::BLK,
                     a.cache.pages + (size_t)(((unsigned)nx_page * a.cache.kv_heads + h) * page_blocks + nx_block) * C::BLK,
                     a.run * C::BLK, full + st);
    };
    auto first_of = [&](long long at) { return (int)max(w_begin - at - kUnitCost, 0ll); };
    auto stop_of = [&](const AttnUnit& n, long long at) { return (int)min(w_end - at - kUnitCost, (long long)n.n_tiles); };
    // the first tile of the units behind (n, at), if there is one
    auto bring_next_unit = [&](AttnUnit n, long long at, int st) {
        while (at + n.n_tiles + kUnitCost < w_end) {
            next_unit(n, at);
            if (stop_of(n, at) > 0) {
                look_up(n, 0);
                copy_in(n.h, st);
                return;
            }
        }
    };
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    if (warp == 0) {
        const int t = first_of(w_at);
        if (t < stop_of(u, w_at)) {
            look_up(u, t);
            copy_in(u.h, 0);
        } else {
            bring_next_unit(u, w_at, 0);
        }
    }

    const int r = lane >> 2, c = lane & 3;      // scores: positions 2 r, 2 r + 1 of a block, rows 2 c, 2 c + 1 of eight
    const int g_own = warp % G, tp = warp / G;  // value pass: group, part of the positions; weights: row r, positions 4 c ..
    const T* qp = (const T*)a.q;
    const T* gatep = (const T*)a.gate;
    T* outp = (T*)a.out;
    float* q_sum = reinterpret_cast<float*>(sm + C::OFF_QS);
    float* row_f = reinterpret_cast<float*>(sm + C::OFF_RF);
    float* refs = reinterpret_cast<float*>(sm + C::OFF_M);
    unsigned* flags = reinterpret_cast<unsigned*>(sm + C::OFF_FL);
    float* sums = reinterpret_cast<float*>(sm + C::OFF_L);
    for (bool more = true; more && ok;) {
        const int t_first = first_of(w_at), t_stop = stop_of(u, w_at);
        if (warp == 0 && t_first + 1 < t_stop) look_up(u, t_first + 1);
        const int rows_all = u.q_len * a.group;
        const int pos_base = u.len - u.q_len;

        // queries of the unit as MMA operands: a warp takes a row at a time; scaled by a power of two so that the largest
        // element lies in [2^14, 2^15)
        // a lane takes eight elements of a row, D / 8 lanes a row; all of a warp's rows are requested before the first is used
        constexpr int LPR = D / 8, RPL = 32 / LPR, NL = ROWS / 4 / RPL > 0 ? ROWS / 4 / RPL : 1;
        const int sub = lane / LPR, lc = lane % LPR;
        if (warp * NL * RPL < ROWS) {  // fewer rows than the four warps' lanes can take: the first warps do it
            float xq[NL][8];
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int rr = u.rt * ROWS + (warp * NL + i) * RPL + sub;
                const bool valid = rr < rows_all;
                const int j = valid ? over_group(rr, a.by_group) : 0, hq = u.h * a.group + (valid ? rr - j * a.group : 0);
#pragma unroll
                for (int k = 0; k < 8; ++k) xq[i][k] = 0.0f;
                if (valid) ld_act8(qp + (int64_t)(u.row0 + j) * a.qt + (int64_t)hq * a.qh + 8 * lc, a.vec_q, xq[i]);
            }
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int row = (warp * NL + i) * RPL + sub;
                float (&x)[8] = xq[i];
                float mx = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(x[k]));
#pragma unroll
                for (int k = 1; k < LPR; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
                const int e = max((int)(__float_as_uint(mx) >> 23) - 127, -110);  // mx in [2^e, 2^(e + 1))
                const float up = pow2f(min(14 - e, 127));
                // elements (0, 4), (1, 5) of the eight are a step's operand, (2, 6), (3, 7) the next one's
                uint32_t hi[4], lo[4];
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float sh = !C::F32 && (k & 1) ? 0.0625f : 1.0f;  // odd words of nibbles_sub count 16 times
                    const float v0 = x[k] * up * sh, v1 = x[k + 4] * up * sh;
                    const __half2 h = __floats2half2_rn(v0, v1);
                    const float2 f = __half22float2(h);
                    hi[k] = h2_bits(h);
                    lo[k] = h2_bits(__floats2half2_rn(v0 - f.x, v1 - f.y));
                    sum = fmaf(C::F32 ? v0 + v1 : f.x + f.y, !C::F32 && (k & 1) ? 16.0f : 1.0f, sum);
                }
#pragma unroll
                for (int k = 1; k < 8; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);  // over the group of 64
                const int g = lc >> 3, cc = (lc >> 1) & 3, jj = lc & 1;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    uint8_t* dst = sm + C::OFF_Q + (((g * 4 + jj * 2 + v) * NT + (row >> 3)) * 32 + (row & 7) * 4 + cc) * C::QW;
                    if constexpr (C::F32) *reinterpret_cast<uint4*>(dst) = make_uint4(hi[2 * v], hi[2 * v + 1], lo[2 * v], lo[2 * v + 1]);
                    else *reinterpret_cast<uint2*>(dst) = make_uint2(hi[2 * v], hi[2 * v + 1]);
                }
                if ((lc & 7) == 0) q_sum[g * ROWS + row] = sum;
                if (lc == 0) row_f[row] = a.scale_log2 * pow2f(max(e - 14, -126));
            }
        }
        compute_barrier();

        // rows 2 c and 2 c + 1 of every eight
        float ref[NT][2], l_run[NT][2], rf[NT][2];
        int see_hi[NT][2], see_lo[NT][2];  // positions the row sees: see_lo <= t <= see_hi
        int all_hi = 0x7FFFFFFF, all_lo = -1;
        float o[NT][4][4], o_bias[NT];     // elements 8 r + 2 x and + 1 of the group, rows 2 c and 2 c + 1; row r
        float power[NT];                   // row r: its products are taken times this power of two, o with them
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            o_bias[nt] = 0.0f;
            power[nt] = pow2f(126);        // the first product lowers it
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                ref[nt][e] = -INFINITY;
                l_run[nt][e] = 0.0f;
                const int row = nt * 8 + 2 * c + e, rr = u.rt * ROWS + row;
                rf[nt][e] = row_f[row];
                // rows behind the last are computed unmasked and not written
                see_hi[nt][e] = rr < rows_all ? pos_base + over_group(rr, a.by_group) : 0x7FFFFFFF;
                see_lo[nt][e] = rr < rows_all ? window_from(a, see_hi[nt][e]) : 0;
                all_hi = min(all_hi, see_hi[nt][e]);
                all_lo = max(all_lo, see_lo[nt][e]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][x][i] = 0.0f;
        }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
            all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, s));
            all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, s));
        }
        float qs_reg[NT == 1 ? G : 1][2];  // sums of the queries' groups, from shared memory where there are more rows
        if constexpr (NT == 1) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                qs_reg[g][0] = q_sum[g * ROWS + 2 * c];
                qs_reg[g][1] = q_sum[g * ROWS + 2 * c + 1];
            }
        }

        // row r's products times 2^k from now on, its sums so far times 2^(by + part) (not above 1)
        auto set_power = [&](int nt, int k, int by, float part) {
            power[nt] = pow2f(k);
            const float f = pow2f(max(by, -126)) * exp2_approx(part);
            const float f0 = __shfl_sync(0xffffffffu, f, 8 * c), f1 = __shfl_sync(0xffffffffu, f, 8 * c + 4);  // of rows 2 c, 2 c + 1
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                o[nt][x][0] *= f0;
                o[nt][x][1] *= f1;
                o[nt][x][2] *= f0;
                o[nt][x][3] *= f1;
            }
        };

        int buf = 0;
        for (int ti = t_first; ti < t_stop; ++ti, buf ^= 1) {
            const int t0 = u.t_lo + ti * TILE;
            ok = mbar_wait(full + stage, phase);
            if (!ok) *abort_flag = 1;
            const uint8_t* st = sm + stage * C::STAGE;
            // ── scores ──
            float s[TB][NT][4];  // (position 2 r, rows 2 c, 2 c + 1), (position 2 r + 1, the same rows)
#pragma unroll
            for (int tb = 0; tb < TB; ++tb) {
                const uint8_t* kb = st + (warp * TB + tb) * C::BLK;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[tb][nt][i] = 0.0f;
                constexpr int U = G >= 2 ? 2 : 1;
#pragma unroll
                for (int it = 0; it < G / U; ++it) {
                    uint32_t kw[2][2 * U];  // position parity, word of (group, j)
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
                        float acc[NT][4], acc_lo[C::F32 ? NT : 1][4];  // f32 rows: high and low terms apart, two chains of MMAs at a time
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            uint32_t nb[2][4];
                            nibbles_sub<C::F32>(kw[0][uu * 2 + j], nb[0]);
                            nibbles_sub<C::F32>(kw[1][uu * 2 + j], nb[1]);
#pragma unroll
                            for (int v = 0; v < 2; ++v) {
                                const uint4 ka = make_uint4(nb[0][2 * v], nb[1][2 * v], nb[0][2 * v + 1], nb[1][2 * v + 1]);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    const uint8_t* qa = sm + C::OFF_Q + (((g * 4 + j * 2 + v) * NT + nt) * 32 + lane) * C::QW;
                                    if constexpr (C::F32) {
                                        const uint4 qf = *reinterpret_cast<const uint4*>(qa);
                                        if (j == 0 && v == 0) {
                                            mma_f16_zero(acc[nt], ka, qf.x, qf.y);
                                            mma_f16_zero(acc_lo[nt], ka, qf.z, qf.w);
                                        } else {
                                            mma_f16(acc[nt], ka, qf.x, qf.y);
                                            mma_f16(acc_lo[nt], ka, qf.z, qf.w);
                                        }
                                    } else {
                                        const uint2 qf = *reinterpret_cast<const uint2*>(qa);
                                        if (j == 0 && v == 0) mma_f16_zero(acc[nt], ka, qf.x, qf.y);
                                        else mma_f16(acc[nt], ka, qf.x, qf.y);
                                    }
                                }
                            }
                        }
                        const uint2 pr = *reinterpret_cast<const uint2*>(kb + 8 * D + g * 64 + r * 8);
                        const uint32_t pw[2] = {pr.x, pr.y};
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float sc = __uint_as_float(pw[k] << 16) * (C::F32 ? kSub / 16.0f : kSub), bi = __uint_as_float(pw[k] & 0xFFFF0000u);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float qs = NT == 1 ? qs_reg[NT == 1 ? g : 0][e] : q_sum[g * ROWS + nt * 8 + 2 * c + e];
                                    const float dot = C::F32 ? acc[nt][2 * k + e] + acc_lo[C::F32 ? nt : 0][2 * k + e] : acc[nt][2 * k + e];
                                    s[tb][nt][2 * k + e] = fmaf(sc, dot, fmaf(bi, qs, s[tb][nt][2 * k + e]));
                                }
                        }
                    }
                }
            }
            // weights
            const bool whole = t0 + TILE - 1 <= all_hi && t0 >= all_lo;
            float use[NT][2], sum[NT][2];
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[tb][nt][i] *= rf[nt][i & 1];
            if (!whole) {
#pragma unroll
                for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int pos = t0 + (warp * TB + tb) * kKv4Block + 2 * r + (i >> 1);
                            if (pos > see_hi[nt][i & 1] || pos < see_lo[nt][i & 1]) s[tb][nt][i] = -INFINITY;
                        }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    use[nt][e] = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
                    for (int tb = 1; tb < TB; ++tb) use[nt][e] = fmaxf(use[nt][e], fmaxf(s[tb][nt][e], s[tb][nt][2 + e]));
                }
#pragma unroll
            for (int k = 4; k < 32; k <<= 1)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) use[nt][e] = fmaxf(use[nt][e], __shfl_xor_sync(0xffffffffu, use[nt][e], k));
            bool moved = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool mv = use[nt][e] > ref[nt][e];
                    moved |= mv;
                    use[nt][e] = mv ? use[nt][e] + kRefAbove : ref[nt][e];
                    const float off = use[nt][e] == -INFINITY ? 0.0f : use[nt][e];
                    sum[nt][e] = 0.0f;
#pragma unroll
                    for (int tb = 0; tb < TB; ++tb) {
                        s[tb][nt][e] = exp2_approx(s[tb][nt][e] - off);
                        s[tb][nt][2 + e] = exp2_approx(s[tb][nt][2 + e] - off);
                        sum[nt][e] += s[tb][nt][e] + s[tb][nt][2 + e];
                        *reinterpret_cast<float2*>(sm + C::OFF_P + buf * C::P_BYTES + (((warp * TB + tb) * ROWS + nt * 8 + 2 * c + e) * PS + 2 * r) * 4) =
                            make_float2(s[tb][nt][e], s[tb][nt][2 + e]);
                    }
                }
            moved = __any_sync(0xffffffffu, moved);
            if (r == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    *reinterpret_cast<float2*>(refs + (buf * 4 + warp) * ROWS + nt * 8 + 2 * c) = make_float2(use[nt][0], use[nt][1]);
            }
            if (lane == 0) flags[buf * 4 + warp] = moved;
            compute_barrier();
            if (*(volatile int*)abort_flag) ok = false;
            if (warp == 0 && ok) {
                if (ti + 1 < t_stop) {
                    copy_in(u.h, stage ^ 1);
                    if (ti + 2 < t_stop) look_up(u, ti + 2);
                } else {
                    bring_next_unit(u, w_at, stage ^ 1);
                }
            }
            // ── values ──
            const uint4 fl = *reinterpret_cast<const uint4*>(flags + buf * 4);
            const bool any_moved = (fl.x | fl.y | fl.z | fl.w) != 0;
            if (any_moved) {
                // rare: the rows' references become the largest of the warps'; every warp corrects the weights it wrote
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float fix[2], up[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = nt * 8 + 2 * c + e;
                        float m = ref[nt][e];
#pragma unroll
                        for (int i = 0; i < 4; ++i) m = fmaxf(m, refs[(buf * 4 + i) * ROWS + row]);
                        const float off = m == -INFINITY ? 0.0f : m, f = exp2_approx(use[nt][e] - off);
                        fix[e] = exp2_approx(ref[nt][e] - off);
                        up[e] = m > ref[nt][e] ? m - ref[nt][e] : 0.0f;  // infinite from none
                        l_run[nt][e] *= fix[e];
                        sum[nt][e] *= f;
                        ref[nt][e] = m;
#pragma unroll
                        for (int tb = 0; tb < TB; ++tb)
                            *reinterpret_cast<float2*>(sm + C::OFF_P + buf * C::P_BYTES + (((warp * TB + tb) * ROWS + row) * PS + 2 * r) * 4) =
                                make_float2(s[tb][nt][e] * f, s[tb][nt][2 + e] * f);
                    }
                    // row r: its correction is held by lane r / 2 (rows 2 c, 2 c + 1)
                    const float x0 = __shfl_sync(0xffffffffu, fix[0], r >> 1), x1 = __shfl_sync(0xffffffffu, fix[1], r >> 1);
                    const float u0 = __shfl_sync(0xffffffffu, up[0], r >> 1), u1 = __shfl_sync(0xffffffffu, up[1], r >> 1);
                    o_bias[nt] *= (r & 1) ? x1 : x0;
                    // the sums of the products stay what they are, their power of two grows with the reference
                    const float u = fminf((r & 1) ? u1 : u0, 1000.0f), whole_u = floorf(u);
                    const int k = exponent_of(power[nt]) + (int)whole_u;
                    set_power(nt, min(k, 126), min(126 - k, 0), whole_u - u);
                }
                compute_barrier();
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) l_run[nt][e] += sum[nt][e];
            float acc[C::F32 ? NT : 1][4][4];  // f32 rows: the tile's sums, added to the unit's with f32 rounding
            // positions 1 and 3 of four: 15 - n under a negative weight, so that the sums of the nibbles, whose middle is 7.5, have
            // no drift: the tensor core's truncating sums then stay relative to what they hold (f32 rows over 250,001 positions:
            // 9.6e-7 off; 1.5e-5 with n - 8 at every position)
            uint8_t* pairs = sm + stage * C::STAGE + 17 * D + g_own * 64 + c * 16;                                          // of positions 4 c ..
            const float* weights = reinterpret_cast<const float*>(sm + C::OFF_P + buf * C::P_BYTES) + r * PS + 4 * c;  // of row r
            using Pairs = uint32_t[NT][2];
            using Lows = uint32_t[C::F32 ? NT : 1][2];
            // operands of a block for this warp's group: weight times scale times the power of two; the weighted sum of the biases
            // so far; the largest product (NaN where there is one)
            auto weigh = [&](int pb, Pairs& b, Lows& lo, float* ob, float& top) {
                const int blk = tp * PB + pb;
                const uint4 pr = *reinterpret_cast<const uint4*>(pairs + blk * C::BLK);
                const uint32_t pw[4] = {pr.x, pr.y, pr.z, pr.w};
                float sc[4], bi[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    sc[k] = __uint_as_float(pw[k] << 16);
                    bi[k] = __uint_as_float(pw[k] & 0xFFFF0000u);
                    if (k & 1) bi[k] = fmaf(15.0f, sc[k], bi[k]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float4 p = *reinterpret_cast<const float4*>(weights + (blk * ROWS + nt * 8) * PS);
                    ob[nt] = fmaf(p.x, bi[0], fmaf(p.y, bi[1], fmaf(p.z, bi[2], fmaf(p.w, bi[3], ob[nt]))));
                    // (in this order nothing that is hidden, a weight of 0, overflows)
                    p.x = p.x * power[nt] * sc[0]; p.y = p.y * power[nt] * sc[1]; p.z = p.z * power[nt] * sc[2]; p.w = p.w * power[nt] * sc[3];
                    top = max_nan(max_nan(top, p.x, p.y), p.z, p.w);
                    const __half2 h02 = __floats2half2_rn(p.x, p.z), h13 = __floats2half2_rn(-p.y, -p.w);
                    b[nt][0] = h2_bits(h02);
                    b[nt][1] = h2_bits(h13);
                    if constexpr (C::F32) {
                        const float2 f02 = __half22float2(h02), f13 = __half22float2(h13);
                        lo[nt][0] = h2_bits(__floats2half2_rn(p.x - f02.x, p.z - f02.y));
                        lo[nt][1] = h2_bits(__floats2half2_rn(-p.y - f13.x, -p.w - f13.y));
                    }
                }
            };
            auto multiply = [&](int pb, auto first, const Pairs& b, const Lows& lo) {
                const uint4 vw = *reinterpret_cast<const uint4*>(st + (tp * PB + pb) * C::BLK + 9 * D + g_own * 512 + lane * 16);
                uint32_t nb[4][4];  // word x: elements 8 r + 2 x, 8 r + 2 x + 1 of positions (0, 2), then of (1, 3)
                nibbles_sub<C::F32, true>(vw.x, nb[0]);
                nibbles_sub<C::F32, true>(vw.y, nb[1]);
                nibbles_sub<C::F32, true>(vw.z, nb[2]);
                nibbles_sub<C::F32, true>(vw.w, nb[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint4 va = make_uint4(nb[x][0], nb[x][1], nb[x][2], nb[x][3]);
                        if constexpr (C::F32) {
                            if constexpr (decltype(first)::value) mma_f16_zero(acc[nt][x], va, b[nt][0], b[nt][1]);
                            else mma_f16(acc[nt][x], va, b[nt][0], b[nt][1]);
                            mma_f16(acc[nt][x], va, lo[nt][0], lo[nt][1]);
                        } else {
                            mma_f16(o[nt][x], va, b[nt][0], b[nt][1]);
                        }
                    }
            };
            // Rare: something is NaN.  Pairs that are (or were never written) are taken out, and the rows that see them get a NaN.
            auto take_out = [&]() {
#pragma unroll 1
                for (int i = 0; i < 4 * PB; ++i) {
                    const int blk = tp * PB + (i >> 2), k = i & 3;
                    uint32_t* at = reinterpret_cast<uint32_t*>(pairs + blk * C::BLK) + k;
                    const float sc = __uint_as_float(*at << 16), bi = __uint_as_float(*at & 0xFFFF0000u);
                    const bool bad = !(fabsf(sc) < INFINITY && fabsf(bi) < INFINITY && fabsf(fmaf(15.0f, sc, bi)) < INFINITY);
                    __syncwarp();  // the rows share the pairs
                    if (!bad) continue;
                    if (r == 0) *at = 0;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        if (weights[(blk * ROWS + nt * 8) * PS + k] != 0.0f) o_bias[nt] = NAN;
                }
                umma::fence_smem_to_async();  // before the copies that come here next
                __syncwarp();
            };
            // Rare: a reference moved or a product is too large.  Smaller powers of two for the rows that need them.
            auto lower_powers = [&]() {
                float m[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) m[nt] = 0.0f;
#pragma unroll(NT == 1 ? PB : 1)
                for (int pb = 0; pb < PB; ++pb) {
                    const uint4 pr = *reinterpret_cast<const uint4*>(pairs + (tp * PB + pb) * C::BLK);
                    const float sc[4] = {__uint_as_float(pr.x << 16), __uint_as_float(pr.y << 16), __uint_as_float(pr.z << 16), __uint_as_float(pr.w << 16)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {  // (fmaxf leaves NaN out)
                        const float4 p = *reinterpret_cast<const float4*>(weights + ((tp * PB + pb) * ROWS + nt * 8) * PS);
                        m[nt] = fmaxf(fmaxf(m[nt], fmaxf(p.x * sc[0], p.y * sc[1])), fmaxf(p.z * sc[2], p.w * sc[3]));
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    m[nt] = fmaxf(m[nt], __shfl_xor_sync(0xffffffffu, m[nt], 1));
                    m[nt] = fmaxf(m[nt], __shfl_xor_sync(0xffffffffu, m[nt], 2));
                    const int old = exponent_of(power[nt]), k = m[nt] * power[nt] > kProdTop ? min(kProdSet - exponent_of(m[nt]), 126) : old;
                    set_power(nt, k, k - old, 0.0f);
                }
            };
            Pairs b[C::F32 ? 1 : PB];
            Lows lo;
            float ob[NT];
            bool again = any_moved;
#pragma unroll 1
            for (int attempt = 0; attempt < 2; ++attempt) {
                if (attempt > 0) take_out();
                if (again) lower_powers();
                float top = 0.0f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) ob[nt] = o_bias[nt];
                // f32 rows add a tile up by itself, so they look at its products afterwards; the others before
                weigh(0, b[0], lo, ob, top);
                if constexpr (C::F32) multiply(0, std::true_type{}, b[0], lo);
#pragma unroll
                for (int pb = 1; pb < PB; ++pb) {
                    weigh(pb, b[C::F32 ? 0 : pb], lo, ob, top);
                    if constexpr (C::F32) multiply(pb, std::false_type{}, b[0], lo);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) top = max_nan(top, ob[nt] * 0.0f, 0.0f);
                again = __any_sync(0xffffffffu, !(top <= kProdTop));
                if (!again) break;
            }
            if constexpr (!C::F32) {
#pragma unroll
                for (int pb = 0; pb < PB; ++pb) multiply(pb, std::false_type{}, b[pb], lo);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) o_bias[nt] = ob[nt];
            if constexpr (C::F32) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[nt][x][i] += acc[nt][x][i];
            }
            phase ^= stage;
            stage ^= 1;
            if (!ok) break;
        }
        if (!ok) break;

        // ── the unit's end: sums of the warps' weights, sums of the value pass ──
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = l_run[nt][e];
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
                if (r == 0) sums[warp * ROWS + nt * 8 + 2 * c + e] = l;
            }
            float ob = o_bias[nt];
            ob += __shfl_xor_sync(0xffffffffu, ob, 1);
            ob += __shfl_xor_sync(0xffffffffu, ob, 2);
            const float down = __uint_as_float(0x7F000000u - __float_as_uint(power[nt]));  // 1 / power
            const float b0 = __shfl_sync(0xffffffffu, ob, 8 * c), b1 = __shfl_sync(0xffffffffu, ob, 8 * c + 4);  // of rows 2 c, 2 c + 1
            const float d0 = __shfl_sync(0xffffffffu, down, 8 * c), d1 = __shfl_sync(0xffffffffu, down, 8 * c + 4);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                o[nt][x][0] = fmaf(o[nt][x][0] * (C::F32 ? kSub / 16.0f : kSub), d0, b0);
                o[nt][x][1] = fmaf(o[nt][x][1] * (C::F32 ? kSub / 16.0f : kSub), d1, b1);
                o[nt][x][2] = fmaf(o[nt][x][2] * (kSub / 16.0f), d0, b0);
                o[nt][x][3] = fmaf(o[nt][x][3] * (kSub / 16.0f), d1, b1);
            }
        }
        const bool whole_unit = w_at >= w_begin && w_at + u.n_tiles + kUnitCost <= w_end;
        const int d0 = 64 * g_own + 8 * r;
        // the gates of all of this lane's rows are requested before the first is used
        float gt[NT][2][8];
        if (gatep && tp == 0 && (!C::SPLIT || whole_unit)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int rr = min(u.rt * ROWS + nt * 8 + 2 * c + e, rows_all - 1);
                    const int j = over_group(rr, a.by_group);
                    ld_act8(gatep + (int64_t)(u.row0 + j) * a.gt + (int64_t)(u.h * a.group + rr - j * a.group) * a.gh + d0, a.vec_gate, gt[nt][e]);
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int n = 0; n < 8; ++n) gt[nt][e][n] = sigmoid<T>(gt[nt][e][n]);
        }
        compute_barrier();
        float* slot = nullptr;
        if (C::SPLIT && !whole_unit) slot = a.part + (size_t)(2 * blockIdx.x + (w_at <= w_begin ? 0 : 1)) * ROWS * (D + 2);
        float* red_o = reinterpret_cast<float*>(sm + C::OFF_P);
        if (C::TP > 1) {
            if (tp > 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float4* d = reinterpret_cast<float4*>(red_o + ((size_t)(tp - 1) * ROWS + nt * 8 + 2 * c + e) * D + d0);
                        d[0] = make_float4(o[nt][0][e], o[nt][0][2 + e], o[nt][1][e], o[nt][1][2 + e]);
                        d[1] = make_float4(o[nt][2][e], o[nt][2][2 + e], o[nt][3][e], o[nt][3][2 + e]);
                    }
            }
            compute_barrier();
        }
        if (tp == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = nt * 8 + 2 * c + e;
                    float y[8];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        y[2 * x] = o[nt][x][e];
                        y[2 * x + 1] = o[nt][x][2 + e];
                    }
#pragma unroll
                    for (int t = 0; t < C::TP - 1; ++t) {
                        const float* d = red_o + ((size_t)t * ROWS + row) * D + d0;
#pragma unroll
                        for (int n = 0; n < 8; ++n) y[n] += d[n];
                    }
                    const float l = (sums[row] + sums[ROWS + row]) + (sums[2 * ROWS + row] + sums[3 * ROWS + row]);
                    if (slot) {
                        st_act8(slot + (size_t)row * D + d0, true, y);
                        if (g_own == 0 && r == 0) {
                            slot[(size_t)ROWS * D + row] = ref[nt][e];
                            slot[(size_t)ROWS * (D + 1) + row] = l;
                        }
                    } else if (u.rt * ROWS + row < rows_all) {
                        const int rr = u.rt * ROWS + row, j = over_group(rr, a.by_group);
                        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            y[n] *= inv;
                            if (gatep) y[n] *= gt[nt][e][n];
                        }
                        st_act8(outp + ((int64_t)(u.row0 + j) * a.heads + u.h * a.group + rr - j * a.group) * D + d0, true, y);
                    }
                }
            }
        }
        compute_barrier();  // the weights' place and the row tables are free again
        more = w_at + u.n_tiles + kUnitCost < w_end;
        if (more) next_unit(u, w_at);
    }
    if (!ok) {  // a copy did not arrive within the limit: reported; the others in flight are waited for (again with a limit)
        if (lane == 0) atomicExch(err, 1u);
        if (warp == 0) mbar_wait(full + (stage ^ 1), stage ? phase ^ 1 : phase);
        compute_barrier();
    }
}

// Joins the partial results of units that were split over CTAs.  grid: x = units (or, where there are more of those, the
// borders between CTAs: a border splits at most one unit, and a unit is joined by the first border inside it), y = pieces of
// a unit's rows x elements: 256 / parts float4 each, `parts` threads of the CTA sharing an element's partial sums (few parts
// where a unit has few partial results).  The plan is made before the wait: the batch's arrays were there before the
// attention kernel.
template <class C, typename T>
__global__ void __launch_bounds__(256) kv4_attn_join_kernel(AttnArgs a, int splits, int row_tiles, int by_border, int parts, unsigned int* err) {
    constexpr int D = C::D, ROWS = C::ROWS;
    __shared__ long long red[8], found[4];
    __shared__ float4 acc_s[256];
    __shared__ float m_s[256], l_s[256];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto cost = [&](int b, int& rts, int& tiles) -> long long {
        int lo;
        const Kv4Seq s = attn_seq(a, b, err);
        attn_seq_tiles<C>(a, s, rts, lo, tiles);
        tiles += kUnitCost;
        return (long long)rts * tiles * a.cache.kv_heads;
    };
    // total of all tiles, and of those of sequences before `b_unit`
    const int b_unit = by_border ? 0 : blockIdx.x / (row_tiles * a.cache.kv_heads);
    long long mine = 0, mine_before = 0;
    for (int i = tid; i < a.seqs.n_seqs; i += 256) {
        int r2, t2;
        const long long cst = cost(i, r2, t2);
        mine += cst;
        if (i < b_unit) mine_before += cst;
    }
    auto block_sum = [&](long long v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane == 0) red[warp] = v;
        __syncthreads();
        long long t = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += red[i];
        return t;
    };
    const long long total = block_sum(mine), n = min((long long)splits, total);
    int b = b_unit, h = 0, rt = 0, tiles = 0;
    long long at = 0;
    bool work = total > 0;
    if (!by_border) {
        int rts;
        at = block_sum(mine_before);
        cost(b, rts, tiles);
        const int in = blockIdx.x % (row_tiles * a.cache.kv_heads);
        h = in / row_tiles;
        rt = in - h * row_tiles;
        work = work && rt < rts;
        at += (long long)(h * rts + rt) * tiles;
    } else {
        const long long border = blockIdx.x + 1;
        work = work && border < n;
        const long long x = work ? total * border / n : 0;
        if (work) {  // the sequence that holds tile x: chunks of 256 sequences, prefix sums by one thread each
            long long carry = 0;
            for (int b0 = 0; b0 < a.seqs.n_seqs; b0 += 256) {
                int r2 = 0, t2 = 0;
                const long long cst = b0 + tid < a.seqs.n_seqs ? cost(b0 + tid, r2, t2) : 0;
                long long inc = cst;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                __syncthreads();
                if (lane == 31) red[warp] = inc;
                __syncthreads();
                long long before = carry, sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (i < warp) before += red[i];
                    sum += red[i];
                }
                const long long lo = before + inc - cst;
                if (x >= lo && x < lo + cst) {
                    const int unit = (int)((x - lo) / t2);
                    found[0] = b0 + tid;
                    found[1] = unit;
                    found[2] = lo + (long long)unit * t2;
                }
                carry += sum;
                if (x < carry) break;
            }
            __syncthreads();
            b = (int)found[0];
            int rts;
            cost(b, rts, tiles);
            h = (int)found[1] / rts;
            rt = (int)found[1] - h * rts;
            at = found[2];
            work = at < x;  // a border between units splits none
        }
    }
    int i0 = 0, i1 = 0;
    if (work) {
        i0 = (int)(((at + 1) * n - 1) / total);
        i1 = (int)(((at + tiles) * n - 1) / total);
        work = i0 < i1 && (!by_border || i0 == (int)blockIdx.x);
    }
    pdl_wait();
    if (!work) return;
    const Kv4Seq s = attn_seq(a, b, err);
    const int rows_all = s.q_len * a.group;
    const bool first_odd = total * i0 / n < at;  // CTA i0 began before this unit: its part is in the odd slot
    auto slot_of = [&](int i) { return a.part + (size_t)(2 * i + (i == i0 && first_odd ? 1 : 0)) * ROWS * (D + 2); };
    const int per = 256 / parts, e = tid % per, part = tid / per, idx = blockIdx.y * per + e;
    const int row = idx / (D / 4), col = idx % (D / 4), rr = rt * ROWS + row;
    const bool live = row < ROWS && rr < rows_all;
    // running reference, sum of weights and sums of values; four partial results requested at a time
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float m2, float l2, const float4& v) {
        const float m_new = fmaxf(m, m2), off = m_new == -INFINITY ? 0.0f : m_new;
        const float f = exp2_approx(m - off), f2 = exp2_approx(m2 - off);
        l = fmaf(l2, f2, l * f);
        acc.x = fmaf(v.x, f2, acc.x * f); acc.y = fmaf(v.y, f2, acc.y * f);
        acc.z = fmaf(v.z, f2, acc.z * f); acc.w = fmaf(v.w, f2, acc.w * f);
        m = m_new;
    };
    if (live) {
        for (int i = i0 + part; i <= i1; i += 4 * parts) {
            float m4[4], l4[4];
            float4 v4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                m4[k] = -INFINITY;
                l4[k] = 0.0f;
                v4[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (i + k * parts <= i1) {
                    const float* sp = slot_of(i + k * parts);
                    m4[k] = sp[(size_t)ROWS * D + row];
                    l4[k] = sp[(size_t)ROWS * (D + 1) + row];
                    v4[k] = reinterpret_cast<const float4*>(sp + (size_t)row * D)[col];
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) add(m4[k], l4[k], v4[k]);
        }
    }
    for (int p = parts; p > 1; p >>= 1) {  // the threads of an element in pairs
        acc_s[tid] = acc;
        m_s[tid] = m;
        l_s[tid] = l;
        __syncthreads();
        if (part < p / 2) add(m_s[tid + p / 2 * per], l_s[tid + p / 2 * per], acc_s[tid + p / 2 * per]);
        __syncthreads();
    }
    if (!live || part != 0) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int j = over_group(rr, a.by_group), hq = h * a.group + rr - j * a.group;
    float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    if (a.gate) {
        const T* gp = (const T*)a.gate + (int64_t)(s.row0 + j) * a.gt + (int64_t)hq * a.gh + 4 * col;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] *= sigmoid<T>(ld_act(gp + i));
    }
    T* dst = (T*)a.out + ((int64_t)(s.row0 + j) * a.heads + hq) * D + 4 * col;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
}

// ─── host side ──────────────────────────────────────────────────────────────
void kv4_destroy(moe_engine* e) {
    if (e->kv4.work) cudaFree(e->kv4.work);
    if (e->kv4.wide) cudaFree(e->kv4.wide);
    e->kv4 = Kv4State{};
}

int kv4_reserve(moe_engine* e, size_t bytes) {
    if (bytes <= e->kv4.work_bytes) return MOE_OK;
    MOE_CUDA(cudaStreamSynchronize(e->stream));
    // by half at least: the chunks of a prompt need a little more each time
    size_t want = e->kv4.work_bytes + e->kv4.work_bytes / 2;
    if (want < bytes) want = bytes;
    if (e->kv4.work) cudaFree(e->kv4.work);
    e->kv4.work = nullptr;
    e->kv4.work_bytes = 0;
    cudaError_t err = cudaMalloc(&e->kv4.work, want);
    if (err != cudaSuccess && want > bytes) {
        cudaGetLastError();
        err = cudaMalloc(&e->kv4.work, want = bytes);
    }
    if (err != cudaSuccess) {
        cudaGetLastError();  // the next call starts clean
        e->kv4.work = nullptr;
        return cuda_fail(err, "kv4_attention: work area", __FILE__, __LINE__);
    }
    e->kv4.work_bytes = want;
    return MOE_OK;
}

template <class C, typename T>
static int run_attn(moe_engine* e, AttnArgs a, int variant, int64_t units, int64_t q_rows, bool dependent) {
    a.run = 1;
    while (a.run < C::NB && a.cache.page_size / kKv4Block % (2 * a.run) == 0) a.run *= 2;
    auto* kernel = kv4_attn_kernel<C, T>;
    int& occ = e->kv4.occupancy[variant];
    if (occ == 0) {
        MOE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        int n = 0;
        MOE_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 128, C::SMEM));
        MOE_REQUIRE(n > 0, "kv4_attention: the kernel does not fit this device");
        occ = n;
    }
    unsigned int* err = e->dec_sync + 2;
    if constexpr (!C::SPLIT) {
        MOE_REQUIRE(units < 0x7FFFFFFF, "kv4_attention: too many rows for one call");
        MOE_CUDA(launch_kernel(false, kernel, dim3((unsigned)units), dim3(128), C::SMEM, e->stream, a, err));
        e->launches++;
        return MOE_OK;
    } else {
        // no more CTAs than tiles there can be
        const int64_t row_tiles = (q_rows + C::ROWS - 1) / C::ROWS;
        const int64_t most = units * ((a.seqs.max_seq_len + C::TILE - 1) / C::TILE + 1 + kUnitCost);
        int64_t grid = (int64_t)e->sm_count * occ;
        if (grid > most) grid = most;
        int rc = kv4_reserve(e, (size_t)grid * 2 * C::ROWS * (C::D + 2) * 4);
        if (rc) return rc;
        a.part = e->kv4.work;
        MOE_CUDA(launch_kernel(dependent, kernel, dim3((unsigned)grid), dim3(128), C::SMEM, e->stream, a, err));
        e->launches++;
        if (grid == 1 || a.whole) return MOE_OK;  // nothing can be split
        const int64_t all = (int64_t)a.seqs.n_seqs * a.cache.kv_heads * row_tiles;
        const bool by_border = all > grid - 1;
        const int64_t x = by_border ? grid - 1 : all;
        int parts = 1;  // two to eight partial results to a thread
        while (parts < 64 && all * parts * 4 <= grid) parts *= 2;
        MOE_CUDA(launch_kernel(true, kv4_attn_join_kernel<C, T>, dim3((unsigned)x, (unsigned)((C::ROWS * (C::D / 4) * parts + 255) / 256)), dim3(256), 0,
                               e->stream, a, (int)grid, (int)row_tiles, by_border ? 1 : 0, parts, err));
        e->launches++;
        return MOE_OK;
    }
}

// Rows of the tile: one column of eight where that holds a sequence's rows, two beyond (four columns share the work on a
// position among more rows, but their 255 registers leave two CTAs to an SM: 162 against 143 us on f32 prompts, 36 against
// 31 us on four-token verification).  f32 rows in units of their own (no splitting) once those fill the GPU four times over.
template <int D, typename T>
static int launch_rows(moe_engine* e, const AttnArgs& a, int64_t q_rows, bool dependent = false) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int V0 = (D == 64 ? 0 : D == 128 ? 8 : 16) + (F32 ? 4 : 0);
    const int64_t n = a.seqs.n_seqs;
    auto units = [&](int rows) {  // at most: whole tiles of all rows, and one that is not full for every sequence
        const int64_t per_seq = (q_rows + rows - 1) / rows;
        const int64_t all = (int64_t)a.seqs.n_tokens * a.group / rows + n;
        return (all < per_seq * n ? all : per_seq * n) * a.cache.kv_heads;
    };
    constexpr int TB = 4 / (D / 64);
    if constexpr (F32) {
        if (q_rows > 16 && units(16) >= 4 * e->sm_count) return run_attn<AttnCfg<D, F32, 2, 1, false>, T>(e, a, V0 + 2, units(16), q_rows, false);
    }
    if (q_rows > 8) return run_attn<AttnCfg<D, F32, 2, 1, true>, T>(e, a, V0 + 1, units(16), q_rows, dependent);
    return run_attn<AttnCfg<D, F32, 1, TB, true>, T>(e, a, V0, units(8), q_rows, dependent);
}

template <int D, typename T>
static int launch_attn(moe_engine* e, const AttnArgs& a) {
    if constexpr (sizeof(T) == 2) {
        if (kv4_prompt_fits<D>(e, a)) {
            AttnArgs few = a;
            const int rc = launch_kv4_prompt<D>(e, few);
            if (rc) return rc;
            const int64_t all_rows = (int64_t)a.seqs.max_q_len * a.group;
            few.hi_rows = 0;
            few.wide_too = 1;
            if (a.seqs.n_seqs == 1) {  // it is its, however many rows it has, or as a whole the other kernel's
                few.whole = 1;
                return launch_rows<D, T>(e, few, all_rows, true);
            }
            few.wide_too = 0;
            // the sequences of fewer rows (the host knows bounds only): single tokens in as small a tile as they need, then the others
            const int one = (a.group + 7) / 8 * 8;
            if (one < kPromptRows) {
                few.hi_rows = one + 1;
                const int rc1 = launch_rows<D, T>(e, few, one);
                if (rc1) return rc1;
                few.lo_rows = one + 1;
            }
            few.hi_rows = kPromptRows;
            few.wide_too = 1;
            return launch_rows<D, T>(e, few, all_rows);
        }
    }
    return launch_rows<D, T>(e, a, (int64_t)a.seqs.max_q_len * a.group);
}

}  // namespace moe

using namespace moe;

extern "C" int moe_kv4_attention_dev(moe_engine_t* e, const moe_kv4_cache_t* cache, const moe_kv4_batch_t* batch, const void* q_dev,
                                     int64_t q_token_stride, int64_t q_head_stride, const void* gate_dev, int64_t gate_token_stride,
                                     int64_t gate_head_stride, void* out_dev, int32_t dtype, int32_t num_heads, float scale, int32_t window) {
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
    const int64_t esize = dtype == MOE_DT_F32 ? 4 : 2, D = cache->head_dim, T = batch->n_tokens;
    auto extent = [&](int64_t ts, int64_t hs) { return ((T - 1) * ts + (num_heads - 1) * hs + D) * esize; };
    MOE_REQUIRE(!ranges_overlap(q_dev, extent(q_token_stride, q_head_stride), out_dev, T * num_heads * D * esize) &&
                    (!gate_dev || !ranges_overlap(gate_dev, extent(gate_token_stride, gate_head_stride), out_dev, T * num_heads * D * esize)),
                "kv4_attention: the output overlaps the queries or gates");
    MOE_REQUIRE(e, "kv4_attention: null engine");
    DeviceScope scope(e->device);
    MOE_CUDA(scope.status);
    cudaStreamCaptureStatus capture;
    MOE_CUDA(cudaStreamIsCapturing(e->stream, &capture));
    if (capture != cudaStreamCaptureStatusNone) {  // a graph would keep the address of a work area that moves when it grows
        set_error("kv4_attention: the engine's stream is being captured");
        return MOE_ERR_STATE;
    }
    AttnArgs a{};
    a.cache = kv4_view(cache);
    a.seqs = kv4_seqs(batch);
    a.q = q_dev; a.gate = gate_dev; a.out = out_dev;
    a.qt = q_token_stride; a.qh = q_head_stride; a.gt = gate_token_stride; a.gh = gate_head_stride;
    a.heads = num_heads;
    a.group = num_heads / cache->num_kv_heads;
    a.by_group = make_group_div((uint32_t)a.group);
    a.by_page = make_group_div((uint32_t)a.cache.page_size);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.window = window;
    a.hi_rows = 0x7FFFFFFF;
    const int vec = dtype == MOE_DT_F32 ? 4 : 8;
    a.vec_q = ((uintptr_t)q_dev & 15) == 0 && (q_token_stride | q_head_stride) % vec == 0;
    a.vec_gate = ((uintptr_t)gate_dev & 15) == 0 && (gate_token_stride | gate_head_stride) % vec == 0;
    const bool f32 = dtype == MOE_DT_F32;
    switch (cache->head_dim) {
        case 64: return f32 ? launch_attn<64, float>(e, a) : launch_attn<64, __nv_bfloat16>(e, a);
        case 128: return f32 ? launch_attn<128, float>(e, a) : launch_attn<128, __nv_bfloat16>(e, a);
        default: return f32 ? launch_attn<256, float>(e, a) : launch_attn<256, __nv_bfloat16>(e, a);
    }
}

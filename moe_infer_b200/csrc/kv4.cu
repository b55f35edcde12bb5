// Writing and reading back the paged 4-bit KV cache (page format: kv4.cuh).
//
// Append: key (rotated on the way) and value rows -> nibbles and (scale, bias) pairs, bit for bit the codec of pack.cu:
//   scale = (max - min) / 15, nibble = trunc((x - min) * (1 / scale) + 0.5), scale and bias = min stored in bf16
// (a group of equal values: scale 0).
// Memory bound (f32, head 256: 2 KB read, 288 B written per position and head).  A CTA takes 16 positions of a sequence (one
// block of the cache) and a head, so what it has to know first (sequence, page) is one chain of loads, and the rows are
// requested before the page is known.  A sub-warp of D / 8 lanes takes one quad (four positions that share words of V) of
// the keys or values; a lane holds eight elements of the four positions, so a group's minimum and maximum are three
// shuffles, the rotation partner is a second (cached) load or sits in the same lane, a lane's eight nibbles are one word of
// K, and the four positions' bytes of V meet in the lane that stores them.  8,192 f32 rows of two heads of 256 (38 MB): 16 us
// to store, 13 to read back; 14,000 bf16 rows of eight heads of 128 (73 MB): 25 and 16 us.
#include "kv4.cuh"

namespace moe {

struct Kv4AppendArgs {
    Kv4View cache;
    Kv4Seqs seqs;
    const void *k, *v;
    int64_t kt, kh, vt, vh;
    const float* table;        // null: no rotation
    int64_t n_positions;
    int rotary, interleaved;
    const int32_t* rope_positions;
    int vec_k, vec_v, vec_partner, vec_table;
};

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Quantises four positions' groups of 64, eight elements each in the lanes 8 k .. 8 k + 7: nibbles as one word per position,
// element i in bits 4 i.  Lane 8 k + i (and + 4) does the two divisions of position i and returns its (scale, bias) pair.
__device__ __forceinline__ uint32_t kv4_quant(const float (&x)[4][8], uint32_t (&word)[4]) {
    const int lane = threadIdx.x & 31;
    float mn[4], mx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        mn[i] = mx[i] = x[i][0];
#pragma unroll
        for (int k = 1; k < 8; ++k) {
            mn[i] = min_nan(mn[i], x[i][k]);
            mx[i] = max_nan(mx[i], x[i][k]);
        }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mn[i] = min_nan(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
            mx[i] = max_nan(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
        }
    const float lo = (lane & 2) ? ((lane & 1) ? mn[3] : mn[2]) : ((lane & 1) ? mn[1] : mn[0]);
    const float hi = (lane & 2) ? ((lane & 1) ? mx[3] : mx[2]) : ((lane & 1) ? mx[1] : mx[0]);
    // equal values: scale 0 (the packer's 1 / 15 stands for the same values, but would enter the attention's sums as s (15 - n))
    const bool flat = hi == lo;
    const float scale = flat ? 0.0f : __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    float inv = flat ? 0.0f : __fdiv_rn(1.0f, scale);
    uint32_t pair = (uint32_t)f32_to_bf16_ref(scale) | (uint32_t)f32_to_bf16_ref(lo) << 16;
    // not finite, or too large for its pair to be: both halves NaN (the attention kernel looks at the scale alone)
    if (!(fabsf(lo) < INFINITY && fabsf(scale) < INFINITY && (pair & 0x7F80u) != 0x7F80u && (pair & 0x7F800000u) != 0x7F800000u)) {
        pair = 0x7FC07FC0u;
        inv = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f = __shfl_sync(0xffffffffu, inv, (lane & 24) + i);
        word[i] = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float t = __fadd_rn(__fmul_rn(__fsub_rn(x[i][k], mn[i]), f), 0.5f);
            word[i] = min(__float2uint_rz(t), 15u) * (1u << (4 * k)) + word[i];
        }
    }
    return pair;
}

// bytes b of four words to word b of four: out[b] = byte b of in[0], in[1], in[2], in[3]
__device__ __forceinline__ void transpose_bytes(const uint32_t (&in)[4], uint32_t (&out)[4]) {
    const uint32_t a = __byte_perm(in[0], in[1], 0x5140), b = __byte_perm(in[2], in[3], 0x5140);
    const uint32_t c = __byte_perm(in[0], in[1], 0x7362), d = __byte_perm(in[2], in[3], 0x7362);
    out[0] = __byte_perm(a, b, 0x5410);
    out[1] = __byte_perm(a, b, 0x7632);
    out[2] = __byte_perm(c, d, 0x5410);
    out[3] = __byte_perm(c, d, 0x7632);
}

// Byte offset inside a block's K nibbles of the word that holds elements 8 l .. 8 l + 7 of position t.
template <int D>
__device__ __forceinline__ int kv4_k_offset(int l, int t) {
    constexpr int U = D >= 128 ? 2 : 1;
    const int g = l >> 3, c = (l >> 1) & 3, j = l & 1;
    return (g / U) * (512 * U) + ((t & 1) * 8 + (t >> 1)) * (32 * U) + c * (8 * U) + (g % U) * 8 + j * 4;
}

// Of a quad's rows row0 + i (positions q0 + i), those that exist (lo <= i < hi) and that the rotary table has a row for, as bits:
// the others are reported, their keys and values not stored.  at: their positions in the table.
__device__ __forceinline__ unsigned kv4_live(const Kv4AppendArgs& a, int64_t row0, int q0, int lo, int hi, int (&at)[4], unsigned int* err) {
    unsigned live = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        at[i] = 0;
        if (i < lo || i >= hi) continue;
        if (a.table) {
            at[i] = a.rope_positions ? a.rope_positions[row0 + i] : q0 + i;
            if (at[i] < 0 || at[i] >= a.n_positions) {
                atomicExch(err, kErrRopePos);
                continue;
            }
        }
        live |= 1u << i;
    }
    return live;
}

// Stores four positions' words and pairs; live: which of the four there are.
template <int D>
__device__ __forceinline__ void kv4_store(uint8_t* nib, bool is_v, int l, int t0, unsigned live, const uint32_t (&word)[4], uint32_t pair) {
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (live >> i & 1) *reinterpret_cast<uint32_t*>(nib + kv4_k_offset<D>(l, t0 + i)) = word[i];
    } else {
        // bytes of the four positions, elements (2x, 2x + 1): word x of the lane's 16
        uint8_t* dst = nib + (l >> 3) * 512 + (l & 7) * 64 + (t0 >> 2) * 16;
        uint32_t w[4];
        transpose_bytes(word, w);
        if (live == 15u) {
            *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int x4 = 0; x4 < 4; ++x4)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (live >> i & 1) dst[4 * x4 + i] = (uint8_t)(w[x4] >> (8 * i));
        }
    }
    const int mine = l & 7;
    if (mine < 4 && (live >> mine & 1)) *(reinterpret_cast<uint32_t*>(nib + 8 * D) + (l >> 3) * 16 + t0 + mine) = pair;
}

enum { kRotNone = 0, kRotHalf = 1, kRotInter = 2 };

// Rows readable 16 bytes at a time and a rotation of whole lanes (rotary a multiple of 16 in the half layout, 8 interleaved):
// a CTA walks `per` heads of its 16 positions, the next head's rows requested before this one's are worked on; in the
// interleaved layout a lane keeps the cosines and sines of its pairs for all of them.
template <typename T, int D, int kRot>
__global__ void __launch_bounds__(D, 512 / D) kv4_append_heads_kernel(Kv4AppendArgs a, int per, unsigned int* err) {
    constexpr int LPT = D / 8, W = sizeof(T) / 2;                    // 16-byte words of a lane's eight elements
    const int l = threadIdx.x % LPT, sub = threadIdx.x / LPT;        // eight sub-warps: four quads of keys, then of values
    const bool is_v = sub >= 4;
    const int b = blockIdx.z, h0 = blockIdx.x * per, h1 = min(h0 + per, a.cache.kv_heads);
    const Kv4Seq s = kv4_seq(a.seqs, b, err);
    const int first = max(s.len - s.q_len, 0);
    const int p0 = (first & ~15) + 16 * (int)blockIdx.y;
    if (p0 >= s.len || s.len <= first) return;
    const int q0 = p0 + 4 * (sub & 3), lo = max(first - q0, 0), hi = min(s.len - q0, 4);
    const int64_t ts = is_v ? a.vt : a.kt, hs = is_v ? a.vh : a.kh;
    const int64_t row0 = s.row0 + s.q_len - s.len + q0;              // row of the quad's first position (may lie before the rows)
    const T* src = (is_v ? (const T*)a.v : (const T*)a.k) + row0 * ts + h0 * hs + 8 * l;
    uint4 raw[4][W];
    auto load = [&](const T* p) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i >= lo && i < hi) {
#pragma unroll
                for (int w = 0; w < W; ++w) raw[i][w] = reinterpret_cast<const uint4*>(p + i * ts)[w];
            }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) raw[i][w] = make_uint4(0, 0, 0, 0);
    load(src);
    float cs[4][4], sn[4][4];  // interleaved: of the lane's four pairs
    const float* turn_at[4];   // half: where those of the lane's eight elements are
    const int half = a.rotary >> 1;
    const bool turns = kRot != kRotNone && !is_v && 8 * l < a.rotary, second = kRot == kRotHalf && 8 * l >= half;
    int at[4];
    const unsigned live = kv4_live(a, row0, q0, lo, hi, at, err), turned = turns ? live : 0;
    if (turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!(turned >> i & 1)) continue;
            turn_at[i] = a.table + (int64_t)at[i] * a.rotary + (kRot == kRotInter ? 4 * l : second ? 8 * l - half : 8 * l);
            if constexpr (kRot == kRotInter) {
                *reinterpret_cast<float4*>(cs[i]) = *reinterpret_cast<const float4*>(turn_at[i]);
                *reinterpret_cast<float4*>(sn[i]) = *reinterpret_cast<const float4*>(turn_at[i] + half);
            }
        }
    }
    uint8_t* blk = kv4_block(a.cache, a.seqs, b, h0, p0, kv4_block_bytes(D), err);
    const size_t head_bytes = (size_t)(a.cache.page_size / kKv4Block) * kv4_block_bytes(D);
    const int partner = (threadIdx.x & 31) + (second ? -(half >> 3) : half >> 3);  // the lane that holds the pairs' other elements
    for (int h = h0; h < h1; ++h) {
        float x[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[i][0]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (W == 2) x[i][k] = __uint_as_float(w[k]);
                else x[i][k] = __uint_as_float((k & 1) ? w[k >> 1] & 0xFFFF0000u : w[k >> 1] << 16);
            }
        }
        src += hs;
        if (h + 1 < h1) load(src);
        if constexpr (kRot == kRotHalf) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool on = turned >> i & 1;
                float c8[8], s8[8];
                if (on) {
                    ld_act8(turn_at[i], true, c8);
                    ld_act8(turn_at[i] + half, true, s8);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float o = __shfl_sync(0xffffffffu, x[i][k], partner & 31);
                    if (on)
                        x[i][k] = second ? __fadd_rn(__fmul_rn(o, s8[k]), __fmul_rn(x[i][k], c8[k]))
                                         : __fsub_rn(__fmul_rn(x[i][k], c8[k]), __fmul_rn(o, s8[k]));
                }
            }
        }
        if constexpr (kRot == kRotInter) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (turned >> i & 1) {
#pragma unroll
                    for (int k = 0; k < 8; k += 2) {
                        const float u = x[i][k], v = x[i][k + 1];
                        x[i][k] = __fsub_rn(__fmul_rn(u, cs[i][k >> 1]), __fmul_rn(v, sn[i][k >> 1]));
                        x[i][k + 1] = __fadd_rn(__fmul_rn(u, sn[i][k >> 1]), __fmul_rn(v, cs[i][k >> 1]));
                    }
                }
        }
        uint32_t word[4];
        const uint32_t pair = kv4_quant(x, word);
        if (blk && live) kv4_store<D>(blk + (h - h0) * head_bytes + (is_v ? 9 * D : 0), is_v, l, q0 % kKv4Block, live, word, pair);
    }
}

// One head to a CTA; any strides and alignment, any rotation.
template <typename T, int D>
__global__ void __launch_bounds__(D, 1024 / D) kv4_append_kernel(Kv4AppendArgs a, unsigned int* err) {
    constexpr int LPT = D / 8;
    const int l = threadIdx.x % LPT, sub = threadIdx.x / LPT;        // eight sub-warps: four quads of keys, then of values
    const bool is_v = sub >= 4;
    const int h = blockIdx.x, b = blockIdx.z;
    const Kv4Seq s = kv4_seq(a.seqs, b, err);
    const int first = max(s.len - s.q_len, 0);                       // first position this call writes
    const int p0 = (first & ~15) + 16 * (int)blockIdx.y;             // the CTA's positions
    if (p0 >= s.len || s.len <= first) return;
    const int q0 = p0 + 4 * (sub & 3);                               // this quad's first position
    const int row_of = s.row0 + s.q_len - s.len;                     // row = row_of + position
    const int lo = max(first - q0, 0), hi = min(s.len - q0, 4);
    uint8_t* const blk = kv4_block(a.cache, a.seqs, b, h, p0, kv4_block_bytes(D), err);

    int at[4];
    const unsigned live = kv4_live(a, (int64_t)row_of + q0, q0, lo, hi, at, err);
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = 0.0f;
        if (!(live >> i & 1)) continue;
        const int64_t row = row_of + (q0 + i);
        const T* src = is_v ? (const T*)a.v + row * a.vt + (int64_t)h * a.vh : (const T*)a.k + row * a.kt + (int64_t)h * a.kh;
        ld_act8(src + 8 * l, is_v ? a.vec_v : a.vec_k, x[i]);
        if (is_v || !a.table || 8 * l >= a.rotary) continue;
        const float* cs = a.table + (int64_t)at[i] * a.rotary;
        const int half = a.rotary >> 1;
        if (a.interleaved) {
            float ct[4], st[4];
            if (a.vec_table) {  // rotary a multiple of 8: the lane's four pairs are all there and contiguous
                *reinterpret_cast<float4*>(ct) = *reinterpret_cast<const float4*>(cs + 4 * l);
                *reinterpret_cast<float4*>(st) = *reinterpret_cast<const float4*>(cs + half + 4 * l);
            }
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const int p = (8 * l + k) >> 1;
                if (8 * l + k >= a.rotary) break;
                const float c = a.vec_table ? ct[k >> 1] : cs[p], sn = a.vec_table ? st[k >> 1] : cs[half + p], u = x[i][k], w = x[i][k + 1];
                x[i][k] = __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, sn));
                x[i][k + 1] = __fadd_rn(__fmul_rn(u, sn), __fmul_rn(w, c));
            }
        } else if (a.vec_partner) {  // half a multiple of 8: a lane's elements have one sign and their partners are contiguous
            const bool second = 8 * l >= half;
            float o[8], c[8], sn[8];
            ld_act8(src + (second ? 8 * l - half : 8 * l + half), true, o);
            const int p = second ? 8 * l - half : 8 * l;
            ld_act8(cs + p, true, c);
            ld_act8(cs + half + p, true, sn);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                x[i][k] = second ? __fadd_rn(__fmul_rn(o[k], sn[k]), __fmul_rn(x[i][k], c[k]))
                                 : __fsub_rn(__fmul_rn(x[i][k], c[k]), __fmul_rn(o[k], sn[k]));
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int d = 8 * l + k;
                if (d >= a.rotary) break;
                const bool second = d >= half;
                const int p = second ? d - half : d;
                const float o = ld_act(src + (second ? d - half : d + half)), c = cs[p], sn = cs[half + p];
                x[i][k] = second ? __fadd_rn(__fmul_rn(o, sn), __fmul_rn(x[i][k], c)) : __fsub_rn(__fmul_rn(x[i][k], c), __fmul_rn(o, sn));
            }
        }
    }
    uint32_t word[4];
    const uint32_t pair = kv4_quant(x, word);
    if (blk && live) kv4_store<D>(blk + (is_v ? 9 * D : 0), is_v, l, q0 % kKv4Block, live, word, pair);
}

// The way back: same mapping, values = nibble * scale + bias (the product is exact, so one rounding).
template <typename T, int D>
__global__ void __launch_bounds__(D) kv4_gather_kernel(Kv4View cache, Kv4Seqs seqs, T* k_out, T* v_out, int vec, unsigned int* err) {
    constexpr int LPT = D / 8;
    const int l = threadIdx.x % LPT, sub = threadIdx.x / LPT;
    const bool is_v = sub >= 4;
    const int h = blockIdx.x, b = blockIdx.z;
    const Kv4Seq s = kv4_seq(seqs, b, err);
    // positions of the rows, those without one (negative) among them: aligned to the block, also below zero
    const int first = s.len - s.q_len;
    const int q0 = (first & ~15) + 16 * (int)blockIdx.y + 4 * (sub & 3);
    if (q0 >= s.len || q0 + 3 < first) return;
    T* out = is_v ? v_out : k_out;
    const uint8_t* blk = q0 >= 0 ? kv4_block(cache, seqs, b, h, q0, kv4_block_bytes(D), err) : nullptr;
    uint32_t word[4] = {}, pair[4] = {};
    if (blk) {
        const int t0 = q0 % kKv4Block;
        const uint8_t* nib = blk + (is_v ? 9 * D : 0);
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) word[i] = *reinterpret_cast<const uint32_t*>(nib + kv4_k_offset<D>(l, t0 + i));
        } else {
            const uint4 q = *reinterpret_cast<const uint4*>(nib + (l >> 3) * 512 + (l & 7) * 64 + (t0 >> 2) * 16);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
            transpose_bytes(w, word);
        }
        const uint4 p = *reinterpret_cast<const uint4*>(nib + 8 * D + ((l >> 3) * 16 + t0) * 4);
        pair[0] = p.x; pair[1] = p.y; pair[2] = p.z; pair[3] = p.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = q0 + i;
        if (pos < first || pos >= s.len) continue;
        const float scale = __uint_as_float(pair[i] << 16), bias = __uint_as_float(pair[i] & 0xFFFF0000u);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf((float)(word[i] >> (4 * k) & 15u), scale, bias);
        const int64_t row = s.row0 + (pos - first);
        st_act8(out + (row * cache.kv_heads + h) * D + 8 * l, vec, v);
    }
}

int check_kv4(const moe_kv4_cache_t* c, const moe_kv4_batch_t* b) {
    MOE_REQUIRE(c && b, "kv4: null argument");
    MOE_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "kv4: head_dim (%d) must be 64, 128 or 256", c->head_dim);
    MOE_REQUIRE(c->page_size > 0 && c->page_size % kKv4Block == 0 && c->page_size <= 65536, "kv4: page_size (%d) must be a positive multiple of 16 up to 65536", c->page_size);
    MOE_REQUIRE(c->num_kv_heads > 0 && c->num_kv_heads <= 65536, "kv4: num_kv_heads (%d) must be positive", c->num_kv_heads);
    MOE_REQUIRE(c->num_pages >= 0 && c->num_pages <= 0x7FFFFFFF, "kv4: num_pages out of range");
    MOE_REQUIRE(c->pages || c->num_pages == 0, "kv4: null pages");
    MOE_REQUIRE(((uintptr_t)c->pages & 15) == 0, "kv4: pages must be 16-byte aligned");
    MOE_REQUIRE(b->n_seqs >= 0 && b->n_tokens >= 0 && b->max_pages >= 0 && b->max_seq_len >= 0 && b->max_q_len >= 0, "kv4: negative size in the batch");
    MOE_REQUIRE(b->max_seq_len <= 0x7FFF0000, "kv4: max_seq_len out of range");
    MOE_REQUIRE(b->n_seqs == 0 || (b->q_start && b->seq_lens), "kv4: null q_start or seq_lens");
    MOE_REQUIRE(b->n_seqs == 0 || b->max_pages == 0 || b->page_table, "kv4: null page_table");
    return MOE_OK;
}
Kv4View kv4_view(const moe_kv4_cache_t* c) { return Kv4View{(uint8_t*)c->pages, c->num_pages, c->page_size, c->num_kv_heads}; }
Kv4Seqs kv4_seqs(const moe_kv4_batch_t* b) {
    return Kv4Seqs{b->q_start, b->seq_lens, b->page_table, b->n_seqs, b->n_tokens, b->max_pages, b->max_seq_len, b->max_q_len};
}

// q rows touch at most this many blocks of 16 positions
static int64_t blocks_of(const moe_kv4_batch_t* b) {
    const int64_t q = b->max_q_len < b->n_tokens ? b->max_q_len : b->n_tokens;
    return (q + 14) / 16 + 1;
}

}  // namespace moe

using namespace moe;

extern "C" {

int moe_kv4_page_bytes(int32_t page_size, int32_t num_kv_heads, int32_t head_dim, int64_t* bytes) {
    MOE_REQUIRE(bytes, "kv4: null argument");
    const moe_kv4_cache_t c{nullptr, 0, page_size, num_kv_heads, head_dim};
    const moe_kv4_batch_t b{};
    int rc = check_kv4(&c, &b);
    if (rc) return rc;
    *bytes = (int64_t)(page_size / kKv4Block) * num_kv_heads * kv4_block_bytes(head_dim);
    return MOE_OK;
}

int moe_kv4_append_dev(moe_engine_t* e, const moe_kv4_cache_t* cache, const moe_kv4_batch_t* batch, const void* k_dev,
                       int64_t k_token_stride, int64_t k_head_stride, const void* v_dev, int64_t v_token_stride,
                       int64_t v_head_stride, int32_t dtype, const moe_rope_t* rope, const int32_t* rope_positions_dev) {
    int rc = check_kv4(cache, batch);
    if (rc) return rc;
    MOE_REQUIRE(dtype == MOE_DT_F32 || dtype == MOE_DT_BF16, "kv4_append: keys and values are f32 or bf16 (got dtype %d)", dtype);
    if (rope && (rc = check_rope(rope, cache->head_dim))) return rc;
    MOE_REQUIRE(rope || !rope_positions_dev, "kv4_append: rope positions without a rope table");
    if (batch->n_seqs == 0 || batch->n_tokens == 0 || batch->max_q_len == 0) return MOE_OK;
    MOE_REQUIRE(k_dev && v_dev, "kv4_append: null argument");
    const uintptr_t amask = dtype == MOE_DT_F32 ? 3 : 1;
    MOE_REQUIRE((((uintptr_t)k_dev | (uintptr_t)v_dev) & amask) == 0, "kv4_append: misaligned pointer");
    MOE_REQUIRE(k_token_stride >= 0 && k_head_stride >= 0 && v_token_stride >= 0 && v_head_stride >= 0, "kv4_append: negative stride");
    MOE_REQUIRE(e, "kv4_append: null engine");
    DeviceScope scope(e->device);
    MOE_CUDA(scope.status);
    const int vec = dtype == MOE_DT_F32 ? 4 : 8;
    Kv4AppendArgs a{};
    a.cache = kv4_view(cache);
    a.seqs = kv4_seqs(batch);
    a.k = k_dev; a.v = v_dev;
    a.kt = k_token_stride; a.kh = k_head_stride; a.vt = v_token_stride; a.vh = v_head_stride;
    if (rope) {
        a.table = rope->cos_sin;
        a.n_positions = rope->n_positions;
        a.rotary = rope->rotary_dim;
        a.interleaved = rope->interleaved;
    }
    a.rope_positions = rope_positions_dev;
    a.vec_k = ((uintptr_t)k_dev & 15) == 0 && (k_token_stride | k_head_stride) % vec == 0;
    a.vec_v = ((uintptr_t)v_dev & 15) == 0 && (v_token_stride | v_head_stride) % vec == 0;
    MOE_REQUIRE(blocks_of(batch) <= 65535 && batch->n_seqs <= 65535, "kv4_append: too many rows or sequences for one call");
    unsigned int* err = e->dec_sync + 2;
    const bool f32 = dtype == MOE_DT_F32;
    const int rot = !rope ? kRotNone : a.interleaved ? kRotInter : kRotHalf;
    a.vec_table = a.rotary % 8 == 0 && ((uintptr_t)a.table & 15) == 0;
    a.vec_partner = a.vec_k && a.rotary % 16 == 0 && a.vec_table;
    const bool whole = a.vec_k && a.vec_v && (!rope || (a.vec_table && a.rotary % (a.interleaved ? 8 : 16) == 0));
    // up to four heads to a CTA where that still leaves every SM four CTAs (14,000 bf16 rows of eight heads: 46 us with one head
    // each, 24 us with four; with few CTAs the one-head kernel's smaller register count is worth more: 8,192 f32 rows of two
    // heads, 16 us against 30)
    int per = 1;
    while (whole && per < 4 && per * 2 <= cache->num_kv_heads && blocks_of(batch) * batch->n_seqs * cache->num_kv_heads / (per * 2) >= 4 * e->sm_count) per *= 2;
    if (per > 1) {
        const dim3 grid((cache->num_kv_heads + per - 1) / per, (unsigned)blocks_of(batch), batch->n_seqs);
        auto run = [&](auto kernel) { kernel<<<grid, cache->head_dim, 0, e->stream>>>(a, per, err); };
        auto by_rot = [&](auto none, auto half, auto inter) { rot == kRotNone ? run(none) : rot == kRotHalf ? run(half) : run(inter); };
#define KV4_HEADS(T, D) by_rot(kv4_append_heads_kernel<T, D, kRotNone>, kv4_append_heads_kernel<T, D, kRotHalf>, kv4_append_heads_kernel<T, D, kRotInter>)
        switch (cache->head_dim) {
            case 64: f32 ? KV4_HEADS(float, 64) : KV4_HEADS(__nv_bfloat16, 64); break;
            case 128: f32 ? KV4_HEADS(float, 128) : KV4_HEADS(__nv_bfloat16, 128); break;
            default: f32 ? KV4_HEADS(float, 256) : KV4_HEADS(__nv_bfloat16, 256); break;
        }
#undef KV4_HEADS
    } else {
        const dim3 grid(cache->num_kv_heads, (unsigned)blocks_of(batch), batch->n_seqs);
        auto run = [&](auto kernel) { kernel<<<grid, cache->head_dim, 0, e->stream>>>(a, err); };
        switch (cache->head_dim) {
            case 64: f32 ? run(kv4_append_kernel<float, 64>) : run(kv4_append_kernel<__nv_bfloat16, 64>); break;
            case 128: f32 ? run(kv4_append_kernel<float, 128>) : run(kv4_append_kernel<__nv_bfloat16, 128>); break;
            default: f32 ? run(kv4_append_kernel<float, 256>) : run(kv4_append_kernel<__nv_bfloat16, 256>); break;
        }
    }
    e->launches++;
    MOE_CUDA(cudaGetLastError());
    return MOE_OK;
}

int moe_kv4_gather_dev(moe_engine_t* e, const moe_kv4_cache_t* cache, const moe_kv4_batch_t* batch, void* k_out_dev, void* v_out_dev,
                       int32_t dtype) {
    int rc = check_kv4(cache, batch);
    if (rc) return rc;
    MOE_REQUIRE(dtype == MOE_DT_F32 || dtype == MOE_DT_BF16, "kv4_gather: outputs are f32 or bf16 (got dtype %d)", dtype);
    if (batch->n_seqs == 0 || batch->n_tokens == 0 || batch->max_q_len == 0) return MOE_OK;
    MOE_REQUIRE(k_out_dev && v_out_dev, "kv4_gather: null argument");
    const uintptr_t amask = dtype == MOE_DT_F32 ? 3 : 1;
    MOE_REQUIRE((((uintptr_t)k_out_dev | (uintptr_t)v_out_dev) & amask) == 0, "kv4_gather: misaligned pointer");
    MOE_REQUIRE(k_out_dev != v_out_dev && !ranges_overlap(k_out_dev, (int64_t)batch->n_tokens * cache->num_kv_heads * cache->head_dim * (dtype == MOE_DT_F32 ? 4 : 2), v_out_dev,
                                                          (int64_t)batch->n_tokens * cache->num_kv_heads * cache->head_dim * (dtype == MOE_DT_F32 ? 4 : 2)),
                "kv4_gather: the outputs overlap");
    MOE_REQUIRE(e, "kv4_gather: null engine");
    DeviceScope scope(e->device);
    MOE_CUDA(scope.status);
    MOE_REQUIRE(blocks_of(batch) <= 65535 && batch->n_seqs <= 65535, "kv4_gather: too many rows or sequences for one call");
    const dim3 grid(cache->num_kv_heads, (unsigned)blocks_of(batch), batch->n_seqs);
    const int vec = (((uintptr_t)k_out_dev | (uintptr_t)v_out_dev) & 15) == 0;
    unsigned int* err = e->dec_sync + 2;
    auto run = [&](auto kernel, auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        kernel<<<grid, cache->head_dim, 0, e->stream>>>(kv4_view(cache), kv4_seqs(batch), (T*)k_out_dev, (T*)v_out_dev, vec, err);
    };
    const bool f32 = dtype == MOE_DT_F32;
    float* f = nullptr;
    __nv_bfloat16* h = nullptr;
    switch (cache->head_dim) {
        case 64: f32 ? run(kv4_gather_kernel<float, 64>, f) : run(kv4_gather_kernel<__nv_bfloat16, 64>, h); break;
        case 128: f32 ? run(kv4_gather_kernel<float, 128>, f) : run(kv4_gather_kernel<__nv_bfloat16, 128>, h); break;
        default: f32 ? run(kv4_gather_kernel<float, 256>, f) : run(kv4_gather_kernel<__nv_bfloat16, 256>, h); break;
    }
    e->launches++;
    MOE_CUDA(cudaGetLastError());
    return MOE_OK;
}

}  // extern "C"

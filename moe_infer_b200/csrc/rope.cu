// Rotary positions: table of cosines and sines (host) and the rotation of query or key heads (device).
//
// For pair i < r / 2 of a head's first r elements, (a, b) = (x[i], x[i + r/2]) in the half layout or (x[2i], x[2i+1]) in
// the interleaved one:  a' = a cos - b sin,  b' = a sin + b cos, each product and sum rounded on its own (the append
// kernel's 4-bit rounding depends on these values: a contracted multiply-add would make it depend on the compiler);
// elements from r on are copied.  Angles reach 10^5 radians and more, where f32 has lost the fraction of a turn: they are
// formed in 64 bits on the host, once, and the kernels read f32 cosines and sines.
//
// Memory bound: 16,384 tokens of 32 bf16 heads of 128 in 44.8 us, 6.2 TB/s (96 % of a copy).
#include <math.h>

#include "kv4.cuh"

namespace moe {

struct RopeArgs {
    const float* table;
    int64_t n_positions;
    int rotary, heads, dim;
    int64_t n_tokens;
    int64_t xt, xh, ot, oh;  // element strides
    const int32_t* positions;
};

// One thread per unit of V elements pairs (or copied elements) and kHeads heads; units of one token are neighbours.
// V = 16 bytes' worth where pointers, strides and sizes allow it, otherwise one pair or element at a time.
template <typename T, int V, bool kInter, int kHeads>
__global__ void __launch_bounds__(256) rope_kernel(const T* x, T* out, RopeArgs a, unsigned int* err) {
    const int pair_units = kInter ? (V > 1 ? a.rotary / V : a.rotary / 2) : a.rotary / 2 / V;
    const int units = pair_units + (a.dim - a.rotary) / V;
    const int groups = (a.heads + kHeads - 1) / kHeads;
    const uint32_t per_token = (uint32_t)units * groups;
    const uint64_t idx = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= (uint64_t)a.n_tokens * per_token) return;
    const int64_t t = idx < 0xFFFFFFFFull ? (int64_t)((uint32_t)idx / per_token) : (int64_t)(idx / per_token);
    const uint32_t rem = (uint32_t)(idx - (uint64_t)t * per_token);
    const int hg = rem / units, u = rem - hg * units;
    const T* xr = x + t * a.xt + (int64_t)hg * kHeads * a.xh;
    T* orow = out + t * a.ot + (int64_t)hg * kHeads * a.oh;
    const int n_here = min(kHeads, a.heads - hg * kHeads);

    if (u >= pair_units) {  // elements behind the rotated part
        const int e = a.rotary + (u - pair_units) * V;
        if constexpr (V > 1) {
            uint4 v[kHeads];
#pragma unroll
            for (int h = 0; h < kHeads; ++h)
                if (h < n_here) v[h] = *reinterpret_cast<const uint4*>(xr + h * a.xh + e);
#pragma unroll
            for (int h = 0; h < kHeads; ++h)
                if (h < n_here) *reinterpret_cast<uint4*>(orow + h * a.oh + e) = v[h];
        } else {
            for (int h = 0; h < n_here; ++h) orow[h * a.oh + e] = xr[h * a.xh + e];
        }
        return;
    }
    const int64_t pos = a.positions[t];
    if (pos < 0 || pos >= a.n_positions) {  // reported; the row is left as it is
        if (u == 0 && hg == 0) atomicExch(err, kErrRopePos);
        return;
    }
    const float* cs = a.table + pos * a.rotary;
    const float* sn = cs + a.rotary / 2;
    if constexpr (V == 1) {
        const int ia = kInter ? 2 * u : u, ib = kInter ? 2 * u + 1 : u + a.rotary / 2;
        const float c = cs[u], s = sn[u];
        for (int h = 0; h < n_here; ++h) {
            const float p = ld_act(xr + h * a.xh + ia), q = ld_act(xr + h * a.xh + ib);
            st_act(orow + h * a.oh + ia, __fsub_rn(__fmul_rn(p, c), __fmul_rn(q, s)));
            st_act(orow + h * a.oh + ib, __fadd_rn(__fmul_rn(p, s), __fmul_rn(q, c)));
        }
    } else {
        constexpr int P = kInter ? V / 2 : V;  // pairs of a unit
        float c[P], s[P];
        if constexpr (P % 4 == 0) {
#pragma unroll
            for (int i = 0; i < P; i += 4) {
                *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(cs + u * P + i);
                *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(sn + u * P + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < P; i += 2) {
                *reinterpret_cast<float2*>(c + i) = *reinterpret_cast<const float2*>(cs + u * P + i);
                *reinterpret_cast<float2*>(s + i) = *reinterpret_cast<const float2*>(sn + u * P + i);
            }
        }
        constexpr int L = kInter ? 1 : 2;  // 16-byte words of a unit
        const int e0 = u * V, e1 = e0 + a.rotary / 2;
        uint4 raw[kHeads][L];
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
            if (h < n_here) {
                raw[h][0] = *reinterpret_cast<const uint4*>(xr + h * a.xh + e0);
                if (!kInter) raw[h][L - 1] = *reinterpret_cast<const uint4*>(xr + h * a.xh + e1);
            }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            if (h >= n_here) continue;
            float v[L * V];
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const uint32_t w[4] = {raw[h][l].x, raw[h][l].y, raw[h][l].z, raw[h][l].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (V == 4) {
                        v[l * V + i] = __uint_as_float(w[i]);
                    } else {
                        v[l * V + 2 * i] = __uint_as_float(w[i] << 16);
                        v[l * V + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < P; ++i) {
                float& p = v[kInter ? 2 * i : i];
                float& q = v[kInter ? 2 * i + 1 : V + i];
                const float np = __fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i]));
                q = __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i]));
                p = np;
            }
#pragma unroll
            for (int l = 0; l < L; ++l) {
                uint4 o;
                if constexpr (V == 4) {
                    o = make_uint4(__float_as_uint(v[l * V]), __float_as_uint(v[l * V + 1]), __float_as_uint(v[l * V + 2]), __float_as_uint(v[l * V + 3]));
                } else {
                    o = make_uint4(pack_bf16(v[l * V], v[l * V + 1]), pack_bf16(v[l * V + 2], v[l * V + 3]),
                                   pack_bf16(v[l * V + 4], v[l * V + 5]), pack_bf16(v[l * V + 6], v[l * V + 7]));
                }
                *reinterpret_cast<uint4*>(orow + h * a.oh + (l == 0 ? e0 : e1)) = o;
            }
        }
    }
}

template <typename T, int V, bool kInter, int kHeads>
static int run_rope(moe_engine* e, const T* x, T* out, const RopeArgs& a) {
    const int pair_units = kInter ? (V > 1 ? a.rotary / V : a.rotary / 2) : a.rotary / 2 / V;
    const uint64_t per_token = (uint64_t)(pair_units + (a.dim - a.rotary) / V) * ((a.heads + kHeads - 1) / kHeads);
    const uint64_t blocks = ((uint64_t)a.n_tokens * per_token + 255) / 256;
    MOE_REQUIRE(per_token < (1ull << 31) && blocks < (1ull << 31), "rope: too many elements for one call");
    rope_kernel<T, V, kInter, kHeads><<<(unsigned)blocks, 256, 0, e->stream>>>(x, out, a, e->dec_sync + 2);
    e->launches++;
    MOE_CUDA(cudaGetLastError());
    return MOE_OK;
}

template <typename T>
static int launch_rope(moe_engine* e, const void* x, void* out, const RopeArgs& a, bool interleaved) {
    constexpr int V = 16 / (int)sizeof(T);
    const T* xs = (const T*)x;
    T* os = (T*)out;
    const bool vec = (((uintptr_t)x | (uintptr_t)out) & 15) == 0 && ((a.xt | a.xh | a.ot | a.oh) % V) == 0 && a.dim % V == 0 &&
                     (interleaved ? a.rotary % (2 * V) : a.rotary / 2 % V) == 0 && ((uintptr_t)a.table & 15) == 0 && a.rotary % 8 == 0;
    if (!vec) return interleaved ? run_rope<T, 1, true, 1>(e, xs, os, a) : run_rope<T, 1, false, 1>(e, xs, os, a);
    // four heads share a thread's cosines and keep four loads in flight once there are enough threads without that
    const bool many = (int64_t)a.n_tokens * a.heads * (a.dim / V) >= (int64_t)e->sm_count * 2048 * 4;
    if (interleaved) return many ? run_rope<T, V, true, 4>(e, xs, os, a) : run_rope<T, V, true, 1>(e, xs, os, a);
    return many ? run_rope<T, V, false, 4>(e, xs, os, a) : run_rope<T, V, false, 1>(e, xs, os, a);
}

int check_rope(const moe_rope_t* r, int32_t head_dim) {
    MOE_REQUIRE(r && r->cos_sin, "rope: null table");
    MOE_REQUIRE(r->rotary_dim > 0 && r->rotary_dim % 2 == 0 && r->rotary_dim <= head_dim,
                "rope: rotary_dim (%d) must be even, positive and at most head_dim (%d)", r->rotary_dim, head_dim);
    MOE_REQUIRE(r->n_positions > 0, "rope: the table has no positions");
    MOE_REQUIRE(((uintptr_t)r->cos_sin & 3) == 0, "rope: the table must be 4-byte aligned");
    return MOE_OK;
}

}  // namespace moe

using namespace moe;

extern "C" {

int moe_rope_table_host(const moe_rope_params_t* p, int64_t first_position, int64_t n_positions, float* cos_sin_host) {
    MOE_REQUIRE(p && cos_sin_host, "rope_table: null argument");
    MOE_REQUIRE(p->rotary_dim > 0 && p->rotary_dim % 2 == 0 && p->rotary_dim <= 65536, "rope_table: rotary_dim (%d) must be even and positive", p->rotary_dim);
    MOE_REQUIRE(p->theta > 1.0 && isfinite(p->theta), "rope_table: theta must be above 1");
    MOE_REQUIRE(first_position >= 0 && n_positions >= 0, "rope_table: negative position");
    MOE_REQUIRE(p->scaling >= MOE_ROPE_PLAIN && p->scaling <= MOE_ROPE_YARN, "rope_table: unknown scaling %d", p->scaling);
    const bool scaled = p->scaling != MOE_ROPE_PLAIN;
    MOE_REQUIRE(!scaled || (p->factor >= 1.0 && isfinite(p->factor)), "rope_table: a scaled table needs a factor of 1 or more");
    MOE_REQUIRE(p->scaling != MOE_ROPE_NTK || p->rotary_dim > 2, "rope_table: ntk scaling needs a rotary_dim above 2");
    MOE_REQUIRE(p->scaling != MOE_ROPE_YARN || (p->original_positions > 0 && p->beta_fast > p->beta_slow && p->beta_slow > 0.0),
                "rope_table: yarn scaling needs original_positions > 0 and beta_fast > beta_slow > 0");
    const int half = p->rotary_dim / 2;
    const double r = p->rotary_dim;
    double theta = p->theta, mul = 1.0;
    if (p->scaling == MOE_ROPE_NTK) theta *= pow(p->factor, r / (r - 2.0));
    double low = 0.0, high = 0.0;
    if (p->scaling == MOE_ROPE_YARN) {
        // the pair index whose wavelength makes `turns` full turns over the original context
        auto at = [&](double turns) { return r * log((double)p->original_positions / (turns * 2.0 * M_PI)) / (2.0 * log(theta)); };
        low = fmax(floor(at(p->beta_fast)), 0.0);
        high = fmin(ceil(at(p->beta_slow)), r - 1.0);
        mul = 0.1 * log(p->factor) + 1.0;
    }
    for (int i = 0; i < half; ++i) {
        double freq = pow(theta, -2.0 * i / r);
        if (p->scaling == MOE_ROPE_LINEAR) freq /= p->factor;
        if (p->scaling == MOE_ROPE_YARN) {
            const double ramp = fmin(fmax((i - low) / fmax(high - low, 1e-3), 0.0), 1.0);
            freq = freq / p->factor * ramp + freq * (1.0 - ramp);
        }
        for (int64_t k = 0; k < n_positions; ++k) {
            const double ang = (double)(first_position + k) * freq;
            cos_sin_host[k * p->rotary_dim + i] = (float)(cos(ang) * mul);
            cos_sin_host[k * p->rotary_dim + half + i] = (float)(sin(ang) * mul);
        }
    }
    return MOE_OK;
}

int moe_rope_dev(moe_engine_t* e, const moe_rope_t* rope, const void* x_dev, int64_t x_token_stride, int64_t x_head_stride,
                 void* out_dev, int64_t out_token_stride, int64_t out_head_stride, int32_t dtype, int64_t n_tokens, int32_t num_heads,
                 int32_t head_dim, const int32_t* positions_dev) {
    MOE_REQUIRE(n_tokens >= 0 && num_heads > 0 && head_dim > 0, "rope: bad shape [%lld, %d, %d]", (long long)n_tokens, num_heads, head_dim);
    int rc = check_rope(rope, head_dim);
    if (rc) return rc;
    MOE_REQUIRE(dtype == MOE_DT_F32 || dtype == MOE_DT_BF16, "rope: activations are f32 or bf16 (got dtype %d)", dtype);
    if (n_tokens == 0) return MOE_OK;
    MOE_REQUIRE(x_dev && out_dev && positions_dev, "rope: null argument");
    const uintptr_t mask = dtype == MOE_DT_F32 ? 3 : 1;
    MOE_REQUIRE((((uintptr_t)x_dev | (uintptr_t)out_dev) & mask) == 0, "rope: misaligned pointer");
    MOE_REQUIRE(x_head_stride >= 0 && x_token_stride >= 0, "rope: negative stride");
    MOE_REQUIRE(rows_disjoint(n_tokens, out_token_stride, num_heads, out_head_stride, head_dim), "rope: output rows overlap");
    MOE_REQUIRE(x_dev != out_dev || (x_token_stride == out_token_stride && x_head_stride == out_head_stride),
                "rope: in place needs equal strides");
    const int64_t esize = dtype == MOE_DT_F32 ? 4 : 2;
    auto extent = [&](int64_t ts, int64_t hs) { return ((n_tokens - 1) * ts + (num_heads - 1) * hs + head_dim) * esize; };
    MOE_REQUIRE(x_dev == out_dev || !ranges_overlap(x_dev, extent(x_token_stride, x_head_stride), out_dev, extent(out_token_stride, out_head_stride)),
                "rope: input and output overlap without being the same");
    MOE_REQUIRE(e, "rope: null engine");
    DeviceScope scope(e->device);
    MOE_CUDA(scope.status);
    RopeArgs a{rope->cos_sin, rope->n_positions, rope->rotary_dim, num_heads, head_dim, n_tokens, x_token_stride, x_head_stride,
               out_token_stride, out_head_stride, positions_dev};
    return dtype == MOE_DT_F32 ? launch_rope<float>(e, x_dev, out_dev, a, rope->interleaved != 0)
                               : launch_rope<__nv_bfloat16>(e, x_dev, out_dev, a, rope->interleaved != 0);
}

}  // extern "C"

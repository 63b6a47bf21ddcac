// AdamW over many tensors in one launch, with states in 32 or in 8 bits, and clipping by the global gradient norm (gfx950).
//
//   c = min(1, max_norm / (|g| + 1e-6)) over all gradients, g' = c g
//   m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g' g'
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// 8-bit states: 256 consecutive elements share a power of two 2^k.  m is e4m3 (OCP, largest 448), v is e5m3 without a sign (the upper
// byte but one of a positive half: largest 61440), both times 2^k, k >= -126 the smallest with which the block's largest magnitude,
// rounded to four significant bits, fits.  Rounded to nearest, ties to even; relative half step 2^-4, for sqrt(v) 2^-5.  With a power
// of two as the scale, dequantising is exact and the rounding of a value in the normal range does not depend on its block.  v' > 0
// that would round to 0 takes the smallest code: no step is divided by eps alone because of the format.  A value that is not finite
// keeps a code of its own (NaN; infinity for v) and no part in its block's scale.
// The moments are formed in 64 bits where they are rounded to 8: which of two codes a value next to their border takes is then a
// matter of the definition and not of f32 rounding (f64 products run at the f32 rate here, and the kernel waits for memory).  Each
// product and sum is rounded by itself, in the order written above, so that the rare exact border falls the same way everywhere.
// The step itself uses the unrounded moments in f32.
#include "common.h"

namespace {

constexpr int kChunk = 4096;        // elements a block of the update takes: 4 waves x 4 blocks of 256
constexpr int kBlock = 256;         // elements that share a scale

typedef float f32x4_a4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a2_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_a1_t __attribute__((aligned(1)));

// four consecutive elements from i on (`left` of them exist), f32 or bf16 at an element-aligned address
__device__ __forceinline__ void load4(const void* base, long i, long left, bool bf16, float* f) {
    if (left >= 4) {
        if (bf16) {
            const u32x2_a2_t u = *(const u32x2_a2_t*)((const uint16_t*)base + i);
            f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
            f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
        } else {
            const f32x4_a4_t u = *(const f32x4_a4_t*)((const float*)base + i);
            f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = e < left ? (bf16 ? BF16::ld(base, i + e) : F32::ld(base, i + e)) : 0.f;
    }
}
__device__ __forceinline__ void store4(void* base, long i, long left, bool bf16, const float* f) {
    if (left >= 4) {
        if (bf16) *(u32x2_a2_t*)((uint16_t*)base + i) = (u32x2_a2_t){pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
        else *(f32x4_a4_t*)((float*)base + i) = (f32x4_a4_t){f[0], f[1], f[2], f[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) { if (bf16) BF16::st(base, i + e, f[e]); else F32::st(base, i + e, f[e]); }
    }
}
// four codes; the code arrays are padded to whole blocks of 256, so a word is always there
__device__ __forceinline__ uint32_t load_codes(const void* base, long i) { return ((const uint32_t*)base)[i >> 2]; }

// ---- the 8-bit forms ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void decode_m(uint32_t c, float scale, float* f) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    f[0] = lo[0] * scale; f[1] = lo[1] * scale; f[2] = hi[0] * scale; f[3] = hi[1] * scale;
}
__device__ __forceinline__ void decode_v(uint32_t c, float scale, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint16_t h = (uint16_t)(((c >> (8 * e)) & 0xffu) << 7);
        f[e] = (float)__builtin_bit_cast(_Float16, h) * scale;
    }
}
// |x| rounded to four significant bits, as (biased exponent of a double) << 3 | mantissa: whole numbers in the order of the magnitudes
__device__ __forceinline__ uint32_t four_bits(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)u, hi = ((uint32_t)(u >> 32) & 0x7fffffffu) | (lo < 1u ? lo : 1u);     // what lies below decides ties
    return (hi + 0xffffu + ((hi >> 17) & 1u)) >> 17;
}
constexpr uint32_t kOver = (1023 + 128) << 3;       // 2^128 and above, infinities, NaN

// whole multiples of 2^(k - s) nearest to |x| (at most a few: what lies below the normal numbers)
__device__ __forceinline__ uint32_t multiples(double x, int sk) {
    const double t = __builtin_fabs(x) * __builtin_bit_cast(double, (uint64_t)(uint32_t)(1023 + sk) << 52);
    return (uint32_t)__builtin_bit_cast(uint64_t, t + 4503599627370496.0);
}
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
#define M_(C) { const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, C, 0xf, 0xf, true); v = v > o ? v : o; }
    M_(0xB1) M_(0x4E) M_(0x141) M_(0x140)
#undef M_
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = r[0] > r[1] ? r[0] : r[1];
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return r[0] > r[1] ? r[0] : r[1];
}
// One block of 256 values, four to a lane -> codes and the block's scale.  SIGNED: e4m3, else e5m3.
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(const double* x, float& scale) {
    constexpr int kBias = SIGNED ? 7 : 15, kTop = SIGNED ? 8 : 15;       // exponent bias, exponent of the largest number
    uint32_t q[4], top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        q[e] = four_bits(x[e]);
        const uint32_t t = q[e] < kOver ? q[e] : 0u;
        top = top > t ? top : t;
    }
    top = max_dpp(top);
    // e4m3 ends at 1.75 x 2^8: 1.875 x 2^n takes the next k
    int k = (int)((SIGNED ? top + 1 : top) >> 3) - 1023 - kTop;
    k = k > -126 ? k : -126;
    scale = __uint_as_float((uint32_t)(k + 127) << 23);
    uint32_t out = 0;
    const int shift = (1023 + k - kBias) << 3;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        int c = (int)q[e] - shift;
        if (c < 8) {                                                       // below the normal numbers
            c = (int)multiples(x[e], kBias + 2 - k);
            if (!SIGNED && c == 0 && x[e] > 0.0) c = 1;
        }
        if (q[e] >= kOver) c = SIGNED ? 0x7f : (x[e] != x[e] ? 0xff : 0xf8);
        if (SIGNED) c |= (int)((__builtin_bit_cast(uint64_t, x[e]) >> 56) & 0x80u);
        out |= (uint32_t)c << (8 * e);
    }
    return out;
}

// rows, kRow doubles per group: {lr, 1 - b1^t, 1 - b2^t, t, b1, b2, eps, weight decay} and, formed with the step count, what the update
// takes: {1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - b1, 1 - b2}; behind the groups {max_norm, c}
constexpr int kRow = BTS_ADAMW_ROW;

__global__ __launch_bounds__(256) void adamw_multi_kernel(const bts_adamw_tensor_t* __restrict__ tensors, const int2* __restrict__ chunks, long n_chunks,
                                                         const double* __restrict__ rows, int n_groups) {
    // last chunk first: behind a norm pass the gradients that were read last are the ones that the cache still holds
    const int2 ch = chunks[n_chunks - 1 - blockIdx.x];
    const bts_adamw_tensor_t t = tensors[ch.x];
    const double* r = rows + kRow * t.group;
    const double clip = rows[kRow * n_groups + 1], b1 = r[4], b2 = r[5], a1 = r[11], a2 = r[12];
    const float decay = (float)r[8], step = (float)r[9], rs = (float)r[10], eps = (float)r[6];
    const bool bf16 = t.flags & BTS_ADAMW_BF16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long base = (long)ch.y * kChunk;
#pragma unroll 1
    for (int it = 0; it < 4; ++it) {
        const long b0 = base + (it * 4 + wave) * kBlock, i = b0 + lane * 4, left = t.n - i;
        if (b0 >= t.n) break;
        float p[4], g[4];
        load4(t.p, i, left, bf16, p);
        load4(t.g, i, left, bf16, g);
        float m32[4], v32[4];
        if (t.flags & BTS_ADAMW_8BIT) {
            float mo[4], vo[4], sm, sv;
            decode_m(load_codes(t.m, i), t.m_scale[b0 / kBlock], mo);
            decode_v(load_codes(t.v, i), t.v_scale[b0 / kBlock], vo);
            double m[4], v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double gd = (double)g[e] * clip;
                m[e] = b1 * (double)mo[e] + a1 * gd;                 // every product and sum rounded, in this order: with gradients of
                v[e] = b2 * (double)vo[e] + a2 * gd * gd;            // few bits (bf16, zeros) one value in a thousand IS a border
                if (e >= left) m[e] = v[e] = 0.0;
                m32[e] = (float)m[e];
                v32[e] = (float)v[e];
            }
            ((uint32_t*)t.m)[i >> 2] = encode<true>(m, sm);
            ((uint32_t*)t.v)[i >> 2] = encode<false>(v, sv);
            if (lane == 0) {
                t.m_scale[b0 / kBlock] = sm;
                t.v_scale[b0 / kBlock] = sv;
            }
        } else {
            load4(t.m, i, left, false, m32);
            load4(t.v, i, left, false, v32);
            const float b1f = (float)b1, b2f = (float)b2, a1f = (float)a1, a2f = (float)a2, c = (float)clip;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float gc = g[e] * c;
                m32[e] = b1f * m32[e] + a1f * gc;
                v32[e] = b2f * v32[e] + a2f * gc * gc;
            }
            store4(t.m, i, left, false, m32);
            store4(t.v, i, left, false, v32);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = p[e] * decay - step * (m32[e] / (sqrtf(v32[e]) * rs + eps));
        store4(t.p, i, left, bf16, p);                                 // bf16 parameters: the one rounding to fewer bits, to nearest even
    }
}

// sum of squares of every gradient, in f64 (no overflow of g^2, no loss over 10^8 terms): one partial sum per block, fixed order
__global__ __launch_bounds__(256) void adamw_norm_kernel(const bts_adamw_tensor_t* __restrict__ tensors, const int2* __restrict__ chunks, long n_chunks,
                                                        double* __restrict__ partials) {
    double s = 0.0;
    for (long c = blockIdx.x; c < n_chunks; c += gridDim.x) {
        const int2 ch = chunks[c];
        const bts_adamw_tensor_t t = tensors[ch.x];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const long i = (long)ch.y * kChunk + it * 1024 + threadIdx.x * 4, left = t.n - i;
            if (left <= 0) break;
            float g[4];
            load4(t.g, i, left, t.flags & BTS_ADAMW_BF16, g);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fma((double)g[e], (double)g[e], s);
        }
    }
    __shared__ double red[4];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partials[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

struct HostHyper {
    double v[BTS_ADAMW_MAX_GROUPS][5];
    double max_norm;
};

// one block: hyper-parameters from the host (if given), step count and bias corrections, norm and clip coefficient
__global__ __launch_bounds__(1024) void adamw_begin_kernel(double* __restrict__ rows, int n_groups, HostHyper hh, int set, int advance,
                                                          const double* __restrict__ partials, int n_partials, float* __restrict__ grad_norm) {
    const int g = threadIdx.x;
    if (g < n_groups) {
        double* r = rows + kRow * g;
        if (set) {
            r[0] = hh.v[g][0]; r[4] = hh.v[g][1]; r[5] = hh.v[g][2]; r[6] = hh.v[g][3]; r[7] = hh.v[g][4];
        }
        if (advance) {
            const double t = r[3] + 1.0;
            r[3] = t;
            r[1] = 1.0 - pow(r[4], t);
            r[2] = 1.0 - pow(r[5], t);
            r[8] = 1.0 - r[0] * r[7];
            r[9] = r[0] / r[1];
            r[10] = 1.0 / sqrt(r[2]);
            r[11] = 1.0 - r[4];
            r[12] = 1.0 - r[5];
        }
    }
    double s = 0.0;
    for (int i = threadIdx.x; i < n_partials; i += 1024) s += partials[i];
    __shared__ double red[16];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double* tail = rows + kRow * n_groups;
        if (set) tail[0] = hh.max_norm;
        double c = 1.0;
        if (partials) {
            double t = 0.0;
#pragma unroll
            for (int i = 0; i < 16; ++i) t += red[i];
            t = sqrt(t);
            *grad_norm = (float)t;
            c = (set ? hh.max_norm : tail[0]) / (t + 1e-6);
            c = c > 1.0 ? 1.0 : c;                                  // a norm that is NaN makes c NaN, and with it every parameter
        }
        if (advance) tail[1] = c;
    }
}

// the moments as f32 values (store = 0: states -> m, v; 1: m, v -> states); offsets[t]: where tensor t begins in m and v
__global__ __launch_bounds__(256) void adamw_moments_kernel(const bts_adamw_tensor_t* __restrict__ tensors, const int2* __restrict__ chunks,
                                                           const long* __restrict__ offsets, float* __restrict__ mf, float* __restrict__ vf, int store) {
    const int2 ch = chunks[blockIdx.x];
    const bts_adamw_tensor_t t = tensors[ch.x];
    float* mo = mf + offsets[ch.x];
    float* vo = vf + offsets[ch.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll 1
    for (int it = 0; it < 4; ++it) {
        const long b0 = (long)ch.y * kChunk + (it * 4 + wave) * kBlock, i = b0 + lane * 4, left = t.n - i;
        if (b0 >= t.n) break;
        float m[4], v[4];
        if (store) {
            load4(mo, i, left, false, m);
            load4(vo, i, left, false, v);
            if (t.flags & BTS_ADAMW_8BIT) {
                double md[4], vd[4];
                float sm, sv;
#pragma unroll
                for (int e = 0; e < 4; ++e) { md[e] = m[e]; vd[e] = v[e]; }
                ((uint32_t*)t.m)[i >> 2] = encode<true>(md, sm);
                ((uint32_t*)t.v)[i >> 2] = encode<false>(vd, sv);
                if (lane == 0) {
                    t.m_scale[b0 / kBlock] = sm;
                    t.v_scale[b0 / kBlock] = sv;
                }
            } else {
                store4(t.m, i, left, false, m);
                store4(t.v, i, left, false, v);
            }
        } else {
            if (t.flags & BTS_ADAMW_8BIT) {
                decode_m(load_codes(t.m, i), t.m_scale[b0 / kBlock], m);
                decode_v(load_codes(t.v, i), t.v_scale[b0 / kBlock], v);
            } else {
                load4(t.m, i, left, false, m);
                load4(t.v, i, left, false, v);
            }
            store4(mo, i, left, false, m);
            store4(vo, i, left, false, v);
        }
    }
}

constexpr int kNormBlocks = 2048;

}  // namespace

extern "C" long bts_adamw_multi_workspace_bytes(void) { return kNormBlocks * (long)sizeof(double); }

extern "C" int bts_adamw_multi_step(const bts_adamw_tensor_t* tensors, const int32_t* chunks, long n_chunks, double* rows, int n_groups,
                                    const double* hyper, void* workspace, float* grad_norm, bts_stream_t stream) {
    BTS_CHECK_ARG(tensors && chunks && rows && n_chunks > 0 && n_chunks <= 0x7fffffff && n_groups > 0 && n_groups <= BTS_ADAMW_MAX_GROUPS);
    BTS_CHECK_ARG(!workspace == !grad_norm && ((uintptr_t)workspace & 7) == 0);
    hipStream_t st = (hipStream_t)stream;
    HostHyper hh = {};
    if (hyper) {
        for (int g = 0; g < n_groups; ++g)
            for (int i = 0; i < 5; ++i) hh.v[g][i] = hyper[5 * g + i];
        hh.max_norm = hyper[5 * n_groups];
    }
    int parts = 0;
    if (workspace) {
        parts = (int)(n_chunks < kNormBlocks ? n_chunks : kNormBlocks);
        hipLaunchKernelGGL(adamw_norm_kernel, dim3((unsigned)parts), dim3(256), 0, st, tensors, (const int2*)chunks, n_chunks, (double*)workspace);
    }
    hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1024), 0, st, rows, n_groups, hh, hyper ? 1 : 0, 1, (const double*)workspace, parts, grad_norm);
    hipLaunchKernelGGL(adamw_multi_kernel, dim3((unsigned)n_chunks), dim3(256), 0, st, tensors, (const int2*)chunks, n_chunks, (const double*)rows,
                       n_groups);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

extern "C" int bts_adamw_multi_set(double* rows, int n_groups, const double* hyper, bts_stream_t stream) {
    BTS_CHECK_ARG(rows && hyper && n_groups > 0 && n_groups <= BTS_ADAMW_MAX_GROUPS);
    HostHyper hh = {};
    for (int g = 0; g < n_groups; ++g)
        for (int i = 0; i < 5; ++i) hh.v[g][i] = hyper[5 * g + i];
    hh.max_norm = hyper[5 * n_groups];
    hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, rows, n_groups, hh, 1, 0, (const double*)nullptr, 0,
                       (float*)nullptr);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

extern "C" int bts_adamw_multi_moments(const bts_adamw_tensor_t* tensors, const int32_t* chunks, long n_chunks, const int64_t* offsets, float* m, float* v,
                                       int store, bts_stream_t stream) {
    BTS_CHECK_ARG(tensors && chunks && offsets && m && v && n_chunks > 0 && n_chunks <= 0x7fffffff && (store == 0 || store == 1));
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)n_chunks), dim3(256), 0, (hipStream_t)stream, tensors, (const int2*)chunks,
                       (const long*)offsets, m, v, store);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

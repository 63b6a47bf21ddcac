// Layer normalisation over the last axis, forward and backward with the gradients of weight and bias (gfx950).
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), xh = (x - mu) r, y = xh w + b
//   h = dy w:  dx = r (h - mean(h) - xh mean(h xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// A row lives in the registers of LANES lanes (K vectors of 16 bytes each), so x (and dy) are read once: the mean first, then the
// centred squares -- no E[x^2] - mu^2 cancellation.  Statistics, sums and parameters are f32; only x, y, dy, dx may be bf16.
#include "common.h"

namespace {

constexpr int kThreads = 256;       // rows of up to 64 lanes: 256 / LANES rows per block and pass

// 16 bytes at an element-aligned address: rows of odd length or odd stride start anywhere (the memory unit takes dwordx4 accesses
// at any alignment), so one kernel serves every width, stride and storage offset
typedef uint32_t u32x4_a2_t __attribute__((ext_vector_type(4), aligned(2)));

// ODD: C is no multiple of the vector, so a row's last vector is taken element by element
template <typename T, bool ODD>
__device__ __forceinline__ u32x4_t load_raw(const void* base, long off, int c0, int C) {
    const typename T::elem_t* p = (const typename T::elem_t*)base + off + c0;
    u32x4_t v = {0, 0, 0, 0};
    if (ODD ? c0 + T::kVec <= C : c0 < C) {
        const u32x4_a2_t u = *(const u32x4_a2_t*)p;
        v = (u32x4_t){u.x, u.y, u.z, u.w};
    } else if (ODD) {
#pragma unroll
        for (int e = 0; e < T::kVec; ++e)
            if (c0 + e < C) v[e * T::kBytes / 4] |= (T::kBytes == 4 ? ((const uint32_t*)p)[e] : (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1)));
    }
    return v;
}
template <typename T, bool ODD>
__device__ __forceinline__ void load_vec(const void* base, long off, int c0, int C, float* f) {
    T::unpack(load_raw<T, ODD>(base, off, c0, C), f);
}
template <typename T, bool ODD>
__device__ __forceinline__ void store_vec(void* base, long off, int c0, int C, const float* f) {
    typename T::elem_t* p = (typename T::elem_t*)base + off + c0;
    if (ODD ? c0 + T::kVec <= C : c0 < C) {
        const u32x4_t v = T::pack(f);
        *(u32x4_a2_t*)p = (u32x4_a2_t){v.x, v.y, v.z, v.w};
    } else if (ODD) {
#pragma unroll
        for (int e = 0; e < T::kVec; ++e)
            if (c0 + e < C) T::st(p, e, f[e]);
    }
}
// per-channel f32 parameters of one vector (V = 4 or 8); absent parameters take `fill`
template <int V, bool ODD>
__device__ __forceinline__ void load_param(const float* w, int c0, int C, float fill, float* f) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = fill;
    if (w) {
#pragma unroll
        for (int i = 0; i < V; i += 4) load_vec<F32, ODD>(w, 0, c0 + i, C, f + i);
    }
}

template <typename T, bool ODD>
__device__ __forceinline__ void store_sums(float* base, int c0, int C, const float* f) {
#pragma unroll
    for (int i = 0; i < T::kVec; i += 4) store_vec<F32, ODD>(base, 0, c0 + i, C, f + i);
}

// v + the value that another lane of the row holds: lanes 1, 2 (quad), then mirrored halves of 8 and 16, then 16 and 32 lanes away by
// the permlane swaps.  Every step leaves equal sums in all lanes that took part, so "mirrored" pairs the same sums as "exchanged",
// and no step goes through the LDS pipe (ds_bpermute, what __shfl_xor makes, costs its latency six times a sum).
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_lane16(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_lane32(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// sum over aligned groups of N lanes (N a power of two, at most the wave)
template <int N>
__device__ __forceinline__ float lane_sum(float v) {
    if constexpr (N >= 2) v = add_dpp<0xB1>(v);        // quad_perm 1,0,3,2
    if constexpr (N >= 4) v = add_dpp<0x4E>(v);        // quad_perm 2,3,0,1
    if constexpr (N >= 8) v = add_dpp<0x141>(v);       // row_half_mirror
    if constexpr (N >= 16) v = add_dpp<0x140>(v);      // row_mirror
    if constexpr (N >= 32) v = add_lane16(v);
    if constexpr (N >= 64) v = add_lane32(v);
    return v;
}

// Sum over the LANES lanes that hold a row.  LANES > 64: the whole block, through LDS (`red`: one float per wave).  Two sums of one
// row use two sets, so one barrier per sum is enough: a set is written again only behind the barrier of the other.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = lane_sum<LANES < 64 ? LANES : 64>(v);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[threadIdx.x & (LANES / 64 - 1)];
        v = lane_sum<LANES / 64>(v);
    }
    return v;
}

// Bound by memory: 856064 x 96 bf16 63 us (5.2 TB/s; a large copy reaches 4.7-5.1), 8192 x 4096 f32 44 us (6.1, partly from the last-level
// cache), 53504 x 128 f32 13.9 us, 418 x 512 bf16 3.3 us (launch and one latency).  Rows at odd addresses take two lines per vector:
// 2000 x 8191 bf16 21.8 us, 3.0 TB/s.  Shared rows keep w and b in registers over the block's rows.
template <typename T, int LANES, int K, bool ODD>
__global__ __launch_bounds__(LANES > 64 ? LANES : kThreads) void ln_fwd_kernel(const void* __restrict__ x, long xs, void* __restrict__ y, long ys,
                                                                               long M, int C, const float* __restrict__ w,
                                                                               const float* __restrict__ b, float eps,
                                                                               float* __restrict__ mean, float* __restrict__ rstd) {
    constexpr int V = T::kVec, RPB = LANES > 64 ? 1 : kThreads / LANES;
    __shared__ float red[2][LANES > 64 ? LANES / 64 : 1];
    const int lane = threadIdx.x % LANES;
    float wv[K][V], bv[K][V];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        load_param<V, ODD>(w, (lane + j * LANES) * V, C, 1.f, wv[j]);
        load_param<V, ODD>(b, (lane + j * LANES) * V, C, 0.f, bv[j]);
    }
    const float inv = 1.f / (float)C;
    for (long r0 = (long)blockIdx.x * RPB; r0 < M; r0 += (long)gridDim.x * RPB) {
        const long row = r0 + threadIdx.x / LANES;
        const bool on = row < M;
        float f[K][V], s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (lane + j * LANES) * V;
            load_vec<T, ODD>(x, on ? row * xs : 0, c0, on ? C : 0, f[j]);
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[j][e];
        }
        const float mu = row_sum<LANES>(s, red[0]) * inv;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                f[j][e] = (lane + j * LANES) * V + e < C ? f[j][e] - mu : 0.f;
                q += f[j][e] * f[j][e];
            }
        const float rs = 1.f / sqrtf(row_sum<LANES>(q, red[1]) * inv + eps);
        if (mean && on && lane == 0) {
            mean[row] = mu;
            rstd[row] = rs;
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = f[j][e] * rs * wv[j][e] + bv[j][e];
            store_vec<T, ODD>(y, on ? row * ys : 0, (lane + j * LANES) * V, on ? C : 0, o);
        }
    }
}

// 856064 x 96 bf16 103 us (4.8 TB/s) + 5 us for the final sums, 8192 x 4096 bf16 41 + 7, 3344 x 2208 f32 18.2 + 4.5, 13376 x 512 bf16
// 9.8 + 4.4, 418 x 512 bf16 3.7 + 3.0.
// Every block walks rows in steps of the grid and keeps the sums of dy xh and dy over its rows in registers; it writes one partial row
// [2][C] (ws), ln_bwd_final_kernel adds the rows in a fixed order: no atomics, the gradients of the parameters are reproducible.
template <typename T, int LANES, int K, bool ODD, bool PARAM>
__global__ __launch_bounds__(LANES > 64 ? LANES : kThreads) void ln_bwd_kernel(const void* __restrict__ dy, long dys, const void* __restrict__ x, long xs,
                                                                               void* __restrict__ dx, long dxs, long M, int C,
                                                                               const float* __restrict__ w, const float* __restrict__ mean,
                                                                               const float* __restrict__ rstd, float* __restrict__ ws) {
    constexpr int V = T::kVec, RPB = LANES > 64 ? 1 : kThreads / LANES;
    __shared__ float red[2][LANES > 64 ? LANES / 64 : 1];
    const int lane = threadIdx.x % LANES;
    float wv[K][V], dw[K][V], db[K][V];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        load_param<V, ODD>(w, (lane + j * LANES) * V, C, 1.f, wv[j]);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[j][e] = db[j][e] = 0.f;
    }
    const float inv = 1.f / (float)C;
    const long step = (long)gridDim.x * RPB;
    long row = (long)blockIdx.x * RPB + threadIdx.x / LANES;
    // bf16: the next row's vectors are on their way while this row's sums are taken (856064 x 96: 107 -> 95 us, 8192 x 4096: 53 -> 49).
    // f32 has twice the bytes in flight as it is, and its raw vectors would cost twice the registers (8192 x 4096: 80 -> 83 us).
    constexpr bool kAhead = T::kBytes == 2;
    u32x4_t xn[K], gn[K];
    float mun = 0.f, rsn = 0.f;
    auto fetch = [&](long r) {
        const bool on = r < M;
        mun = on ? mean[r] : 0.f;
        rsn = on ? rstd[r] : 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (lane + j * LANES) * V;
            xn[j] = load_raw<T, ODD>(x, on ? r * xs : 0, c0, on ? C : 0);
            gn[j] = load_raw<T, ODD>(dy, on ? r * dys : 0, c0, on ? C : 0);
        }
    };
    if (kAhead) fetch(row);
    for (long r0 = (long)blockIdx.x * RPB; r0 < M; r0 += step, row += step) {
        const bool on = row < M;
        if (!kAhead) fetch(row);
        const float mu = mun, rs = rsn;
        float f[K][V], g[K][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            T::unpack(xn[j], f[j]);
            T::unpack(gn[j], g[j]);
        }
        if (kAhead) fetch(row + step);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (lane + j * LANES) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                f[j][e] = on && c0 + e < C ? (f[j][e] - mu) * rs : 0.f;
                const float h = g[j][e] * wv[j][e];
                s1 += h;
                s2 += h * f[j][e];
                if constexpr (PARAM) {
                    dw[j][e] += g[j][e] * f[j][e];
                    db[j][e] += g[j][e];
                }
            }
        }
        if (dx) {
            const float m1 = row_sum<LANES>(s1, red[0]) * inv, m2 = row_sum<LANES>(s2, red[1]) * inv;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rs * (g[j][e] * wv[j][e] - m1 - f[j][e] * m2);
                store_vec<T, ODD>(dx, on ? row * dxs : 0, (lane + j * LANES) * V, on ? C : 0, o);
            }
        }
    }
    if constexpr (PARAM) {
        float* out = ws + (long)blockIdx.x * 2 * C;
        if constexpr (RPB == 1) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                store_sums<T, ODD>(out, (lane + j * LANES) * V, C, dw[j]);
                store_sums<T, ODD>(out + C, (lane + j * LANES) * V, C, db[j]);
            }
        } else {
            // the block's RPB rows of sums, through LDS: first dw, then db
            constexpr int W = LANES * K * V;
            __shared__ float part[RPB * W];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (t) __syncthreads();
#pragma unroll
                for (int j = 0; j < K; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) part[(threadIdx.x / LANES) * W + (lane + j * LANES) * V + e] = t ? db[j][e] : dw[j][e];
                __syncthreads();
                for (int c = threadIdx.x; c < C; c += kThreads) {
                    float a = 0.f;
#pragma unroll 8
                    for (int i = 0; i < RPB; ++i) a += part[i * W + c];
                    out[(long)t * C + c] = a;
                }
            }
        }
    }
}

// ws [rows][2][C] -> dw, db: 16 of the 2 C columns x 64 row lanes per block, combined in a fixed order
__global__ __launch_bounds__(1024) void ln_bwd_final_kernel(const float* __restrict__ ws, int rows, int C, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float part[64][17];
    const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const long c = (long)blockIdx.x * 16 + cl, n = 2l * C;
    float s = 0.f;
    if (c < n) {
#pragma unroll 8
        for (int r = rl; r < rows; r += 64) s += ws[r * n + c];
    }
    part[rl][cl] = s;
    __syncthreads();
    // 16 waves: wave i adds the 64 sums of column i
    const int col = threadIdx.x >> 6;
    const float t = lane_sum<64>(part[threadIdx.x & 63][col]);
    const long cc = (long)blockIdx.x * 16 + col;
    if ((threadIdx.x & 63) == 0 && cc < n) {
        if (cc < C) { if (dw) dw[cc] = t; }
        else if (db) db[cc - C] = t;
    }
}

struct LnPlan {
    int lanes, k;
    long blocks;
};

constexpr int kLnMaxC = 16384;

// Lanes of a row and vectors per lane.  A row of up to 64 vectors takes one vector per lane: neighbouring lanes read neighbouring 16
// bytes and several rows share a wave.  Up to 64 lanes x 16 elements stay in one wave (no barrier), longer rows take a block at 8
// elements per lane, and 16 above 8192 elements.  Both sides, forward / backward with its sums, us: 856064 x 96 bf16 16 x 1: 70 / 106,
// 8 x 2: 71 / 102, 4 x 3: 95 / 166; 400000 x 32 f32 8 x 1: 20.3 / 32.6, 2 x 4: 26.3 / 44.5; 13376 x 512 bf16 64 x 1: 7.3 / 15.8,
// 16 x 4: 34 / 59; 16384 x 1024 bf16 64 x 2: 14.8 / 27.7, 128 x 1: 15.7 / 32.9; 8192 x 4096 bf16 512 x 1: 28.3 / 52, 256 x 2: 31.6 / 58.
static void ln_lanes(int V, int C, int& lanes, int& k) {
    const int nv = (C + V - 1) / V;
    int kmax = 1;
    if (nv > 64) kmax = C <= 1024 ? 16 / V : (C <= 8192 ? 8 / V : 16 / V);
    lanes = 1;
    while (lanes * kmax < nv) lanes *= 2;
    if (nv > 64 && C <= 1024) lanes = 64;
    else if (nv > 64 && lanes < 256) lanes = 256;
    k = (nv + lanes - 1) / lanes;
}
static LnPlan ln_plan(int dtype, long M, int C, int threads_per_cu) {
    LnPlan p;
    ln_lanes(dtype == BTS_F32 ? 4 : 8, C, p.lanes, p.k);
    const int threads = p.lanes > 64 ? p.lanes : kThreads;
    const long want = (M + threads / p.lanes - 1) / (threads / p.lanes), cap = (long)bts_cu_count() * (threads_per_cu / threads);
    p.blocks = want < cap ? want : cap;
    return p;
}
// Threads per CU: all 2048 where nothing is summed over rows; half of them in the backward pass with the parameters' gradients, whose
// blocks each leave a row of sums (us at 2048 / 1024 / 512: 856064 x 96 bf16 107 / 95 / 124, 3344 x 2208 f32 30 / 24 / 28; without
// the sums 95 / 108 / 170 and 17.5 / 18.7 / 24).
static LnPlan ln_fwd_plan(int dtype, long M, int C) { return ln_plan(dtype, M, C, 2048); }
static LnPlan ln_bwd_plan(int dtype, long M, int C, bool sums) { return ln_plan(dtype, M, C, sums ? 1024 : 2048); }

static bool ln_args(const void* x, int dtype, long M, int C) {
    return x && (dtype == BTS_F32 || dtype == BTS_BF16) && M > 0 && C > 0 && ((uintptr_t)x & (dtype == BTS_F32 ? 3 : 1)) == 0;
}

}  // namespace

#define LN_ODD(T, L, K, F) \
    if (C % T::kVec) { F(T, L, K, true); } else { F(T, L, K, false); }
#define LN_K2(T, L, F) \
    if (p.k == 1) { LN_ODD(T, L, 1, F) } else { LN_ODD(T, L, 2, F) }
#define LN_K4(T, L, F)                                         \
    switch (p.k) {                                             \
        case 1: LN_ODD(T, L, 1, F) break;                      \
        case 2: LN_ODD(T, L, 2, F) break;                      \
        case 3: LN_ODD(T, L, (T::kVec == 4 ? 3 : 2), F) break; \
        default: LN_ODD(T, L, (T::kVec == 4 ? 4 : 2), F)       \
    }
#define LN_LANES(T, F)                      \
    switch (p.lanes) {                      \
        case 1: LN_ODD(T, 1, 1, F) break;   \
        case 2: LN_ODD(T, 2, 1, F) break;   \
        case 4: LN_ODD(T, 4, 1, F) break;   \
        case 8: LN_ODD(T, 8, 1, F) break;   \
        case 16: LN_ODD(T, 16, 1, F) break; \
        case 32: LN_ODD(T, 32, 1, F) break; \
        case 64: LN_K4(T, 64, F) break;     \
        case 256: LN_K2(T, 256, F) break;   \
        case 512: LN_K2(T, 512, F) break;   \
        default: LN_K4(T, 1024, F)          \
    }

extern "C" int bts_layernorm_fwd(const void* x, int dtype, long x_stride, void* y, long y_stride, long M, int C, const float* w, const float* b,
                                 float eps, float* mean, float* rstd, bts_stream_t stream) {
    BTS_CHECK_ARG(ln_args(x, dtype, M, C) && y && y != x && x_stride >= 0 && y_stride >= C && !mean == !rstd && eps >= 0.f);
    BTS_CHECK_ARG(((uintptr_t)y & (dtype == BTS_F32 ? 3 : 1)) == 0);
    if (C > kLnMaxC) return BTS_ERR_UNSUPPORTED;
    const LnPlan p = ln_fwd_plan(dtype, M, C);
    hipStream_t st = (hipStream_t)stream;
#define L_(T, LANES, K, ODD)                                                                                                                 \
    hipLaunchKernelGGL((ln_fwd_kernel<T, LANES, K, ODD>), dim3((unsigned)p.blocks), dim3(LANES > 64 ? LANES : kThreads), 0, st, x, x_stride, y, \
                       y_stride, M, C, w, b, eps, mean, rstd)
    if (dtype == BTS_F32) { LN_LANES(F32, L_) } else { LN_LANES(BF16, L_) }
#undef L_
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

extern "C" long bts_layernorm_bwd_workspace_bytes(int dtype, long M, int C) {
    if ((dtype != BTS_F32 && dtype != BTS_BF16) || M <= 0 || C <= 0 || C > kLnMaxC) return 0;
    return ln_bwd_plan(dtype, M, C, true).blocks * 2 * C * (long)sizeof(float);
}

extern "C" int bts_layernorm_bwd(const void* dy, long dy_stride, const void* x, long x_stride, void* dx, long dx_stride, int dtype, long M, int C,
                                 const float* w, const float* mean, const float* rstd, float* dw, float* db, void* workspace,
                                 bts_stream_t stream) {
    BTS_CHECK_ARG(ln_args(x, dtype, M, C) && ln_args(dy, dtype, M, C) && mean && rstd && (dx || dw || db) && x_stride >= 0 && dy_stride >= 0);
    BTS_CHECK_ARG(!dx || (dx != x && dx != dy && dx_stride >= C && ((uintptr_t)dx & (dtype == BTS_F32 ? 3 : 1)) == 0));
    BTS_CHECK_ARG(!(dw || db) || (workspace && ((uintptr_t)workspace & 3) == 0));
    if (C > kLnMaxC) return BTS_ERR_UNSUPPORTED;
    const LnPlan p = ln_bwd_plan(dtype, M, C, dw || db);
    hipStream_t st = (hipStream_t)stream;
    float* ws = (float*)workspace;
#define L_(T, LANES, K, ODD)                                                                                                         \
    if (dw || db)                                                                                                                    \
        hipLaunchKernelGGL((ln_bwd_kernel<T, LANES, K, ODD, true>), dim3((unsigned)p.blocks), dim3(LANES > 64 ? LANES : kThreads), 0, st, \
                           dy, dy_stride, x, x_stride, dx, dx_stride, M, C, w, mean, rstd, ws);                                      \
    else                                                                                                                             \
        hipLaunchKernelGGL((ln_bwd_kernel<T, LANES, K, ODD, false>), dim3((unsigned)p.blocks), dim3(LANES > 64 ? LANES : kThreads), 0, st, \
                           dy, dy_stride, x, x_stride, dx, dx_stride, M, C, w, mean, rstd, ws)
    if (dtype == BTS_F32) { LN_LANES(F32, L_) } else { LN_LANES(BF16, L_) }
#undef L_
    if (dw || db) hipLaunchKernelGGL(ln_bwd_final_kernel, dim3(ceil_div(2l * C, 16)), dim3(1024), 0, st, ws, (int)p.blocks, C, dw, db);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

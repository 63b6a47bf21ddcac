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

template <typename T>
__device__ __forceinline__ void load_vec(const void* base, long off, int c0, int C, float* f) {
    const typename T::elem_t* p = (const typename T::elem_t*)base + off + c0;
    if (c0 + T::kVec <= C) {
        const u32x4_a2_t u = *(const u32x4_a2_t*)p;
        const u32x4_t v = {u.x, u.y, u.z, u.w};
        T::unpack(v, f);
    } else {
#pragma unroll
        for (int e = 0; e < T::kVec; ++e) f[e] = c0 + e < C ? T::ld(p, e) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store_vec(void* base, long off, int c0, int C, const float* f) {
    typename T::elem_t* p = (typename T::elem_t*)base + off + c0;
    if (c0 + T::kVec <= C) {
        const u32x4_t v = T::pack(f);
        *(u32x4_a2_t*)p = (u32x4_a2_t){v.x, v.y, v.z, v.w};
    } else {
#pragma unroll
        for (int e = 0; e < T::kVec; ++e)
            if (c0 + e < C) T::st(p, e, f[e]);
    }
}
// per-channel f32 parameters of one vector; absent channels take `fill`
template <int V>
__device__ __forceinline__ void load_param(const float* w, int c0, int C, float fill, float* f) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = w && c0 + e < C ? w[c0 + e] : fill;
}

// Sum over the LANES lanes that hold a row.  LANES > 64: the whole block, through LDS (`red`: one float per wave, two sets used in
// turn so that one barrier per sum is enough).
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
    if constexpr (LANES <= 64) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
        return v;
    } else {
        constexpr int W = LANES / 64;
        v = wave_sum(v);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) s += red[i];
        return s;
    }
}

template <typename T, int LANES, int K>
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
        load_param<V>(w, (lane + j * LANES) * V, C, 1.f, wv[j]);
        load_param<V>(b, (lane + j * LANES) * V, C, 0.f, bv[j]);
    }
    const float inv = 1.f / (float)C;
    for (long r0 = (long)blockIdx.x * RPB; r0 < M; r0 += (long)gridDim.x * RPB) {
        const long row = r0 + threadIdx.x / LANES;
        const bool on = row < M;
        float f[K][V], s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (lane + j * LANES) * V;
            load_vec<T>(x, on ? row * xs : 0, c0, on ? C : 0, f[j]);
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
            store_vec<T>(y, on ? row * ys : 0, (lane + j * LANES) * V, on ? C : 0, o);
        }
    }
}

// Every block walks rows in steps of the grid and keeps the sums of dy xh and dy over its rows in registers; it writes one partial row
// [2][C] (ws), ln_bwd_final_kernel adds the rows in a fixed order: no atomics, the gradients of the parameters are reproducible.
template <typename T, int LANES, int K, bool PARAM>
__global__ __launch_bounds__(LANES > 64 ? LANES : kThreads) void ln_bwd_kernel(const void* __restrict__ dy, long dys, const void* __restrict__ x, long xs,
                                                                               void* __restrict__ dx, long dxs, long M, int C,
                                                                               const float* __restrict__ w, const float* __restrict__ mean,
                                                                               const float* __restrict__ rstd, float* __restrict__ ws) {
    constexpr int V = T::kVec, RPB = LANES > 64 ? 1 : kThreads / LANES;
    __shared__ float red[2][2][LANES > 64 ? LANES / 64 : 1];
    const int lane = threadIdx.x % LANES;
    float wv[K][V], dw[K][V], db[K][V];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        load_param<V>(w, (lane + j * LANES) * V, C, 1.f, wv[j]);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[j][e] = db[j][e] = 0.f;
    }
    const float inv = 1.f / (float)C;
    int turn = 0;
    for (long r0 = (long)blockIdx.x * RPB; r0 < M; r0 += (long)gridDim.x * RPB, turn ^= 1) {
        const long row = r0 + threadIdx.x / LANES;
        const bool on = row < M;
        const float mu = on ? mean[row] : 0.f, rs = on ? rstd[row] : 0.f;
        float f[K][V], g[K][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (lane + j * LANES) * V;
            load_vec<T>(x, on ? row * xs : 0, c0, on ? C : 0, f[j]);
            load_vec<T>(dy, on ? row * dys : 0, c0, on ? C : 0, g[j]);
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
            const float m1 = row_sum<LANES>(s1, red[turn][0]) * inv, m2 = row_sum<LANES>(s2, red[turn][1]) * inv;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rs * (g[j][e] * wv[j][e] - m1 - f[j][e] * m2);
                store_vec<T>(dx, on ? row * dxs : 0, (lane + j * LANES) * V, on ? C : 0, o);
            }
        }
    }
    if constexpr (PARAM) {
        float* out = ws + (long)blockIdx.x * 2 * C;
        if constexpr (LANES >= 256) {
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int c = (lane + j * LANES) * V + e;
                    if (c < C) {
                        out[c] = dw[j][e];
                        out[C + c] = db[j][e];
                    }
                }
        } else {
            // the block's kThreads / LANES rows: within a wave by exchange, across its four waves through LDS
            __shared__ float part[kThreads / 64][2][LANES * K * V];
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float a = dw[j][e], c = db[j][e];
#pragma unroll
                    for (int o = LANES; o < 64; o <<= 1) {
                        a += __shfl_xor(a, o, 64);
                        c += __shfl_xor(c, o, 64);
                    }
                    if ((int)(threadIdx.x & 63) < LANES) {
                        part[threadIdx.x >> 6][0][(lane + j * LANES) * V + e] = a;
                        part[threadIdx.x >> 6][1][(lane + j * LANES) * V + e] = c;
                    }
                }
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += kThreads) {
                float a = 0.f, d = 0.f;
#pragma unroll
                for (int i = 0; i < kThreads / 64; ++i) {
                    a += part[i][0][c];
                    d += part[i][1][c];
                }
                out[c] = a;
                out[C + c] = d;
            }
        }
    }
}

// ws [rows][2][C] -> dw, db: 16 columns of the 2 C x 16 row lanes per block, combined in a fixed order
__global__ __launch_bounds__(256) void ln_bwd_final_kernel(const float* __restrict__ ws, int rows, int C, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float part[16][17];
    const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const long c = (long)blockIdx.x * 16 + cl, n = 2l * C;
    float s = 0.f;
    if (c < n)
        for (int r = rl; r < rows; r += 16) s += ws[r * n + c];
    part[rl][cl] = s;
    __syncthreads();
    if (rl == 0 && c < n) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += part[i][cl];
        if (c < C) { if (dw) dw[c] = t; }
        else if (db) db[c - C] = t;
    }
}

struct LnPlan {
    int lanes, k;
    long blocks;
};

constexpr int kLnMaxC = 16384;

// lanes (a power of four) and vectors per lane (<= kmax): the fewest lanes that hold a row
static LnPlan ln_plan(int V, long M, int C, int kmax, int per_cu) {
    const int nv = (C + V - 1) / V;
    LnPlan p;
    p.lanes = 1;
    while (p.lanes * kmax < nv) p.lanes *= 4;
    p.k = (nv + p.lanes - 1) / p.lanes;
    const int rpb = p.lanes > 64 ? 1 : kThreads / p.lanes;
    const long want = (M + rpb - 1) / rpb, cap = (long)bts_cu_count() * per_cu;
    p.blocks = want < cap ? want : cap;
    return p;
}
static LnPlan ln_bwd_plan(int dtype, long M, int C) { return ln_plan(dtype == BTS_F32 ? 4 : 8, M, C, 4, C > 1024 ? 2 : 4); }

static bool ln_args(const void* x, int dtype, long M, int C) {
    return x && (dtype == BTS_F32 || dtype == BTS_BF16) && M > 0 && C > 0 && ((uintptr_t)x & (dtype == BTS_F32 ? 3 : 1)) == 0;
}

}  // namespace

#define LN_K(T, L, F)               \
    switch (p.k) {                  \
        case 1: F(T, L, 1); break;  \
        case 2: F(T, L, 2); break;  \
        case 3: F(T, L, 3); break;  \
        default: F(T, L, 4); break; \
    }
#define LN_LANES(T, F)                       \
    switch (p.lanes) {                       \
        case 1: LN_K(T, 1, F) break;         \
        case 4: LN_K(T, 4, F) break;         \
        case 16: LN_K(T, 16, F) break;       \
        case 64: LN_K(T, 64, F) break;       \
        case 256: LN_K(T, 256, F) break;     \
        default: LN_K(T, 1024, F) break;     \
    }

extern "C" int bts_layernorm_fwd(const void* x, int dtype, long x_stride, void* y, long y_stride, long M, int C, const float* w, const float* b,
                                 float eps, float* mean, float* rstd, bts_stream_t stream) {
    BTS_CHECK_ARG(ln_args(x, dtype, M, C) && y && y != x && x_stride >= 0 && y_stride >= C && !mean == !rstd && eps >= 0.f);
    BTS_CHECK_ARG(((uintptr_t)y & (dtype == BTS_F32 ? 3 : 1)) == 0);
    if (C > kLnMaxC) return BTS_ERR_UNSUPPORTED;
    const LnPlan p = ln_plan(dtype == BTS_F32 ? 4 : 8, M, C, 4, 8);
    hipStream_t st = (hipStream_t)stream;
#define L_(T, LANES, K)                                                                                                              \
    hipLaunchKernelGGL((ln_fwd_kernel<T, LANES, K>), dim3((unsigned)p.blocks), dim3(LANES > 64 ? LANES : kThreads), 0, st, x, x_stride, y, \
                       y_stride, M, C, w, b, eps, mean, rstd)
    if (dtype == BTS_F32) { LN_LANES(F32, L_) } else { LN_LANES(BF16, L_) }
#undef L_
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

extern "C" long bts_layernorm_bwd_workspace_bytes(int dtype, long M, int C) {
    if ((dtype != BTS_F32 && dtype != BTS_BF16) || M <= 0 || C <= 0 || C > kLnMaxC) return 0;
    return ln_bwd_plan(dtype, M, C).blocks * 2 * C * (long)sizeof(float);
}

extern "C" int bts_layernorm_bwd(const void* dy, long dy_stride, const void* x, long x_stride, void* dx, long dx_stride, int dtype, long M, int C,
                                 const float* w, const float* mean, const float* rstd, float* dw, float* db, void* workspace,
                                 bts_stream_t stream) {
    BTS_CHECK_ARG(ln_args(x, dtype, M, C) && ln_args(dy, dtype, M, C) && mean && rstd && (dx || dw || db) && x_stride >= 0 && dy_stride >= 0);
    BTS_CHECK_ARG(!dx || (dx != x && dx != dy && dx_stride >= C && ((uintptr_t)dx & (dtype == BTS_F32 ? 3 : 1)) == 0));
    BTS_CHECK_ARG(!(dw || db) || (workspace && ((uintptr_t)workspace & 3) == 0));
    if (C > kLnMaxC) return BTS_ERR_UNSUPPORTED;
    const LnPlan p = ln_bwd_plan(dtype, M, C);
    hipStream_t st = (hipStream_t)stream;
    float* ws = (float*)workspace;
#define L_(T, LANES, K)                                                                                                                        \
    if (dw || db)                                                                                                                              \
        hipLaunchKernelGGL((ln_bwd_kernel<T, LANES, K, true>), dim3((unsigned)p.blocks), dim3(LANES > 64 ? LANES : kThreads), 0, st, dy, dy_stride, \
                           x, x_stride, dx, dx_stride, M, C, w, mean, rstd, ws);                                                             \
    else                                                                                                                                       \
        hipLaunchKernelGGL((ln_bwd_kernel<T, LANES, K, false>), dim3((unsigned)p.blocks), dim3(LANES > 64 ? LANES : kThreads), 0, st, dy,        \
                           dy_stride, x, x_stride, dx, dx_stride, M, C, w, mean, rstd, ws)
    if (dtype == BTS_F32) { LN_LANES(F32, L_) } else { LN_LANES(BF16, L_) }
#undef L_
    if (dw || db) hipLaunchKernelGGL(ln_bwd_final_kernel, dim3(ceil_div(2l * C, 16)), dim3(256), 0, st, ws, (int)p.blocks, C, dw, db);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

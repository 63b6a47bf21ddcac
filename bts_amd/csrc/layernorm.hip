// Layer normalisation over the last axis, forward and backward with the gradients of weight and bias (gfx950).
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), xh = (x - mu) r, y = xh w + b
//   h = dy w:  dx = r (h - mean(h) - xh mean(h xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// A row lives in the registers of LANES lanes (K vectors of 16 bytes each), so x (and dy) are read once: the mean first, then the
// centred squares -- no E[x^2] - mu^2 cancellation.  Where a row lies far from zero for its spread, the mean's own rounding is taken out
// again.  Statistics, sums and parameters are f32; only x, y, dy, dx may be bf16.
#include "common.h"

namespace {

constexpr int kThreads = 256;       // rows of up to 64 lanes: 256 / LANES rows per block and pass

// 16 bytes at an element-aligned address: rows of odd length or odd stride start anywhere (the memory unit takes dwordx4 accesses
// at any alignment), so one kernel serves every width, stride and storage offset
typedef uint32_t u32x4_a2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a2_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_a2_t __attribute__((aligned(2)));
typedef float f32x4_a4_t __attribute__((ext_vector_type(4), aligned(4)));

// v without its first n elements (n <= kVec), zeros behind
template <typename T>
__device__ __forceinline__ u32x4_t drop_first(u32x4_t v, int n) {
    const int d = T::kBytes == 2 ? n >> 1 : n;                              // whole dwords
    if (d & 4) v = (u32x4_t){0, 0, 0, 0};
    if (d & 2) v = (u32x4_t){v.z, v.w, 0, 0};
    if (d & 1) v = (u32x4_t){v.y, v.z, v.w, 0};
    if (T::kBytes == 2) {
        const uint32_t h = (n & 1) * 16;
        v = (u32x4_t){__builtin_amdgcn_alignbit(v.y, v.x, h), __builtin_amdgcn_alignbit(v.z, v.y, h), __builtin_amdgcn_alignbit(v.w, v.z, h), v.w >> h};
    }
    return v;
}
// A row's K vectors of one lane, as they are loaded: K - 1 whole ones, then one that may lie behind the row's end or, ODD (C is no multiple
// of the vector), reach over it.  That one is loaded from where it still ends inside the row, so that no branch holds the loads up, and
// settle() shifts it into place, zeros behind the row, when it is used.  Only rows shorter than a vector (one lane, one vector) go
// element by element.  Stored in at most three pieces.  Against up to seven masked element accesses in every row it takes off the
// forward / backward pass: 20000 x 1001 bf16 12 / 33 %, 8000 x 2207 bf16 22 / 44 %, 20000 x 1001 f32 3 / 13 %.
// AHEAD or not: where the row is used at once and C is a multiple of the vector, lanes behind the row's end skip their load instead (3344 x
// 2208 f32, 472 idle lanes of 512 in the second vector: 0.8 us of 13 in the forward pass).
template <typename T, int LANES, int K, bool ODD, bool AHEAD>
__device__ __forceinline__ void load_row(const void* base, long off, int lane, int C, u32x4_t* v) {
    constexpr int V = T::kVec;
    const typename T::elem_t* p = (const typename T::elem_t*)base + off;
    if constexpr (ODD && LANES == 1 && K == 1) {
        if (C < V) {
            v[0] = (u32x4_t){0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < V - 1; ++e)
                if (e < C) v[0][e * T::kBytes / 4] |= (T::kBytes == 4 ? ((const uint32_t*)p)[e] : (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1)));
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const int c0 = (lane + j * LANES) * V;
        if (ODD || AHEAD || j < K - 1) {
            const u32x4_a2_t u = *(const u32x4_a2_t*)(p + (j < K - 1 || c0 + V <= C ? c0 : C - V));
            v[j] = (u32x4_t){u.x, u.y, u.z, u.w};
        } else {
            v[j] = (u32x4_t){0, 0, 0, 0};
            if (c0 < C) {
                const u32x4_a2_t u = *(const u32x4_a2_t*)(p + c0);
                v[j] = (u32x4_t){u.x, u.y, u.z, u.w};
            }
        }
    }
}
template <typename T, int LANES, int K, bool ODD, bool AHEAD>
__device__ __forceinline__ u32x4_t settle(u32x4_t v, int lane, int j, int C) {
    if (j < K - 1 || !(ODD || AHEAD)) return v;
    const int over = (lane + j * LANES) * T::kVec + T::kVec - C;             // elements of the vector that are not the row's
    if (!ODD) return over > 0 ? (u32x4_t){0, 0, 0, 0} : v;
    if (LANES == 1 && K == 1) return v;                                      // (C < kVec: a longer row has more vectors, an equal one is not ODD)
    return drop_first<T>(v, over > 0 ? (over < T::kVec ? over : T::kVec) : 0);
}
template <typename T, bool ODD>
__device__ __forceinline__ void store_vec(void* base, long off, int c0, int C, const float* f) {
    typename T::elem_t* p = (typename T::elem_t*)base + off + c0;
    const u32x4_t v = T::pack(f);
    if (ODD ? c0 + T::kVec <= C : c0 < C) {
        *(u32x4_a2_t*)p = (u32x4_a2_t){v.x, v.y, v.z, v.w};
    } else if (ODD && c0 < C) {
        const int n = C - c0;                                                // 1 .. kVec - 1 elements
        const int half = T::kVec / 2;
        if (n & half) *(u32x2_a2_t*)p = (u32x2_a2_t){v.x, v.y};
        const u32x2_t r = n & half ? (u32x2_t){v.z, v.w} : (u32x2_t){v.x, v.y};
        p += n & half;
        if (T::kBytes == 4) {
            if (n & 1) *(uint32_t*)p = r.x;
        } else {
            if (n & 2) *(u32_a2_t*)p = r.x;
            if (n & 1) *(uint16_t*)(p + (n & 2)) = (uint16_t)(n & 2 ? r.y : r.x);
        }
    }
}
// per-channel f32 parameters of one vector (V = 4 or 8); absent parameters take `fill`
template <int V, bool ODD>
__device__ __forceinline__ void load_param(const float* w, int c0, int C, float fill, float* f) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = fill;
    if (w) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            if (ODD ? c0 + i + 4 <= C : c0 < C) {
                const f32x4_a4_t u = *(const f32x4_a4_t*)(w + c0 + i);
                f[i] = u.x; f[i + 1] = u.y; f[i + 2] = u.z; f[i + 3] = u.w;
            } else if (ODD) {
#pragma unroll
                for (int e = i; e < i + 4; ++e)
                    if (c0 + e < C) f[e] = w[c0 + e];
            }
        }
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

// A barrier for what goes through LDS.  __syncthreads() also waits for every global access of the wave: the row behind, whose stores are
// still under way, and the next row, which was asked for ahead of time.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Sum over the LANES lanes that hold a row.  LANES > 64: the whole block, through LDS (`red`: kRed<LANES> floats, one per wave, 0 where there
// is no wave).  Two sums of one row use two sets, so one barrier per sum is enough: a set is written again only behind the barrier of
// the other.
template <int LANES>
constexpr int kRed = LANES <= 128 ? 2 : LANES <= 256 ? 4 : LANES <= 512 ? 8 : 16;
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = lane_sum<LANES < 64 ? LANES : 64>(v);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        lds_barrier();
        v = lane_sum<kRed<LANES>>(red[threadIdx.x & (kRed<LANES> - 1)]);
    }
    return v;
}
template <int LANES, int SETS>
__device__ __forceinline__ void clear_sums(float* red) {                     // the entries that no wave writes
    if constexpr (LANES > 64 && LANES != 64 * kRed<LANES>) {
        if (threadIdx.x < SETS * kRed<LANES>) red[threadIdx.x] = 0.f;
        __syncthreads();
    }
}

// The mean of a row is off by its own rounding and the sum's, a few 2^-24 of |mu|; divided by the deviation that is nothing for most
// rows and everything for a row of equal elements, where the deviation is sqrt(eps) (1000 in 7 columns: 0.019 instead of 0).  The
// centred elements are small, so their mean says by how much it is off (divided by C, not multiplied by 1 / C: exact where all are
// equal).  Rows with |mu| > 4 sqrt(var + eps) pay for it; what it would take out of the others is at most 5 times their sum's roundings.
// us where no row / every row is one: 856064 x 96 bf16 63 / 84, 8192 x 4096 bf16 26 / 34, f32 43.5 / 45, 3344 x 2208 f32 12.6 / 15.9;
// taken for every row regardless it costs rows near zero 71, 31, 44 and 14.3.
constexpr float kFar = 16.f;

// Bound by memory: 856064 x 96 bf16 64 us (5.1 TB/s; a large copy reaches 4.7-5.1), 8192 x 4096 f32 43.5 us (6.2, partly from the last-level
// cache), 53504 x 128 f32 13.2 us, 418 x 512 bf16 3.0 us (launch and one latency), 2000 x 16384 bf16 27.4 us, f32 47 us.  Rows at odd
// addresses, 2000 x 8191 bf16: 19.5 us, 3.4 TB/s.  The bytes from and to memory are those of even rows; the L1 counts 2.7 times the
// accesses (backward 3.2 times), since it takes unaligned 16-byte vectors apart.  Shared rows keep w and b in registers over
// the block's rows.
// Rows of 1024 lanes are held to 64 registers where that spills nothing: two blocks a CU (2000 x 12288 bf16: 21 us, 26 at 68 registers).
template <typename T, int LANES, int K, bool ODD>
__global__ __launch_bounds__(LANES > 64 ? LANES : kThreads, LANES == 1024 && !ODD ? 8 : 1) void ln_fwd_kernel(const void* __restrict__ x, long xs, void* __restrict__ y, long ys,
                                                                               long M, int C, const float* __restrict__ w,
                                                                               const float* __restrict__ b, float eps,
                                                                               float* __restrict__ mean, float* __restrict__ rstd) {
    constexpr int V = T::kVec, RPB = LANES > 64 ? 1 : kThreads / LANES;
    __shared__ float red[4][kRed<LANES>];
    clear_sums<LANES, 4>(red[0]);
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
        u32x4_t raw[K];
        load_row<T, LANES, K, ODD, false>(x, (on ? row : M - 1) * xs, lane, C, raw);
        float f[K][V], s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            T::unpack(settle<T, LANES, K, ODD, false>(raw[j], lane, j, C), f[j]);
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[j][e];
        }
        float mu = row_sum<LANES>(s, red[0]) * inv;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = f[j][e] - mu;
                f[j][e] = j < K - 1 || (lane + j * LANES) * V + (ODD ? e : 0) < C ? d : 0.f;
                q += f[j][e] * f[j][e];
            }
        q = row_sum<LANES>(q, red[1]) * inv;
        if (mu * mu > kFar * (q + eps)) {                                    // the same for all lanes of a row
            float off = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) off += f[j][e];
            off = row_sum<LANES>(off, red[2]) / (float)C;
            mu += off;
            q = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    f[j][e] -= off;
                    if (j < K - 1 || (lane + j * LANES) * V + (ODD ? e : 0) < C) q += f[j][e] * f[j][e];
                }
            q = row_sum<LANES>(q, red[3]) * inv;
        }
        const float rs = 1.f / sqrtf(q + eps);
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

// 856064 x 96 bf16 102 us (4.8 TB/s) + 5 us for the final sums, 8192 x 4096 bf16 35.6 + 4.8, 3344 x 2208 f32 17.4 + 3.9, 13376 x 512 bf16
// 9.8 + 3.8, 2000 x 8191 bf16 27 + 6, 418 x 512 bf16 3.5 + 3.4, 4001 x 667 f32 9.2 + 5.7 (every block walks once and leaves its row of
// sums: 5.3 MB written and read beside 32), 2000 x 16384 bf16 40 + 7, f32 83 + 7.
// Registers with the sums: 64 lanes with two bf16 vectors or, odd, four f32 ones take 130 - 149, three waves a SIMD, so one of the four
// blocks of a CU that the grid counts on waits; 1024 lanes with two bf16 vectors spill 2 (odd widths 8) of 128.
// Every block walks rows in steps of the grid and keeps the sums of dy xh and dy over its rows in registers; it writes one partial row
// [2][C] (ws), ln_bwd_final_kernel adds the rows in a fixed order: no atomics, the gradients of the parameters are reproducible.
template <typename T, int LANES, int K, bool ODD, bool PARAM>
__global__ __launch_bounds__(LANES > 64 ? LANES : kThreads) void ln_bwd_kernel(const void* __restrict__ dy, long dys, const void* __restrict__ x, long xs,
                                                                               void* __restrict__ dx, long dxs, long M, int C,
                                                                               const float* __restrict__ w, const float* __restrict__ mean,
                                                                               const float* __restrict__ rstd, float* __restrict__ ws) {
    constexpr int V = T::kVec, RPB = LANES > 64 ? 1 : kThreads / LANES;
    __shared__ float red[2][kRed<LANES>];
    clear_sums<LANES, 2>(red[0]);
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
    // bf16: the next row's vectors are on their way while this row's sums are taken (856064 x 96: 11 % of the pass, 8192 x 4096: 8 %).
    // f32 has twice the bytes in flight as it is, and its raw vectors would cost twice the registers (8192 x 4096: 4 % longer).
    constexpr bool kAhead = T::kBytes == 2;
    u32x4_t xn[K], gn[K];
    float mun = 0.f, rsn = 0.f;
    auto fetch = [&](long r) {
        r = r < M ? r : M - 1;                                              // rows behind the last one: dy counts as 0 below
        mun = mean[r];
        rsn = rstd[r];
        load_row<T, LANES, K, ODD, kAhead>(x, r * xs, lane, C, xn);
        load_row<T, LANES, K, ODD, kAhead>(dy, r * dys, lane, C, gn);
    };
    if (kAhead) fetch(row);
    for (long r0 = (long)blockIdx.x * RPB; r0 < M; r0 += step, row += step) {
        const bool on = row < M;
        if (!kAhead) fetch(row);
        const float mu = mun, rs = rsn;
        float f[K][V], g[K][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            T::unpack(settle<T, LANES, K, ODD, kAhead>(xn[j], lane, j, C), f[j]);
            const u32x4_t gv = settle<T, LANES, K, ODD, kAhead>(gn[j], lane, j, C);
            T::unpack(on ? gv : (u32x4_t){0, 0, 0, 0}, g[j]);
        }
        if (kAhead && r0 + step < M) fetch(row + step);
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                f[j][e] = (f[j][e] - mu) * rs;                                // an element that is not there has g = 0 and adds nothing
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

// ws [rows][2][C] -> dw, db: 32 of the 2 C columns x 32 row lanes per block, combined in a fixed order (16 or 64 columns make the whole
// backward pass 7 or 11 % longer for 13376 x 512 bf16, 9 or 3 % for 3344 x 2208 f32, 7 or 0 % for 8192 x 4096 bf16).
__global__ __launch_bounds__(1024) void ln_bwd_final_kernel(const float* __restrict__ ws, int rows, int C, float* __restrict__ dw, float* __restrict__ db) {
    constexpr int CL = 32, RL = 1024 / CL;
    __shared__ float part[RL][CL + 1];
    const int cl = threadIdx.x % CL, rl = threadIdx.x / CL;
    const long c = (long)blockIdx.x * CL + cl, n = 2l * C;
    float s = 0.f;
    if (c < n) {
#pragma unroll 8
        for (int r = rl; r < rows; r += RL) s += ws[r * n + c];
    }
    part[rl][cl] = s;
    __syncthreads();
    const int col = threadIdx.x / RL;                                        // the RL sums of a column in neighbouring lanes
    const float t = lane_sum<RL>(part[threadIdx.x % RL][col]);
    const long cc = (long)blockIdx.x * CL + col;
    if (threadIdx.x % RL == 0 && cc < n) {
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
// elements per lane, and 16 above 8192 elements.  The other side against this one, time of the forward / backward pass with its sums:
// 856064 x 96 bf16 16 lanes x 1: 8 x 2 1.01 / 0.96, 4 x 3 1.36 / 1.57; 400000 x 32 f32 8 x 1: 2 x 4 1.30 / 1.37; 13376 x 512 bf16 64 x 1:
// 16 x 4 4.7 / 3.7; 16384 x 1024 bf16 64 x 2: 128 x 1 1.06 / 1.19; 8192 x 4096 bf16 512 x 1: 256 x 2 1.12 / 1.12.
// bf16 rows of 3, 5 or 6 waves take just those (4, 8 and 8 instead: 20000 x 1025 1.14 / 1.10, 30000 x 2049 1.06 / 1.28); wider rows, and
// f32 with its two vectors per lane, do not gain by it (4000 x 5120 bf16 1.15 - 1.33, 8000 x 2208 f32 1.04 / 1.20).
static void ln_lanes(int V, int C, int& lanes, int& k) {
    const int nv = (C + V - 1) / V;
    int kmax = 1;
    if (nv > 64) kmax = C <= 1024 ? 16 / V : (C <= 8192 ? 8 / V : 16 / V);
    lanes = 1;
    while (lanes * kmax < nv) lanes *= 2;
    if (nv > 64 && C <= 1024) lanes = 64;
    else if (nv > 64 && V == 8 && nv <= 384) lanes = (nv + 63) / 64 * 64;
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
// blocks each leave a row of sums (2048 or 512 against 1024: 856064 x 96 bf16 1.13 or 1.31, 3344 x 2208 f32 1.25 or 1.17; without the
// sums 1024 or 512 against 2048: 1.14 or 1.79, 1.07 or 1.37).  Both shapes walk several rows a block; fewer blocks for inputs whose
// blocks would walk one were not tried.
static LnPlan ln_fwd_plan(int dtype, long M, int C) { return ln_plan(dtype, M, C, 2048); }
static LnPlan ln_bwd_plan(int dtype, long M, int C, bool sums) { return ln_plan(dtype, M, C, sums ? 1024 : 2048); }

static bool ln_args(const void* x, int dtype, long M, int C) {
    return x && (dtype == BTS_F32 || dtype == BTS_BF16) && M > 0 && C > 0 && ((uintptr_t)x & (dtype == BTS_F32 ? 3 : 1)) == 0;
}

}  // namespace

// every (lanes, vectors per lane) that ln_lanes gives for a type
#define LN_CASE(T, L, K, F)                                            \
    if (p.lanes == L && p.k == K) {                                    \
        if (C % T::kVec) { F(T, L, K, true); } else { F(T, L, K, false); } \
    } else
#define LN_SHORT(T, F) LN_CASE(T, 1, 1, F) LN_CASE(T, 2, 1, F) LN_CASE(T, 4, 1, F) LN_CASE(T, 8, 1, F) LN_CASE(T, 16, 1, F) LN_CASE(T, 32, 1, F) LN_CASE(T, 64, 1, F) LN_CASE(T, 64, 2, F)
#define LN_LAUNCH(F)                                                                                                                                \
    if (dtype == BTS_F32) {                                                                                                                         \
        LN_SHORT(F32, F) LN_CASE(F32, 64, 3, F) LN_CASE(F32, 64, 4, F) LN_CASE(F32, 256, 2, F) LN_CASE(F32, 512, 2, F)                              \
        LN_CASE(F32, 1024, 2, F) LN_CASE(F32, 1024, 3, F) LN_CASE(F32, 1024, 4, F) return BTS_ERR_UNSUPPORTED;                                      \
    } else {                                                                                                                                        \
        LN_SHORT(BF16, F) LN_CASE(BF16, 192, 1, F) LN_CASE(BF16, 256, 1, F) LN_CASE(BF16, 320, 1, F) LN_CASE(BF16, 384, 1, F)                       \
        LN_CASE(BF16, 512, 1, F) LN_CASE(BF16, 1024, 1, F) LN_CASE(BF16, 1024, 2, F) return BTS_ERR_UNSUPPORTED;                                    \
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
    LN_LAUNCH(L_)
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
    LN_LAUNCH(L_)
#undef L_
    if (dw || db) hipLaunchKernelGGL(ln_bwd_final_kernel, dim3(ceil_div(2l * C, 32)), dim3(1024), 0, st, ws, (int)p.blocks, C, dw, db);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

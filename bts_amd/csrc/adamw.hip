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
// Blocks that a wave loads before it works on the first.  112.8 M f32 / 16.3 M bf16 parameters with 8-bit states, us: 1 (54 registers)
// 334 / 36.4, 2 (68) 332 / 35.0, 4 (106) 328 / 37.2.
constexpr int kAhead = 2;

// Addresses come out of the tensor table; told that they are global memory, the compiler takes global instead of flat accesses (which
// wait for LDS, too).  Four consecutive elements are one access at any element alignment.
#define GLOBAL_ __attribute__((address_space(1)))
typedef float f32x4_a4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a2_t __attribute__((ext_vector_type(2), aligned(2)));

template <bool BF>
struct Raw4 {
    u32x4_t u;
};
template <>
struct Raw4<true> {
    u32x2_t u;
};
// elements i .. i + 3 of an f32 / bf16 array; !FULL: only the first `left` of them exist, the others are 0
template <bool BF, bool FULL>
__device__ __forceinline__ Raw4<BF> load4(const void* base, long i, long left) {
    Raw4<BF> r;
    if constexpr (BF) {
        const GLOBAL_ uint16_t* p = (const GLOBAL_ uint16_t*)(uintptr_t)base + i;
        if (FULL || left >= 4) {
            const u32x2_a2_t t = *(const GLOBAL_ u32x2_a2_t*)p;
            r.u = (u32x2_t){t.x, t.y};
        } else {
            r.u = (u32x2_t){0, 0};
            if (left > 0) r.u.x = p[0];
            if (left > 1) r.u.x |= (uint32_t)p[1] << 16;
            if (left > 2) r.u.y = p[2];
        }
    } else {
        const GLOBAL_ float* p = (const GLOBAL_ float*)(uintptr_t)base + i;
        if (FULL || left >= 4) {
            const f32x4_a4_t t = *(const GLOBAL_ f32x4_a4_t*)p;
            r.u = (u32x4_t){__float_as_uint(t.x), __float_as_uint(t.y), __float_as_uint(t.z), __float_as_uint(t.w)};
        } else {
            r.u = (u32x4_t){0, 0, 0, 0};
            if (left > 0) r.u.x = __float_as_uint(p[0]);
            if (left > 1) r.u.y = __float_as_uint(p[1]);
            if (left > 2) r.u.z = __float_as_uint(p[2]);
        }
    }
    return r;
}
template <bool BF>
__device__ __forceinline__ void unpack4(const Raw4<BF>& r, float* f) {
    if constexpr (BF) {
        f[0] = __uint_as_float(r.u.x << 16); f[1] = __uint_as_float(r.u.x & 0xffff0000u);
        f[2] = __uint_as_float(r.u.y << 16); f[3] = __uint_as_float(r.u.y & 0xffff0000u);
    } else {
        f[0] = __uint_as_float(r.u.x); f[1] = __uint_as_float(r.u.y); f[2] = __uint_as_float(r.u.z); f[3] = __uint_as_float(r.u.w);
    }
}
template <bool BF, bool FULL>
__device__ __forceinline__ void store4(void* base, long i, long left, const float* f) {
    if constexpr (BF) {
        GLOBAL_ uint16_t* p = (GLOBAL_ uint16_t*)(uintptr_t)base + i;
        const uint32_t a = pack_bf16x2(f[0], f[1]), b = pack_bf16x2(f[2], f[3]);
        if (FULL || left >= 4) *(GLOBAL_ u32x2_a2_t*)p = (u32x2_a2_t){a, b};
        else {
            if (left > 0) p[0] = (uint16_t)a;
            if (left > 1) p[1] = (uint16_t)(a >> 16);
            if (left > 2) p[2] = (uint16_t)b;
        }
    } else {
        GLOBAL_ float* p = (GLOBAL_ float*)(uintptr_t)base + i;
        if (FULL || left >= 4) *(GLOBAL_ f32x4_a4_t*)p = (f32x4_a4_t){f[0], f[1], f[2], f[3]};
        else {
            if (left > 0) p[0] = f[0];
            if (left > 1) p[1] = f[1];
            if (left > 2) p[2] = f[2];
        }
    }
}
// four codes; the code arrays are padded to whole blocks of 256, so a word is always there
__device__ __forceinline__ uint32_t load_codes(const void* base, long i) { return ((const GLOBAL_ uint32_t*)(uintptr_t)base)[i >> 2]; }
__device__ __forceinline__ void store_codes(void* base, long i, uint32_t c) { ((GLOBAL_ uint32_t*)(uintptr_t)base)[i >> 2] = c; }
__device__ __forceinline__ float load_scale(const float* base, long b) { return ((const GLOBAL_ float*)(uintptr_t)base)[b]; }
__device__ __forceinline__ void store_scale(float* base, long b, float v) { ((GLOBAL_ float*)(uintptr_t)base)[b] = v; }

// ---- the 8-bit forms ---------------------------------------------------------------------------------------------------------
// the numbers that four codes stand for, without the block's scale
__device__ __forceinline__ void decode_m(uint32_t c, float* f) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    f[0] = lo[0]; f[1] = lo[1]; f[2] = hi[0]; f[3] = hi[1];
}
__device__ __forceinline__ void decode_v(uint32_t c, float* f) {
    const uint32_t even = (c & 0x00ff00ffu) << 7, odd = ((c >> 8) & 0x00ff00ffu) << 7;      // two halves each
    f[0] = (float)__builtin_bit_cast(_Float16, (uint16_t)even);
    f[1] = (float)__builtin_bit_cast(_Float16, (uint16_t)odd);
    f[2] = (float)__builtin_bit_cast(_Float16, (uint16_t)(even >> 16));
    f[3] = (float)__builtin_bit_cast(_Float16, (uint16_t)(odd >> 16));
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
// One block of 256 values, four to a lane -> codes (low word) and the block's scale (high word).  SIGNED: e4m3, else e5m3.  Whatever
// the values are; not inlined, since the update takes it for unusual blocks only.
template <bool SIGNED>
__device__ __noinline__ uint64_t encode_any(double x0, double x1, double x2, double x3) {
    const double x[4] = {x0, x1, x2, x3};
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
    return out | (uint64_t)(uint32_t)(k + 127) << 55;
}

// The same for a block whose largest magnitude is neither tiny nor near the end of f32, from the f32 values: rounding to 24 bits
// first changes the result only where that lands ON a border between two codes, i.e. where the low 19 bits of the f32 value are 0
// (every border has at most five significant bits).  Those few are moved one step towards the value that they came from.
__device__ __forceinline__ void off_the_border(const double* x, uint32_t* u) {
    uint32_t least = u[0] << 13;
#pragma unroll
    for (int e = 1; e < 4; ++e) least = least < (u[e] << 13) ? least : (u[e] << 13);
    if (__any(least == 0)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double d = (double)__uint_as_float(u[e]), ax = __builtin_fabs(x[e]), ad = __builtin_fabs(d);
            if ((u[e] << 13) == 0) u[e] = ax > ad ? u[e] + 1 : (ax < ad ? u[e] - 1 : u[e]);
        }
    }
}
constexpr uint32_t kTiny = 27u << 23, kHuge = 0x7f780000u;       // 2^-100; 2^128 in four bits
__device__ __forceinline__ uint32_t round_four(uint32_t u) { return (u + 0x7ffffu + ((u >> 20) & 1u)) >> 20; }

__device__ __forceinline__ uint32_t encode_m(const double* x, const float* x32, float& scale) {
    uint32_t u[4], top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(x32[e]);
    off_the_border(x, u);
#pragma unroll
    for (int e = 0; e < 4; ++e) top = top > (u[e] & 0x7fffffffu) ? top : (u[e] & 0x7fffffffu);
    top = max_dpp(top);
    if (top < kTiny || top >= kHuge) {
        const uint64_t r = encode_any<true>(x[0], x[1], x[2], x[3]);
        scale = __uint_as_float((uint32_t)(r >> 32));
        return (uint32_t)r;
    }
    int k = (int)((round_four(top) + 1) >> 3) - 127 - 8;                   // e4m3 ends at 1.75 x 2^8: 1.875 x 2^n takes the next k
    k = k > -126 ? k : -126;
    scale = __uint_as_float((uint32_t)(k + 127) << 23);
    const float inv = __uint_as_float((uint32_t)(127 - k) << 23);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(u[0]) * inv, __uint_as_float(u[1]) * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(u[2]) * inv, __uint_as_float(u[3]) * inv, c, true);
}
__device__ __forceinline__ uint32_t encode_v(const double* x, const float* x32, float& scale) {
    uint32_t u[4], top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(x32[e]);
    off_the_border(x, u);
#pragma unroll
    for (int e = 0; e < 4; ++e) top = top > u[e] ? top : u[e];
    top = max_dpp(top);
    if (top < kTiny || top >= kHuge) {
        const uint64_t r = encode_any<false>(x[0], x[1], x[2], x[3]);
        scale = __uint_as_float((uint32_t)(r >> 32));
        return (uint32_t)r;
    }
    int k = (int)(round_four(top) >> 3) - 127 - 15;
    k = k > -126 ? k : -126;
    scale = __uint_as_float((uint32_t)(k + 127) << 23);
    const int shift = (127 + k - 15) << 3;
    int c[4];
    bool low = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        c[e] = (int)round_four(u[e]) - shift;
        low |= c[e] < 8;
    }
    if (__any(low)) {                                                      // below the normal numbers
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c[e] < 8) {
                c[e] = (int)multiples(x[e], 17 - k);
                if (c[e] == 0 && u[e] != 0) c[e] = 1;
            }
    }
    return (uint32_t)(c[0] | (c[1] << 8)) | ((uint32_t)(c[2] | (c[3] << 8)) << 16);
}

// rows, kRow doubles per group: {lr, 1 - b1^t, 1 - b2^t, t, b1, b2, eps, weight decay} and, formed with the step count, what the update
// takes: {1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - b1, 1 - b2}; behind the groups {max_norm, c}
constexpr int kRow = BTS_ADAMW_ROW;

struct Hyper {
    double b1, b2, a1, a2, clip;
    float decay, step, rs, eps;
};

// what one wave reads of one block of 256 elements
template <bool BF, bool B8>
struct Block {
    Raw4<BF> p, g;
    Raw4<false> m, v;
    uint32_t mc, vc;
    float ms, vs;
};
template <bool BF, bool B8, bool FULL>
__device__ __forceinline__ void load_block(const bts_adamw_tensor_t& t, long b0, int lane, Block<BF, B8>& k) {
    const long i = b0 + lane * 4, left = t.n - i;
    k.p = load4<BF, FULL>(t.p, i, left);
    k.g = load4<BF, FULL>(t.g, i, left);
    if constexpr (B8) {
        k.mc = load_codes(t.m, i);
        k.vc = load_codes(t.v, i);
        k.ms = load_scale(t.m_scale, b0 / kBlock);
        k.vs = load_scale(t.v_scale, b0 / kBlock);
    } else {
        k.m = load4<false, FULL>(t.m, i, left);
        k.v = load4<false, FULL>(t.v, i, left);
    }
}
template <bool BF, bool B8, bool FULL>
__device__ __forceinline__ void update_block(const bts_adamw_tensor_t& t, long b0, int lane, const Block<BF, B8>& k, const Hyper& h) {
    const long i = b0 + lane * 4, left = t.n - i;
    float p[4], g[4], m32[4], v32[4];
    unpack4(k.p, p);
    unpack4(k.g, g);
    if constexpr (B8) {
        float mo[4], vo[4], sm, sv;
        decode_m(k.mc, mo);
        decode_v(k.vc, vo);
        const double b1 = h.b1 * (double)k.ms, b2 = h.b2 * (double)k.vs;       // powers of two: (b1 s) x rounds like b1 (s x)
        double m[4], v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double gd = (double)g[e] * h.clip;
            m[e] = b1 * (double)mo[e] + h.a1 * gd;               // every product and sum rounded, in this order: with gradients of
            v[e] = b2 * (double)vo[e] + h.a2 * gd * gd;          // few bits (bf16, zeros) one value in a thousand IS a border
            if (!FULL && e >= left) m[e] = v[e] = 0.0;
            m32[e] = (float)m[e];
            v32[e] = (float)v[e];
        }
        store_codes(t.m, i, encode_m(m, m32, sm));
        store_codes(t.v, i, encode_v(v, v32, sv));
        if (lane == 0) {
            store_scale(t.m_scale, b0 / kBlock, sm);
            store_scale(t.v_scale, b0 / kBlock, sv);
        }
    } else {
        unpack4(k.m, m32);
        unpack4(k.v, v32);
        const float b1 = (float)h.b1, b2 = (float)h.b2, a1 = (float)h.a1, a2 = (float)h.a2, c = (float)h.clip;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float gc = g[e] * c;
            m32[e] = b1 * m32[e] + a1 * gc;
            v32[e] = b2 * v32[e] + a2 * gc * gc;
        }
        store4<false, FULL>(t.m, i, left, m32);
        store4<false, FULL>(t.v, i, left, v32);
    }
    // The hardware's root and reciprocal (each within one step of f32) do where eps keeps the divisor far from the subnormal numbers,
    // which they flush; otherwise the correctly rounded ones.
    if (h.eps >= 1e-12f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = fmaf(p[e], h.decay, -h.step * (m32[e] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v32[e]) * h.rs + h.eps)));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = fmaf(p[e], h.decay, -h.step * (m32[e] / (sqrtf(v32[e]) * h.rs + h.eps)));
    }
    store4<BF, FULL>(t.p, i, left, p);                                     // bf16 parameters: the one rounding to fewer bits, to nearest even
}
template <bool BF, bool B8>
__device__ __forceinline__ void update_chunk(const bts_adamw_tensor_t& t, long base, int wave, int lane, const Hyper& h) {
    if (base + kChunk <= t.n) {
#pragma unroll 1
        for (int it = 0; it < 4; it += kAhead) {
            Block<BF, B8> k[kAhead];                                       // the loads of kAhead blocks before the first use
#pragma unroll
            for (int j = 0; j < kAhead; ++j) load_block<BF, B8, true>(t, base + ((it + j) * 4 + wave) * kBlock, lane, k[j]);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) update_block<BF, B8, true>(t, base + ((it + j) * 4 + wave) * kBlock, lane, k[j], h);
        }
    } else {
#pragma unroll 1
        for (int it = 0; it < 4; ++it) {
            const long b0 = base + (it * 4 + wave) * kBlock;
            if (b0 >= t.n) break;
            Block<BF, B8> k;
            load_block<BF, B8, false>(t, b0, lane, k);
            update_block<BF, B8, false>(t, b0, lane, k, h);
        }
    }
}

// One block per chunk: the tensors' sizes differ by five orders of magnitude, equal chunks make equal blocks.  Bound by memory: 550 tensors,
// 47.0 M f32 parameters with 8-bit states take 157-168 us for 752 MB (4.5-4.8 TB/s; a large copy reaches 4.7-5.1) at 51 VALU instructions an
// element, 61 us of issue; counted traffic is 484 MB read, 288 MB written.  16.3 M bf16: 35 us, 163 MB.  20.5 M bf16 parameters with
// 32-bit states: 90 us, 451 MB.  (With flat accesses, one path for all types and the general encoder: 194, 71 and 98 us.)
__global__ __launch_bounds__(256) void adamw_multi_kernel(const bts_adamw_tensor_t* __restrict__ tensors, const int2* __restrict__ chunks, long n_chunks,
                                                         const double* __restrict__ rows, int n_groups) {
    // last chunk first: behind a norm pass the gradients that were read last are the ones that the cache still holds
    const int2 ch = chunks[n_chunks - 1 - blockIdx.x];
    const bts_adamw_tensor_t t = tensors[ch.x];
    const double* r = rows + kRow * t.group;
    const Hyper h = {r[4], r[5], r[11], r[12], rows[kRow * n_groups + 1], (float)r[8], (float)r[9], (float)r[10], (float)r[6]};
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long base = (long)ch.y * kChunk;
    if (t.flags & BTS_ADAMW_8BIT) {
        if (t.flags & BTS_ADAMW_BF16) update_chunk<true, true>(t, base, wave, lane, h);
        else update_chunk<false, true>(t, base, wave, lane, h);
    } else {
        if (t.flags & BTS_ADAMW_BF16) update_chunk<true, false>(t, base, wave, lane, h);
        else update_chunk<false, false>(t, base, wave, lane, h);
    }
}

// sum of squares of every gradient, in f64 (no overflow of g^2, no loss over 10^8 terms): one partial sum per block, fixed order.
// 1000 M f32 gradients: 710 us, 5.6 TB/s; 112.8 M: 53 us, more than memory gives, since a part is in the last-level cache still.
template <bool BF>
__device__ __forceinline__ void add_squares(const bts_adamw_tensor_t& t, long base, double& s) {
    Raw4<BF> r[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const long i = base + it * 1024 + threadIdx.x * 4, left = t.n - i;
        r[it] = load4<BF, false>(t.g, i, left);
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        float g[4];
        unpack4(r[it], g);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fma((double)g[e], (double)g[e], s);
    }
}
__global__ __launch_bounds__(256) void adamw_norm_kernel(const bts_adamw_tensor_t* __restrict__ tensors, const int2* __restrict__ chunks, long n_chunks,
                                                        double* __restrict__ partials) {
    double s = 0.0;
    for (long c = blockIdx.x; c < n_chunks; c += gridDim.x) {
        const int2 ch = chunks[c];
        const bts_adamw_tensor_t t = tensors[ch.x];
        if (t.flags & BTS_ADAMW_BF16) add_squares<true>(t, (long)ch.y * kChunk, s);
        else add_squares<false>(t, (long)ch.y * kChunk, s);
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
            const double most = set ? hh.max_norm : tail[0];
            c = most / (t + 1e-6);
            c = c > 1.0 ? 1.0 : c;                                  // a norm that is NaN makes c NaN, and with it every parameter
            if (most == __builtin_inf()) c = 1.0;                   // only measured: whatever the norm is
        }
        if (advance) tail[1] = c;
    }
}

// 47.0 M elements: 95 us for 470 MB.
// the moments as f32 values (store = 0: states -> m, v; 1: m, v -> states); offsets[t]: where tensor t begins in m and v
__global__ __launch_bounds__(256) void adamw_moments_kernel(const bts_adamw_tensor_t* __restrict__ tensors, const int2* __restrict__ chunks,
                                                           const long* __restrict__ offsets, float* __restrict__ mf, float* __restrict__ vf, int store) {
    const int2 ch = chunks[blockIdx.x];
    const bts_adamw_tensor_t t = tensors[ch.x];
    float* mo = mf + offsets[ch.x];
    float* vo = vf + offsets[ch.x];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool eight = t.flags & BTS_ADAMW_8BIT;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const long b0 = (long)ch.y * kChunk + (it * 4 + wave) * kBlock, i = b0 + lane * 4, left = t.n - i;
        if (b0 >= t.n) break;
        float m[4], v[4];
        if (store) {
            unpack4(load4<false, false>(mo, i, left), m);
            unpack4(load4<false, false>(vo, i, left), v);
            if (eight) {
                const uint64_t rm = encode_any<true>(m[0], m[1], m[2], m[3]), rv = encode_any<false>(v[0], v[1], v[2], v[3]);
                store_codes(t.m, i, (uint32_t)rm);
                store_codes(t.v, i, (uint32_t)rv);
                if (lane == 0) {
                    store_scale(t.m_scale, b0 / kBlock, __uint_as_float((uint32_t)(rm >> 32)));
                    store_scale(t.v_scale, b0 / kBlock, __uint_as_float((uint32_t)(rv >> 32)));
                }
            } else {
                store4<false, false>(t.m, i, left, m);
                store4<false, false>(t.v, i, left, v);
            }
        } else {
            if (eight) {
                const float ms = load_scale(t.m_scale, b0 / kBlock), vs = load_scale(t.v_scale, b0 / kBlock);
                decode_m(load_codes(t.m, i), m);
                decode_v(load_codes(t.v, i), v);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m[e] *= ms;
                    v[e] *= vs;
                }
            } else {
                unpack4(load4<false, false>(t.m, i, left), m);
                unpack4(load4<false, false>(t.v, i, left), v);
            }
            store4<false, false>(mo, i, left, m);
            store4<false, false>(vo, i, left, v);
        }
    }
}

constexpr int kNormBlocks = 2048;

}  // namespace

extern "C" long bts_adamw_multi_workspace_bytes(void) { return kNormBlocks * (long)sizeof(double); }

extern "C" int bts_adamw_multi_step(const bts_adamw_tensor_t* tensors, const int32_t* chunks, long n_chunks, double* rows, int n_groups,
                                    const double* hyper, void* workspace, float* grad_norm, bts_stream_t stream) {
    BTS_CHECK_ARG(tensors && chunks && rows && n_chunks > 0 && n_chunks <= 0xffffff && n_groups > 0 && n_groups <= BTS_ADAMW_MAX_GROUPS);
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
    BTS_CHECK_ARG(tensors && chunks && offsets && m && v && n_chunks > 0 && n_chunks <= 0xffffff && (store == 0 || store == 1));
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)n_chunks), dim3(256), 0, (hipStream_t)stream, tensors, (const int2*)chunks,
                       (const long*)offsets, m, v, store);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

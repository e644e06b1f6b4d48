// kv4.cu -- writing rows of the 4-bit K/V cache (kv4.cuh) and reading them back.
//
// Quantiser, for the 64 elements x of a group, lo = min x, hi = max x:
//     c = f16(lo + (hi - lo) * (8/15))                    (f32 steps, then nearest f16)
//     d = the least number >= max((c - lo) / 8, (hi - c) / 7) that has 8 significant
//         bits and is a multiple of 2^-24
//     n' = floor((x - c) / d + 1/2),  0 where d = 0
// The choice of d makes every n' fall into -8..7 without clamping and leaves every element
// within d / 2 of its value.  The comparisons are exact (no rounding decides a code), so
// the result does not depend on how the division is carried out.  A group with an element
// that is NaN, infinite or larger than 57344 in magnitude gets c = NaN, d = 0 and reads
// back as NaN; 57344 keeps 8 d below the largest f16.
//
// Both kernels move bytes, and the arithmetic per byte decides how near they come to the memory's
// rate.  Storing, four lanes share a group (lane j: elements 16 j .. 16 j + 15, code words 2 j and
// 2 j + 1): with eight lanes of eight elements the range, c and d, which every lane computes for
// itself, cost as much again.  Loading, eight lanes share a group.  One CTA takes up to 32
// consecutive rows of one (slot, head), K and V, so its 32-byte code rows are one run.
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include "internal.h"
#include "kv4.cuh"

namespace madi {
namespace {

constexpr int kThr = 128;
constexpr int kRows = 32;      // rows per CTA: small CTAs, whose loads and arithmetic overlap one another's
constexpr float kLimit = 57344.f;

MADI_DEV __half2 as_h2(uint32_t w) { return *reinterpret_cast<__half2 *>(&w); }
MADI_DEV float min_nan(float x, float y) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
MADI_DEV float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
// Sixteen consecutive elements as loaded.  range: the smallest and largest element of the group,
// in all of its four lanes; NaN if one of the 64 is.  f16: on packed pairs, the largest as the
// smallest of the negated, so that one shuffle carries both.
template <typename T> struct Src16;
template <> struct Src16<float> {
    float4 v[4];
    MADI_DEV void load(const float *p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = reinterpret_cast<const float4 *>(p)[i];
    }
    MADI_DEV void f32(float (&f)[16]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[4 * i] = v[i].x;
            f[4 * i + 1] = v[i].y;
            f[4 * i + 2] = v[i].z;
            f[4 * i + 3] = v[i].w;
        }
    }
    MADI_DEV void range(float &lo, float &hi) const {
        lo = v[0].x;
        hi = v[0].x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo = min_nan(min_nan(lo, min_nan(v[i].x, v[i].y)), min_nan(v[i].z, v[i].w));
            hi = max_nan(max_nan(hi, max_nan(v[i].x, v[i].y)), max_nan(v[i].z, v[i].w));
        }
#pragma unroll
        for (int o = 2; o; o >>= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
    }
};
template <> struct Src16<__half> {
    uint32_t w[8];
    MADI_DEV void load(const __half *p) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 u = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = u.x;
            w[4 * i + 1] = u.y;
            w[4 * i + 2] = u.z;
            w[4 * i + 3] = u.w;
        }
    }
    MADI_DEV void f32(float (&f)[16]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = __half22float2(as_h2(w[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
    MADI_DEV void range(float &lo, float &hi) const {
        __half2 a = as_h2(w[0]), b = a;
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            a = __hmin2_nan(a, as_h2(w[i]));
            b = __hmax2_nan(b, as_h2(w[i]));
        }
        __half2 m = __halves2half2(__hmin_nan(__low2half(a), __high2half(a)),
                                   __hneg(__hmax_nan(__low2half(b), __high2half(b))));
#pragma unroll
        for (int o = 2; o; o >>= 1) m = __hmin2_nan(m, as_h2(__shfl_xor_sync(0xffffffffu, h2_as_u32(m), o)));
        lo = __low2float(m);
        hi = -__high2float(m);
    }
};

// The step d: the least number with 8 significant bits that is a multiple of 2^-24, with
// 8 d >= c - lo and 7 d >= hi - c.  (Differences rounded up compare with 7 d and 8 d as the exact
// ones do, since both products are f32 numbers.)  An estimate from below by the reciprocal of 7 is
// raised to the grid, and raised once more if 7 d falls short, or 8 d: an eighth of a few 2^-149 is 0.
MADI_DEV float step_of(float lo, float hi, float c) {
    const float up = __fsub_ru(hi, c), down = __fsub_ru(c, lo);
    const float r = fmaxf(down * 0.125f, up * 0.14285707f);       // (1/7)(1 - 5e-7)
    float d;
    if (r < 7.62939453125e-06f) {                        // below 2^-17 the multiples of 2^-24 are the coarser grid
        d = ceilf(r * 16777216.f) * 5.9604644775390625e-08f;
        if (d * 7.f < up || d * 8.f < down) d += 5.9604644775390625e-08f;
    } else {
        uint32_t b = (__float_as_uint(r) + 0xFFFFu) & 0xFFFF0000u;
        if (__uint_as_float(b) * 7.f < up) b += 0x10000u;
        d = __uint_as_float(b);
    }
    return d;
}

// n' of x, exactly.  The quotient with the reciprocal is within one of the answer; the two
// comparisons x - c >= (n' -+ 1/2) d settle it: x - c = t + e without error, the product (at most
// 5 by 8 bits) and its difference from t decide by sign, e on equality (|e| is below the spacing
// of that difference).
MADI_DEV float code_exact(float x, float c, float d, float inv) {
    const float t = x - c;
    const float b = t - x;
    const float e = (x - (t - b)) + (-c - b);
    float g = rintf(t * inv);
    const float lo = fmaf(0.5f - g, d, t);               // t - (g - 1/2) d
    const float hi = fmaf(-0.5f - g, d, t);              // t - (g + 1/2) d
    if (lo < 0.f || (lo == 0.f && e < 0.f)) g -= 1.f;
    else if (hi > 0.f || (hi == 0.f && e >= 0.f)) g += 1.f;
    return g;
}

// The code words of sixteen elements.  Adding 1.5 x 2^23 and taking it off rounds the quotient to
// n' (packed arithmetic); four codes at a time are collected as the f32 integer
// ((n'3 16 + n'2) 16 + n'1) 16 + n'0, exactly.  The quotient is taken of t + 2^-18 d, t = x - c, so
// that a half, which f16 inputs hit once in some hundred elements, is rounded up although the
// reciprocal is not exact (its error and the product's are 2^-19 together).  The remainder r = t -
// n' d has to lie in [-d/2, d/2): codes that it shows to be wrong, within 2^-18 of a border, are rare, and
// then all sixteen are decided one by one.  Where r = -d/2, two things are looked at: r is exact but for
// a t just below d/2 = 2^k (its last place is half of r's), so t - (n' - 1/2) d, which is, decides; and if that is
// 0, x - c must not lie below t.
MADI_DEV void code_words(const float (&x)[16], float c, float d, uint32_t (&w)[2]) {
    constexpr float kMagic = 12582912.f;
    const float inv = rcp_approx(d), h = 0.5f * d, c2 = fmaf(-3.814697265625e-06f, d, c);
    float least = 0.f, most = 0.f, z[16];
#pragma unroll
    for (int q = 0; q < 16; q += 2) {
        float t0, t1, g0, g1, r0, r1;
        add2(g0, g1, x[q], x[q + 1], -c2, -c2);
        fma2(g0, g1, g0, g1, inv, inv, kMagic, kMagic);
        add2(z[q], z[q + 1], g0, g1, -kMagic, -kMagic);
        add2(t0, t1, x[q], x[q + 1], -c, -c);
        fma2(r0, r1, z[q], z[q + 1], -d, -d, t0, t1);
        asm("min.f32 %0, %1, %2, %3;" : "=f"(least) : "f"(least), "f"(r0), "f"(r1));
        asm("max.f32 %0, %1, %2, %3;" : "=f"(most) : "f"(most), "f"(r0), "f"(r1));
    }
    if (!(least > -h && most < h)) {
        bool wrong = least < -h || most >= h;
        if (!wrong) {                                        // t - (n' - 1/2) d + (x - c - t) < 0 only if r = -d/2
#pragma unroll
            for (int q = 0; q < 16; q += 2) {
                float t0, t1, b0, b1, u0, u1, e0, e1, s0, s1;
                add2(t0, t1, x[q], x[q + 1], -c, -c);
                add2(b0, b1, t0, t1, -x[q], -x[q + 1]);
                add2(u0, u1, t0, t1, -b0, -b1);
                add2(u0, u1, x[q], x[q + 1], -u0, -u1);
                add2(e0, e1, -c, -c, -b0, -b1);
                add2(e0, e1, u0, u1, e0, e1);
                add2(s0, s1, -z[q], -z[q + 1], 0.5f, 0.5f);
                fma2(s0, s1, s0, s1, d, d, t0, t1);
                wrong = wrong || s0 + e0 < 0.f || s1 + e1 < 0.f;
            }
        }
        if (wrong) {
#pragma unroll
            for (int q = 0; q < 16; ++q) z[q] = code_exact(x[q], c, d, inv);
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint32_t h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float *y = z + 8 * k + 4 * i;
            const float f = fmaf(fmaf(fmaf(y[3], 16.f, y[2]), 16.f, y[1]), 16.f, y[0]);
            h[i] = __float_as_uint(f + (kMagic + 34952.f));   // + 0x8888: the eights of n' + 8
        }
        w[k] = __byte_perm(h[0], h[1], 0x5410);
    }
}

// Bound by its instructions and the latency of its loads: 23.0 us for 8 x 1500 f16 rows of 20 heads (79 MB,
// 3.4 TB/s), 24.5 for f32 ones (140 MB, 5.7 TB/s).  Six CTAs per SM: 80 registers, of which two spill.  Measured at an
// earlier state that took 24.8: 30.5 with the 102 registers it would take, 30.8 with 64; 26.6 with CTAs of 256
// threads and 64 rows.
// No pointer of these kernels is __restrict__: their memory is written while they are already resident (by the
// kernel before them, until pdl_wait), so loads through the read-only path would be wrong.
template <typename T>
__global__ void __launch_bounds__(kThr, 6) kv4_store_kernel(uint8_t *data, long long slot_bytes, long long head_bytes,
                                                            int max_tok, const T *k, const T *v, long long slot_stride,
                                                            long long row_stride, int rows, const uint32_t *pos,
                                                            const uint32_t *n) {
    pdl_trigger();
    pdl_wait();
    const int h = blockIdx.y, r0 = (int)blockIdx.x * kRows, s = blockIdx.z;
    const int nr = min(kv4_rows(n, s, rows) - r0, kRows);       // rows of this CTA
    const unsigned long long first = (pos ? (unsigned long long)pos[s] : 0ull) + (unsigned)r0;
    if (nr <= 0 || first >= (unsigned long long)max_tok) return;     // padding, or past the cache
    const int at0 = (int)first;
    uint8_t *head = data + s * slot_bytes + h * head_bytes;
    const int j = threadIdx.x & 3, grp = threadIdx.x >> 2, ng = blockDim.x >> 2;
    const long long src0 = s * slot_stride + r0 * row_stride + h * kKv4Hd + 16 * j;
    for (int i = 0; i < nr; i += ng) {                        // the same trips for every lane: shuffles inside
        const int r = min(i + grp, nr - 1);
        Src16<T> src[2];
        src[0].load(k + src0 + r * row_stride);
        src[1].load(v + src0 + r * row_stride);
        const uint32_t at = (uint32_t)(at0 + r);              // below 2^30 + 64
        const bool store = i + grp < nr && at < (uint32_t)max_tok;       // rows past the cache are dropped
        uint8_t *blk = head + (long long)(at / kKv4Blk) * kKv4Block;
        const int off = (int)(at % kKv4Blk);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float lo, hi, x[16];
            src[b].range(lo, hi);
            src[b].f32(x);
            const bool ok = lo >= -kLimit && hi <= kLimit;    // false for NaN
            const float c = __half2float(__float2half_rn(__fadd_rn(lo, __fmul_rn(__fsub_rn(hi, lo), 8.f / 15.f))));
            const float d = ok ? step_of(lo, hi, c) : 0.f;
            uint32_t w[2] = {0x88888888u, 0x88888888u};
            if (d > 0.f) code_words(x, c, d, w);
            if (!store) continue;
            reinterpret_cast<uint2 *>(blk + b * kKv4Half + off * 32)[j] = make_uint2(w[0], w[1]);
            if (j == 0)
                *reinterpret_cast<uint32_t *>(blk + b * kKv4Half + kKv4Codes + off * 4) =
                    h2_as_u32(__halves2half2(__float2half_rn(ok ? c : CUDART_NAN_F), __float2half_rn(d)));
        }
    }
}

// The values of a group that lane j of eight writes, value = c + d n' rounded once (f32: one FMA,
// d n' being exact; f16: one f16 FMA): 16 bytes at a time, so that the eight lanes' stores are
// one run -- f16: elements 8 j .. (code word j); f32: elements 4 j .. and 32 + 4 j .. (half of
// code words j / 2 and 4 + j / 2).
struct Codes2 {
    uint32_t w[2];
};
MADI_DEV Codes2 ld_codes(const float *, const uint8_t *row, int j) {
    return {{reinterpret_cast<const uint32_t *>(row)[j >> 1], reinterpret_cast<const uint32_t *>(row)[4 + (j >> 1)]}};
}
MADI_DEV Codes2 ld_codes(const __half *, const uint8_t *row, int j) {
    return {{reinterpret_cast<const uint32_t *>(row)[j], 0u}};
}
MADI_DEV void st_values(float *p, const Codes2 &u, __half2 cd, int j) {
    const float c = __low2float(cd), d = __high2float(cd);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        // nibble q kept in place under the exponent of 2^23 is 2^23 + z 16^q; taking off 2^23 +
        // 8 x 16^q leaves n' 16^q, and d / 16^q goes with it (all exact)
        const uint32_t w = u.w[k] >> (16 * (j & 1));
        float f[4];
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            const float s0 = q ? 256.f : 1.f, s1 = q ? 4096.f : 16.f;
            const float z0 = __uint_as_float((w & (15u << (4 * q))) | 0x4B000000u);
            const float z1 = __uint_as_float((w & (15u << (4 * q + 4))) | 0x4B000000u);
            add2(f[q], f[q + 1], z0, z1, -8388608.f - 8.f * s0, -8388608.f - 8.f * s1);
            fma2(f[q], f[q + 1], f[q], f[q + 1], d / s0, d / s1, c, c);
        }
        reinterpret_cast<float4 *>(p)[8 * k + j] = make_float4(f[0], f[1], f[2], f[3]);
    }
}
MADI_DEV void st_values(__half *p, const Codes2 &u, __half2 cd, int j) {
    const __half2 c = __low2half2(cd), d = __high2half2(cd);
    const __half2 k1032 = __float2half2_rn(1032.f), k16 = __float2half2_rn(0.0625f), km72 = __float2half2_rn(-72.f);
    uint32_t o[4], e[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // elements (0, 4), (1, 5), (2, 6), (3, 7) under the f16 exponent of 1024: 1024 + z and
        // 1024 + 16 z become z - 8 exactly
        const uint32_t v = i ? u.w[0] >> 8 : u.w[0];
        const uint32_t a = (v & 0x000F000Fu) | 0x64006400u, b = (v & 0x00F000F0u) | 0x64006400u;
        o[2 * i] = h2_as_u32(__hfma2(d, __hsub2(as_h2(a), k1032), c));
        o[2 * i + 1] = h2_as_u32(__hfma2(d, __hfma2(as_h2(b), k16, km72), c));
    }
    e[0] = __byte_perm(o[0], o[1], 0x5410);
    e[1] = __byte_perm(o[2], o[3], 0x5410);
    e[2] = __byte_perm(o[0], o[1], 0x7632);
    e[3] = __byte_perm(o[2], o[3], 0x7632);
    reinterpret_cast<uint4 *>(p)[j] = make_uint4(e[0], e[1], e[2], e[3]);
}

// Bound by its writes: 24.2 us for those rows as f32 (140 MB, 5.8 TB/s = 88 % of a copy's rate).
template <typename T>
__global__ void __launch_bounds__(kThr) kv4_load_kernel(const uint8_t *data, long long slot_bytes, long long head_bytes,
                                                        int max_tok, T *k, T *v, long long slot_stride,
                                                        long long row_stride, int rows, const uint32_t *pos,
                                                        const uint32_t *n) {
    constexpr int kB = 2;                                     // rows whose loads are in flight together
    pdl_trigger();
    pdl_wait();
    const int h = blockIdx.y, r0 = (int)blockIdx.x * kRows, s = blockIdx.z;
    int nr = min(kv4_rows(n, s, rows) - r0, kRows);
    const unsigned long long first = (pos ? (unsigned long long)pos[s] : 0ull) + (unsigned)r0;
    if (nr <= 0 || first >= (unsigned long long)max_tok) return;
    const int at0 = (int)first;
    nr = min(nr, max_tok - at0);                              // rows past the cache stay as they were
    const uint8_t *head = data + s * slot_bytes + h * head_bytes;
    const long long dst0 = s * slot_stride + r0 * row_stride + h * kKv4Hd;
    const int j = threadIdx.x & 7, grp = threadIdx.x >> 3, ng = blockDim.x >> 3;
    for (int i = grp; i < nr; i += kB * ng) {
        Codes2 u[kB][2];
        uint32_t cd[kB][2];
#pragma unroll
        for (int b = 0; b < kB; ++b) {
            const uint32_t at = (uint32_t)(at0 + min(i + b * ng, nr - 1));
            const uint8_t *blk = head + (long long)(at / kKv4Blk) * kKv4Block;
            const int off = (int)(at % kKv4Blk);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                u[b][y] = ld_codes(k, blk + y * kKv4Half + off * 32, j);
                cd[b][y] = *reinterpret_cast<const uint32_t *>(blk + y * kKv4Half + kKv4Codes + off * 4);
            }
        }
#pragma unroll
        for (int b = 0; b < kB; ++b) {
            if (i + b * ng >= nr) break;
            const long long dst = dst0 + (i + b * ng) * row_stride;
            st_values(k + dst, u[b][0], as_h2(cd[b][0]), j);
            st_values(v + dst, u[b][1], as_h2(cd[b][1]), j);
        }
    }
}

long long head_bytes(const Kv4Args &a) { return (long long)((a.max_tok + kKv4Blk - 1) / kKv4Blk) * kKv4Block; }

// Threads per CTA: `lanes` per row, at most kThr.
int threads_for(int rows, int lanes) { return rows * lanes >= kThr ? kThr : (rows * lanes + 31) / 32 * 32; }

template <typename T>
cudaError_t store_t(const Kv4Args &a, const T *k, const T *v, int rows, long long slot_stride, long long row_stride,
                    const uint32_t *pos, const uint32_t *n, cudaStream_t st) {
    const long long hb = head_bytes(a);
    const dim3 grid((unsigned)((rows + kRows - 1) / kRows), (unsigned)a.kv_heads, (unsigned)a.slots);
    return launch_k(kv4_store_kernel<T>, grid, threads_for(rows, 4), 0, st, 1, a.data, hb * a.kv_heads, hb, a.max_tok, k, v,
                    slot_stride, row_stride, rows, pos, n);
}
template <typename T>
cudaError_t load_t(const Kv4Args &a, T *k, T *v, int rows, long long slot_stride, long long row_stride,
                   const uint32_t *pos, const uint32_t *n, cudaStream_t st) {
    const long long hb = head_bytes(a);
    const dim3 grid((unsigned)((rows + kRows - 1) / kRows), (unsigned)a.kv_heads, (unsigned)a.slots);
    return launch_k(kv4_load_kernel<T>, grid, threads_for(rows, 8), 0, st, 1, (const uint8_t *)a.data, hb * a.kv_heads, hb,
                    a.max_tok, k, v, slot_stride, row_stride, rows, pos, n);
}

}  // namespace

cudaError_t launch_kv4_store(const Kv4Args &a, const void *k, const void *v, bool f16, int rows, long long slot_stride,
                             long long row_stride, const uint32_t *pos, const uint32_t *n, cudaStream_t st) {
    return f16 ? store_t(a, static_cast<const __half *>(k), static_cast<const __half *>(v), rows, slot_stride, row_stride,
                         pos, n, st)
               : store_t(a, static_cast<const float *>(k), static_cast<const float *>(v), rows, slot_stride, row_stride,
                         pos, n, st);
}

cudaError_t launch_kv4_load(const Kv4Args &a, void *k, void *v, bool f16, int rows, long long slot_stride,
                            long long row_stride, const uint32_t *pos, const uint32_t *n, cudaStream_t st) {
    return f16 ? load_t(a, static_cast<__half *>(k), static_cast<__half *>(v), rows, slot_stride, row_stride, pos, n, st)
               : load_t(a, static_cast<float *>(k), static_cast<float *>(v), rows, slot_stride, row_stride, pos, n, st);
}

}  // namespace madi

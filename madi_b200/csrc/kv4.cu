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
// Both kernels move bytes: eight lanes per group, lane j its elements 8 j .. 8 j + 7 (one
// 16-byte load of f16, two of f32) and code word j.  One CTA takes up to 64 consecutive
// rows of one (slot, head), K and V, so its 32-byte code rows are written as one run.
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include "internal.h"
#include "kv4.cuh"

namespace madi {
namespace {

constexpr int kThr = 256;
constexpr int kRows = 64;      // rows per CTA
constexpr float kLimit = 57344.f;

MADI_DEV void ld8(const float *p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
MADI_DEV void ld8(const __half *p, float (&f)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}

// The least number >= r (r >= 0, far below the largest f16) with 8 significant bits that is
// a multiple of 2^-24.  r is itself rounded up from the exact ratio; rounding up twice
// gives the same as once, since every such number is an f32.
MADI_DEV float step_up(float r) {
    if (r < 7.62939453125e-06f)                          // 2^-17: the multiples of 2^-24 are the coarser grid
        return ceilf(r * 16777216.f) * 5.9604644775390625e-08f;
    return __uint_as_float((__float_as_uint(r) + 0xFFFFu) & 0xFFFF0000u);
}

// n' + 8 of x.  The quotient with the reciprocal is within one of the answer; the two
// comparisons x - c >= (n' -+ 1/2) d settle it exactly: x - c = t + e without error, the
// product (at most 5 by 8 bits) and its difference from t decide by sign, e on equality
// (|e| is below the spacing of that difference).
MADI_DEV uint32_t code_of(float x, float c, float d, float inv) {
    const float t = x - c;
    const float b = t - x;
    const float e = (x - (t - b)) + (-c - b);
    float g = rintf(t * inv);
    const float lo = fmaf(0.5f - g, d, t);               // t - (g - 1/2) d
    const float hi = fmaf(-0.5f - g, d, t);              // t - (g + 1/2) d
    if (lo < 0.f || (lo == 0.f && e < 0.f)) g -= 1.f;
    else if (hi > 0.f || (hi == 0.f && e >= 0.f)) g += 1.f;
    return (uint32_t)((int)g + 8);
}

// Row r's code word j and (c, d) of the K (or V) half at `half` of the blocks at `head`.
MADI_DEV uint32_t *code_word(uint8_t *half, int off, int j) {
    return reinterpret_cast<uint32_t *>(half + off * 32) + j;
}
MADI_DEV uint32_t *cd_word(uint8_t *half, int off) {
    return reinterpret_cast<uint32_t *>(half + kKv4Codes + off * 4);
}

template <typename T>
__global__ void __launch_bounds__(kThr) kv4_store_kernel(uint8_t *__restrict__ data, long long slot_bytes,
                                                         long long head_bytes, int kv_heads, int max_tok,
                                                         const T *__restrict__ k, const T *__restrict__ v,
                                                         long long slot_stride, long long row_stride, int rows,
                                                         const uint32_t *__restrict__ pos,
                                                         const uint32_t *__restrict__ n) {
    pdl_trigger();
    pdl_wait();
    const int h = blockIdx.x % kv_heads, r0 = (int)(blockIdx.x / kv_heads) * kRows, s = blockIdx.y;
    const int nr = min(kv4_rows(n, s, rows) - r0, kRows);     // rows of this CTA
    const unsigned long long at0 = (pos ? (unsigned long long)pos[s] : 0ull) + (unsigned)r0;
    uint8_t *head = data + s * slot_bytes + h * head_bytes;
    const long long src0 = s * slot_stride + r0 * row_stride + h * kKv4Hd;
    const int j = threadIdx.x & 7, grp = threadIdx.x >> 3, ng = blockDim.x >> 3;
    for (int i = grp; i < 2 * nr; i += ng) {                  // nr <= 0: nothing
        const bool is_v = i >= nr;
        const int r = is_v ? i - nr : i;
        float x[8];
        ld8((is_v ? v : k) + src0 + r * row_stride + 8 * j, x);
        float lo = x[0], hi = x[0];
        bool ok = fabsf(x[0]) <= kLimit;
#pragma unroll
        for (int q = 1; q < 8; ++q) {
            lo = fminf(lo, x[q]);
            hi = fmaxf(hi, x[q]);
            ok = ok && fabsf(x[q]) <= kLimit;
        }
        // the eight lanes of a group are active together (i is theirs alone)
        const uint32_t mask = 0xFFu << (threadIdx.x & 24);
#pragma unroll
        for (int o = 4; o; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
        }
        ok = __all_sync(mask, ok);
        const float c = __half2float(__float2half_rn(__fadd_rn(lo, __fmul_rn(__fsub_rn(hi, lo), 8.f / 15.f))));
        float d = step_up(fmaxf(__fsub_ru(c, lo) * 0.125f, __fdiv_ru(__fsub_ru(hi, c), 7.f)));
        if (!ok) d = 0.f;
        uint32_t w = 0x88888888u;
        if (d > 0.f) {
            const float inv = 1.0f / d;
            w = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) w |= code_of(x[q], c, d, inv) << (4 * q);
        }
        const unsigned long long at = at0 + (unsigned)r;
        if (at >= (unsigned long long)max_tok) continue;       // past the cache: dropped
        uint8_t *half = head + (long long)(at / kKv4Blk) * kKv4Block + (is_v ? kKv4Half : 0);
        const int off = (int)(at % kKv4Blk);
        *code_word(half, off, j) = w;
        if (j == 0)
            *cd_word(half, off) = h2_as_u32(__halves2half2(__float2half_rn(ok ? c : CUDART_NAN_F), __float2half_rn(d)));
    }
}

// value = c + d n' rounded once: f32 by one FMA (d n' is exact), f16 by one f16 FMA.
MADI_DEV void st8(float *p, uint32_t w, __half2 cd) {
    const float c = __low2float(cd), d = __high2float(cd);
    float f[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) f[q] = fmaf(d, (float)((int)((w >> (4 * q)) & 15u) - 8), c);
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
MADI_DEV void st8(__half *p, uint32_t w, __half2 cd) {
    const __half2 c = __low2half2(cd), d = __high2half2(cd);
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        // nibbles 2q and 2q + 1 under the f16 exponent of 1024: 1024 + n' + 8, exactly
        const uint32_t b = (w >> (8 * q)) & 0xFFu;
        const uint32_t u = 0x64006400u | (b & 15u) | ((b >> 4) << 16);
        const __half2 z = __hsub2(*reinterpret_cast<const __half2 *>(&u), __float2half2_rn(1032.f));
        o[q] = h2_as_u32(__hfma2(d, z, c));
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename T>
__global__ void __launch_bounds__(kThr) kv4_load_kernel(uint8_t *__restrict__ data, long long slot_bytes,
                                                        long long head_bytes, int kv_heads, int max_tok,
                                                        T *__restrict__ k, T *__restrict__ v, long long slot_stride,
                                                        long long row_stride, int rows,
                                                        const uint32_t *__restrict__ pos,
                                                        const uint32_t *__restrict__ n) {
    pdl_trigger();
    pdl_wait();
    const int h = blockIdx.x % kv_heads, r0 = (int)(blockIdx.x / kv_heads) * kRows, s = blockIdx.y;
    int nr = min(kv4_rows(n, s, rows) - r0, kRows);
    const unsigned long long at0 = (pos ? (unsigned long long)pos[s] : 0ull) + (unsigned)r0;
    if (nr <= 0 || at0 >= (unsigned long long)max_tok) return;
    nr = min(nr, (int)((unsigned long long)max_tok - at0));    // rows past the cache stay as they were
    uint8_t *head = data + s * slot_bytes + h * head_bytes;
    const long long dst0 = s * slot_stride + r0 * row_stride + h * kKv4Hd;
    const int j = threadIdx.x & 7, grp = threadIdx.x >> 3, ng = blockDim.x >> 3;
    for (int i = grp; i < 2 * nr; i += ng) {
        const bool is_v = i >= nr;
        const int r = is_v ? i - nr : i;
        const int at = (int)at0 + r;
        uint8_t *half = head + (long long)(at / kKv4Blk) * kKv4Block + (is_v ? kKv4Half : 0);
        const uint32_t cd = *cd_word(half, at % kKv4Blk);
        st8((is_v ? v : k) + dst0 + r * row_stride + 8 * j, *code_word(half, at % kKv4Blk, j),
            *reinterpret_cast<const __half2 *>(&cd));
    }
}

long long head_bytes(const Kv4Args &a) { return (long long)((a.max_tok + kKv4Blk - 1) / kKv4Blk) * kKv4Block; }

// Threads per CTA: eight per group, K and V of the CTA's rows, at most 256.
int threads_for(int rows) { return rows >= kThr / 16 ? kThr : (rows * 16 + 31) / 32 * 32; }

}  // namespace

cudaError_t launch_kv4_store(const Kv4Args &a, const void *k, const void *v, bool f16, int rows, long long slot_stride,
                             long long row_stride, const uint32_t *pos, const uint32_t *n, cudaStream_t st) {
    const long long hb = head_bytes(a);
    const dim3 grid((unsigned)(a.kv_heads * ((rows + kRows - 1) / kRows)), (unsigned)a.slots);
    if (f16)
        return launch_k(kv4_store_kernel<__half>, grid, threads_for(rows), 0, st, 1, a.data, hb * a.kv_heads, hb,
                        a.kv_heads, a.max_tok, static_cast<const __half *>(k), static_cast<const __half *>(v),
                        slot_stride, row_stride, rows, pos, n);
    return launch_k(kv4_store_kernel<float>, grid, threads_for(rows), 0, st, 1, a.data, hb * a.kv_heads, hb,
                    a.kv_heads, a.max_tok, static_cast<const float *>(k), static_cast<const float *>(v), slot_stride,
                    row_stride, rows, pos, n);
}

cudaError_t launch_kv4_load(const Kv4Args &a, void *k, void *v, bool f16, int rows, long long slot_stride,
                            long long row_stride, const uint32_t *pos, const uint32_t *n, cudaStream_t st) {
    const long long hb = head_bytes(a);
    const dim3 grid((unsigned)(a.kv_heads * ((rows + kRows - 1) / kRows)), (unsigned)a.slots);
    if (f16)
        return launch_k(kv4_load_kernel<__half>, grid, threads_for(rows), 0, st, 1, a.data, hb * a.kv_heads, hb,
                        a.kv_heads, a.max_tok, static_cast<__half *>(k), static_cast<__half *>(v), slot_stride,
                        row_stride, rows, pos, n);
    return launch_k(kv4_load_kernel<float>, grid, threads_for(rows), 0, st, 1, a.data, hb * a.kv_heads, hb, a.kv_heads,
                    a.max_tok, static_cast<float *>(k), static_cast<float *>(v), slot_stride, row_stride, rows, pos, n);
}

}  // namespace madi

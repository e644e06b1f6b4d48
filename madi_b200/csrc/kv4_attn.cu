// kv4_attn.cu -- attention over the 4-bit K/V cache (kv4.cuh).
//
// Query row i of a slot and head h attends keys j < L (kv4_keys):
//     s_j = (q . k_j) / 8 = (d_j (q . n'_j) + c_j sum(q)) / 8
//     out = sum_j p_j v_j,  p = softmax(s);   sum p v = sum (p_j d_j) n'_j + sum p_j c_j
// so a group's two numbers multiply one score and one weight, and the matrix products run
// on the codes themselves.  L = 0 gives a zero row.
//
// Streaming form: one thread-block cluster of ns CTAs per (slot, kv head, tile of query
// columns), a column being one (query row, query head of the kv head).  The slot's blocks
// of 64 keys are dealt to the ns x 4 warps in turn; each warp runs its own ring of bulk
// copies (4608 contiguous bytes a block: nothing is shared between warps, so there is no
// block-wide barrier in the stream) and its own online softmax, and the warps and then
// the cluster's CTAs are joined by log-sum-exp at the end through distributed shared
// memory: no scratch, one launch, a fixed order of sums.
//
// The products are mma.m16n8k16 with f16 operands and f32 sums.  A cache read once per
// token is bound by its bytes, not by the tensor cores, and this shape takes the codes
// straight from their packed form:
//   * a nibble z = n' + 8 kept in place under a mask IS the f16 subnormal z 2^-24 (low nibble
//     of a byte) or z 2^-20 (high nibble): one logic instruction unpacks two codes, and the
//     power of two goes into q (keys) or into the result (values);
//   * the eight columns of an instruction hold four query columns as two f16 numbers each,
//     x = hi + lo with hi on a fixed grid: hi's products and their sums are exact in the tensor
//     core, and lo's are 2^10 times smaller, so f32 queries and outputs lose nothing to
//     f16 operands or to how the tensor core aligns its addends (with hi = f16(x), whose
//     products differ in exponent, f32 results were 2e-5 off in norm);
//   * S is computed as [keys x columns], O as [dims x columns]; the weights turn from
//     the first product's result into the second's operand by one movmatrix a key group.
// Row r of a 16-key tile is key r ^ ((r >> 2) & 1): with this order the word loads of the
// value product (keys 2t and 2t + 1 per lane) touch 32 different banks.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>

#include "internal.h"
#include "kv4.cuh"

namespace cg = cooperative_groups;

namespace madi {
namespace {

constexpr int kWarps = 4;
constexpr int kThr = kWarps * 32;
constexpr int kMaxNs = 16;                     // CTAs of a cluster (above 8: non-portable size)
constexpr int kMaxStages = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kUp24 = 16777216.f;            // 2^24

MADI_DEV void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// D += A B, 16 x 8 x 16, f16 operands, f32 sums.
MADI_DEV void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
MADI_DEV uint32_t movm_trans(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
MADI_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}
// 1.5 x 2^23 grid steps: adding and subtracting it rounds to the grid.
constexpr float kGrid8 = 12582912.f * 8.f, kGrid4 = 12582912.f * 4.f;
// A weight 0 <= x < 2^15 as {hi, lo}: hi the nearest f16, on the grid of 4 where f16 is finer;
// lo the rest, at most 2^-12 of x or 2.
MADI_DEV uint32_t split_weight(float x) {
    const float hi = __fsub_rn(__fadd_rn(__half2float(__float2half_rn(x)), kGrid4), kGrid4);
    return h2_as_u32(__floats2half2_rn(hi, x - hi));
}
MADI_DEV void ld16(const float *p, float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 v = reinterpret_cast<const float4 *>(p)[i];
        f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
    }
}
MADI_DEV void ld16(const __half *p, float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 u = reinterpret_cast<const uint4 *>(p)[i];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
            f[8 * i + 2 * k] = v.x;
            f[8 * i + 2 * k + 1] = v.y;
        }
    }
}
MADI_DEV void stf(float *p, float v) { *p = v; }
MADI_DEV void stf(__half *p, float v) { *p = __float2half_rn(v); }
// 2^e for -126 <= e <= 127.
MADI_DEV float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// floor(log2 x) of a positive normal f32.
MADI_DEV int ilog2f_(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }

// One warp's partial result for a column: running max (base 2), sum, and unnormalised output.
constexpr int kPart = 2 + kKv4Hd;

// NT groups of four query columns per CTA.
template <int NT, typename T>
__global__ void __launch_bounds__(kThr) kv4_stream_kernel(const Kv4AttnArgs a, long long slot_bytes, long long head_bytes,
                                                          int group, int tiles, int ns, int stages) {
    constexpr int kCols = 4 * NT;
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    __shared__ __align__(8) uint64_t full[kWarps][kMaxStages];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % ns;
    const int tile = (int)(blockIdx.x / ns) % tiles, kvh = (int)(blockIdx.x / ns) / tiles, s = blockIdx.y;
    uint8_t *ring = kv4_smem + (size_t)warp * stages * kKv4Block;
    pdl_trigger();
    if (lane == 0)
        for (int i = 0; i < stages; ++i) mbar_init(&full[warp][i], 1);
    if (tid == 0) abort_flag = 0;
    fence_mbar_init();
    pdl_wait();
    __syncthreads();

    // this CTA's columns: col0 .. col0 + ncol - 1; column x is row x / group, head kvh * group + x % group
    const int total = kv4_rows(a.n, s, a.rows) * group;
    const int col0 = tile * kCols, ncol = min(total - col0, kCols);
    if (ncol <= 0) return;                                  // padding only (the whole cluster leaves)
    const int lmax = kv4_keys(a.pos, a.lens, s, (col0 + ncol - 1) / group, a.c.max_tok);
    const int lmin = kv4_keys(a.pos, a.lens, s, col0 / group, a.c.max_tok);
    const int nblk = (lmax + kKv4Blk - 1) / kKv4Blk, units = ns * kWarps, unit = rank * kWarps + warp;
    const int mine = nblk > unit ? (nblk - unit + units - 1) / units : 0;      // blocks unit, unit + units, ...
    const uint8_t *src = a.c.data + s * slot_bytes + kvh * head_bytes;
    auto issue = [&](int i) {
        const int st = i % stages;
        mbar_arrive_expect_tx(&full[warp][st], kKv4Block);
        bulk_load(ring + st * kKv4Block, src + (long long)(unit + (long long)i * units) * kKv4Block, kKv4Block,
                  &full[warp][st]);
    };
    if (lane == 0)
        for (int i = 0; i < min(mine, stages); ++i) issue(i);
    if (ns > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");

    // Per lane: column 4 nt + t.  The query in base 2 and the softmax scale, times the power
    // of two 2^e that brings its largest element into [2^13, 2^14), is split on a fixed grid: hi
    // a multiple of 8 (11 bits; even columns of the product), lo the rest (odd columns).  hi's
    // products with the codes are then whole multiples of 8 that stay below 2^24 x 8, so the
    // tensor core's sum of them is exact, whatever it does to addends of different size, and
    // lo's, at most 4 each, round 2^11 times finer than q.  Starting the sums from -8 sum(hi) and
    // -8 sum(lo) turns z = n' + 8 into n'.  Lanes with the same g hold column g's 16 dims of
    // their t.
    uint32_t qb[NT][4][2];
    float qsum[NT], qinv[NT], s0[NT][2];
    int len[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int col = 4 * nt + (g >> 1);                  // the column whose product operand this lane builds
        float f[16], mx = 0.f, sum = 0.f;
        if (col < ncol) {
            const int x = col0 + col, i = x / group, h = kvh * group + x % group;
            ld16(static_cast<const T *>(a.q) + s * a.q_slot + i * a.q_row + h * kKv4Hd + 16 * t, f);
#pragma unroll
            for (int d = 0; d < 16; ++d) {
                f[d] *= 0.125f * kLog2e;
                mx = fmaxf(mx, fabsf(f[d]));
                sum += f[d];
            }
        } else {
#pragma unroll
            for (int d = 0; d < 16; ++d) f[d] = 0.f;
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = mx > 0.f ? min(max(13 - ilog2f_(mx), -100), 100) : 0;
        const float up = pow2i(e);
        float part = 0.f;
#pragma unroll
        for (int d = 0; d < 16; ++d) {
            const float y = f[d] * up, hi = __fsub_rn(__fadd_rn(y, kGrid8), kGrid8);
            f[d] = (g & 1) ? y - hi : hi;
            part += f[d];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        part += __shfl_xor_sync(0xffffffffu, part, 1);
        part += __shfl_xor_sync(0xffffffffu, part, 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // the code operand of step j holds dims b, b + 4 and b + 2, b + 6 (of 16 t ..); its
            // high nibbles (odd j) carry 2^-20, not 2^-24
            const int b = 8 * (j >> 1) + (j & 1);
            const float sc = (j & 1) ? 0.0625f : 1.f;
            qb[nt][j][0] = h2_as_u32(__floats2half2_rn(f[b] * sc, f[b + 4] * sc));
            qb[nt][j][1] = h2_as_u32(__floats2half2_rn(f[b + 2] * sc, f[b + 6] * sc));
        }
        qsum[nt] = __shfl_sync(0xffffffffu, sum, 8 * t);
        qinv[nt] = __shfl_sync(0xffffffffu, pow2i(-e) * kUp24, 8 * t);
        s0[nt][0] = __shfl_sync(0xffffffffu, part, 8 * t) * (-8.f / kUp24);
        s0[nt][1] = __shfl_sync(0xffffffffu, part, 8 * t + 4) * (-8.f / kUp24);
        const int mycol = 4 * nt + t;
        len[nt] = mycol < ncol ? kv4_keys(a.pos, a.lens, s, (col0 + mycol) / group, a.c.max_tok) : 0;
    }

    float m[NT], l[NT], oc[NT], o[NT][4][4], tot[NT][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -CUDART_INF_F;
        l[nt] = oc[nt] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nt][i >> 2][i & 3] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) tot[nt][i] = 0.f;
    }
    auto flush = [&](int nt, float f) {                     // the accumulators' columns 2t, 2t + 1 are this lane's column t
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tot[nt][2 * i] = (tot[nt][2 * i] + (o[nt][i][0] + o[nt][i][1])) * f;
            tot[nt][2 * i + 1] = (tot[nt][2 * i + 1] + (o[nt][i][2] + o[nt][i][3])) * f;
            o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
    };
    // The weights p d enter the second product times 2^we, with d's largest exponent so far
    // brought to 14.  hi is a multiple of 4, so sums of hi n' are exact up to 2^26 = 256 keys x 8
    // x 2^15; lo, at most 2^-12 of the weight (or 2 of 2^15), leaves no weight more than 2^-23
    // of itself (or 2^-27 of the largest) off.  After every 256 keys, and when the scale moves,
    // the products' sums are added to f32 totals and start anew: a total that had been scaled by
    // something else than its grid would be cut to the grid by the next product.
    float dcap = 0.f;                                       // largest d the scale allows for
    int we = 0, since = 0;                                  // blocks since the sums were flushed
    const int kr = g ^ ((g >> 2) & 1);                      // key of row g in a 16-key tile
    const int kv0 = 2 * t ^ ((t >> 1) & 1), kv1 = (2 * t + 1) ^ ((t >> 1) & 1);     // keys of rows 2t, 2t + 1

    bool alive = true;
    int ib = 0;
    for (; ib < mine; ++ib) {
        const int st = ib % stages;
        if (!warp_wait_all(&full[warp][st], (uint32_t)(ib / stages) & 1u, &abort_flag, a.dev_err)) {
            alive = false;
            break;
        }
        const uint8_t *kb = ring + st * kKv4Block, *vb = kb + kKv4Half;
        const int key0 = (unit + ib * units) * kKv4Blk;     // fits: nblk * 64 <= 2^30 + 63
        const bool whole = key0 + kKv4Blk <= lmin;          // every column attends every key of the block
        // ------------------------------------------------ scores
        float sc[NT][8];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            const uint2 wa = *reinterpret_cast<const uint2 *>(kb + (16 * kt + kr) * 32 + 8 * t);
            const uint2 wb = *reinterpret_cast<const uint2 *>(kb + (16 * kt + 8 + kr) * 32 + 8 * t);
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                acc[nt][0] = acc[nt][2] = s0[nt][0];
                acc[nt][1] = acc[nt][3] = s0[nt][1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t mask = (j & 1) ? 0x00F000F0u : 0x000F000Fu;
                const uint32_t u = j < 2 ? wa.x : wa.y, w = j < 2 ? wb.x : wb.y;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma16816(acc[nt], u & mask, w & mask, (u >> 8) & mask, (w >> 8) & mask, qb[nt][j][0], qb[nt][j][1]);
            }
            const float2 pa = __half22float2(*reinterpret_cast<const __half2 *>(kb + kKv4Codes + (16 * kt + kr) * 4));
            const float2 pb = __half22float2(*reinterpret_cast<const __half2 *>(kb + kKv4Codes + (16 * kt + 8 + kr) * 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                sc[nt][2 * kt] = fmaf(pa.y, (acc[nt][0] + acc[nt][1]) * qinv[nt], pa.x * qsum[nt]);
                sc[nt][2 * kt + 1] = fmaf(pb.y, (acc[nt][2] + acc[nt][3]) * qinv[nt], pb.x * qsum[nt]);
            }
        }
        // ------------------------------------------------ weights
        float dv[8], cv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 p = __half22float2(
                *reinterpret_cast<const __half2 *>(vb + kKv4Codes + (16 * (i >> 1) + 8 * (i & 1) + kr) * 4));
            cv[i] = p.x;
            dv[i] = p.y;
        }
        if (!whole) {
            // masked keys score -inf; rows behind the last key may hold anything, so their c and
            // d are not used at all
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = key0 + 16 * (i >> 1) + 8 * (i & 1) + kr;
                if (key >= lmax) cv[i] = dv[i] = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (key >= len[nt]) sc[nt][i] = -CUDART_INF_F;
            }
        }
        float dm = dv[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) dm = fmaxf(dm, dv[i]);
        bool grow = dm > dcap;
        float mx[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            mx[nt] = sc[nt][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) mx[nt] = fmaxf(mx[nt], sc[nt][i]);
            grow = grow || mx[nt] > m[nt];
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, x));
            float ds = 1.f;
            if (dm > dcap) {
                const int w2 = 14 - ilog2f_(dm);            // d >= 2^-24, a normal f32
                ds = dcap > 0.f ? pow2i(max(w2 - we, -126)) : 1.f;
                we = w2;
                dcap = pow2i(15 - we) * 0.99609375f;        // the largest 8-bit number below 2^(15 - we)
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx[nt] = fmaxf(mx[nt], __shfl_xor_sync(0xffffffffu, mx[nt], x));
                const float mn = fmaxf(m[nt], mx[nt]);
                const float al = mn == m[nt] ? 1.f : ex2_approx(m[nt] - mn);
                m[nt] = mn;
                l[nt] *= al;
                oc[nt] *= al;
                flush(nt, al * ds);
            }
            since = 0;
        } else if (++since == 4) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) flush(nt, 1.f);
            since = 0;
        }
        const float wscale = pow2i(we);
        uint32_t pw[NT][8];                                 // p d 2^we, split
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float mref = m[nt] == -CUDART_INF_F ? 0.f : m[nt];       // no key yet: every score is -inf
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = ex2_approx(sc[nt][i] - mref);
                l[nt] += p;
                // a masked key's weight is exactly 0, but its c may be NaN for this column only
                oc[nt] = (whole || sc[nt][i] != -CUDART_INF_F) ? fmaf(p, cv[i], oc[nt]) : oc[nt];
                pw[nt][i] = split_weight(p * dv[i] * wscale);
            }
        }
        // ------------------------------------------------ O += V^T p, on z - 8
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            const uint8_t *vr = vb + (16 * kt) * 32 + 4 * g;
            const uint32_t w0 = *reinterpret_cast<const uint32_t *>(vr + kv0 * 32);
            const uint32_t w1 = *reinterpret_cast<const uint32_t *>(vr + kv1 * 32);
            const uint32_t w2 = *reinterpret_cast<const uint32_t *>(vr + (kv0 + 8) * 32);
            const uint32_t w3 = *reinterpret_cast<const uint32_t *>(vr + (kv1 + 8) * 32);
            // pairs of keys side by side: dims 8g .. 8g+3 (x) and 8g+4 .. 8g+7 (y)
            const uint32_t xa = prmt(w0, w1, 0x5410), ya = prmt(w0, w1, 0x7632);
            const uint32_t xb = prmt(w2, w3, 0x5410), yb = prmt(w2, w3, 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t b0 = movm_trans(pw[nt][2 * kt]), b1 = movm_trans(pw[nt][2 * kt + 1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t mask = (i & 1) ? 0x00F000F0u : 0x000F000Fu;
                    const uint32_t u = i < 2 ? xa : ya, w = i < 2 ? xb : yb;
                    // -8 of every code first: sums of z alone would grow with the weights and
                    // then cancel
                    const uint32_t mid = (i & 1) ? 0x80808080u : 0x80088008u;
                    mma16816(o[nt][i], mid, mid, mid, mid, b0, b1);
                    mma16816(o[nt][i], u & mask, (u >> 8) & mask, w & mask, (w >> 8) & mask, b0, b1);
                }
            }
        }
        __syncwarp();                                       // the stage's last reads, before it is filled again
        if (lane == 0 && ib + stages < mine) issue(ib + stages);
    }

    // ------------------------------------------------ this warp's (m, l, o) per column
    // The ring is free: every copy issued has landed (after an expired wait, the copies still
    // in flight are waited for first, with the same bound).
    if (!alive && lane == 0)
        for (int i = ib; i < min(mine, ib + stages); ++i) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&full[warp][i % stages], (uint32_t)(i / stages) & 1u))
                if (clock64() - t0 > kWaitBudgetCycles) break;
        }
    __syncwarp();
    float *wp = reinterpret_cast<float *>(ring);            // [kCols][kPart]
    const float back = pow2i(-we) * kUp24;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], x);
            oc[nt] += __shfl_xor_sync(0xffffffffu, oc[nt], x);
        }
        flush(nt, 1.f);
        float *p = wp + (4 * nt + t) * kPart;
        if (g == 0) {
            p[0] = alive ? m[nt] : -CUDART_INF_F;
            p[1] = alive ? l[nt] : 0.f;
        }
        // accumulator i: dims 8g + {0, 2}, {1, 3}, {4, 6}, {5, 7}; odd ones in units of 2^-20
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float b = (i & 1) ? back * 0.0625f : back;
            const int d = 8 * g + 4 * (i >> 1) + (i & 1);
            p[2 + d] = fmaf(tot[nt][2 * i], b, oc[nt]);
            p[2 + d + 2] = fmaf(tot[nt][2 * i + 1], b, oc[nt]);
        }
    }
    __syncthreads();

    // ------------------------------------------------ join the warps, then the cluster
    // Column x's partials of all CTAs meet in CTA x % ns, at recv[x / ns][rank].
    float *recv = reinterpret_cast<float *>(kv4_smem + (size_t)kWarps * stages * kKv4Block);
    if (ns > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
    for (int x = tid; x < ncol * kKv4Hd; x += kThr) {
        const int col = x / kKv4Hd, d = x % kKv4Hd;
        float mm = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            mm = fmaxf(mm, reinterpret_cast<const float *>(kv4_smem + (size_t)w * stages * kKv4Block)[col * kPart]);
        const float ref = mm == -CUDART_INF_F ? 0.f : mm;
        float ll = 0.f, oo = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float *p = reinterpret_cast<const float *>(kv4_smem + (size_t)w * stages * kKv4Block) + col * kPart;
            const float f = ex2_approx(p[0] - ref);
            ll = fmaf(p[1], f, ll);
            oo = fmaf(p[2 + d], f, oo);
        }
        if (ns > 1) {
            float *to = cg::this_cluster().map_shared_rank(recv, col % ns) + ((col / ns) * ns + rank) * kPart;
            to[2 + d] = oo;
            if (d == 0) {
                to[0] = mm;
                to[1] = ll;
            }
        } else {
            const int q = col0 + col;
            stf(static_cast<T *>(a.out) + s * a.o_slot + (q / group) * a.o_row + (kvh * group + q % group) * kKv4Hd + d,
                ll == 0.f ? 0.f : oo / ll);
        }
    }
    if (ns == 1) return;
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    for (int x = tid; x < (ncol - rank + ns - 1) / ns * kKv4Hd; x += kThr) {
        const int col = rank + x / kKv4Hd * ns, d = x % kKv4Hd;
        const float *p = recv + (x / kKv4Hd) * ns * kPart;
        float mm = -CUDART_INF_F;
        for (int r = 0; r < ns; ++r) mm = fmaxf(mm, p[r * kPart]);
        const float ref = mm == -CUDART_INF_F ? 0.f : mm;
        float ll = 0.f, oo = 0.f;
        for (int r = 0; r < ns; ++r) {
            const float f = ex2_approx(p[r * kPart] - ref);
            ll = fmaf(p[r * kPart + 1], f, ll);
            oo = fmaf(p[r * kPart + 2 + d], f, oo);
        }
        const int q = col0 + col;
        stf(static_cast<T *>(a.out) + s * a.o_slot + (q / group) * a.o_row + (kvh * group + q % group) * kKv4Hd + d,
            ll == 0.f ? 0.f : oo / ll);
    }
}

template <int NT, typename T>
cudaError_t launch_stream(const Kv4AttnArgs &a, cudaStream_t st) {
    auto fn = kv4_stream_kernel<NT, T>;
    const int group = a.heads / a.c.kv_heads;
    const long long cols = (long long)a.rows * group;
    const long long tiles = (cols + 4 * NT - 1) / (4 * NT);
    const int nblk = (a.c.max_tok + kKv4Blk - 1) / kKv4Blk;
    const long long hb = (long long)nblk * kKv4Block;
    const long long pairs = tiles * a.c.kv_heads * a.c.slots;
    constexpr size_t kMaxSmem = (size_t)kWarps * kMaxStages * kKv4Block + (size_t)(4 * NT + kMaxNs) * kPart * sizeof(float);
    static int max_ns = 1;                               // largest power of two the device schedules
    static std::once_flag once;
    static cudaError_t once_status;
    if (cudaError_t e = run_once(once, once_status, [&] {
            cudaError_t e1 = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
            if (e1 == cudaSuccess) e1 = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = kMaxNs;
            cfg.blockDim = kThr;
            cfg.dynamicSmemBytes = kMaxSmem;
            int most = 0;
            if (e1 == cudaSuccess) e1 = cudaOccupancyMaxPotentialClusterSize(&most, fn, &cfg);
            while (max_ns * 2 <= std::min(most, kMaxNs)) max_ns *= 2;
            return e1;
        }))
        return e;
    // Cluster size: split the keys while that gives CTAs to idle SMs and leaves each warp two blocks.
    int ns = 1;
    while (ns < max_ns && pairs * ns < 4LL * num_sms() && nblk >= 2 * kWarps * 2 * ns) ns *= 2;
    const int per_warp = (nblk + ns * kWarps - 1) / (ns * kWarps);
    const int stages = std::max(1, std::min(per_warp, kMaxStages));
    const size_t smem = (size_t)kWarps * stages * kKv4Block +
                        (ns > 1 ? (size_t)((4 * NT + ns - 1) / ns) * ns * kPart * sizeof(float) : 0);
    if (tiles * a.c.kv_heads * ns > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_k(fn, dim3((unsigned)(tiles * a.c.kv_heads * ns), (unsigned)a.c.slots), kThr, smem, st, ns, a,
                    hb * a.c.kv_heads, hb, group, (int)tiles, ns, stages);
}

}  // namespace

cudaError_t launch_kv4_attn(const Kv4AttnArgs &a, bool f16, cudaStream_t st) {
    const long long cols = (long long)a.rows * (a.heads / a.c.kv_heads);
    if (f16 && cols >= 33) return launch_kv4_flash(a, st);
    if (f16)
        return cols <= 4 ? launch_stream<1, __half>(a, st)
                         : cols <= 8 ? launch_stream<2, __half>(a, st) : launch_stream<4, __half>(a, st);
    return cols <= 4 ? launch_stream<1, float>(a, st)
                     : cols <= 8 ? launch_stream<2, float>(a, st) : launch_stream<4, float>(a, st);
}

}  // namespace madi

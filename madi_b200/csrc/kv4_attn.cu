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
// of 64 keys are dealt to the cluster's warps in turn; each warp runs its own ring of bulk
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
//     x = hi + lo.  The tensor core aligns a subnormal as if it were a normal number, and cuts
//     there: with hi = f16(x), whose products differ in exponent, f32 results were 2e-5 off in
//     norm.  So queries (and the weights of f16 outputs) have hi on a fixed grid, where its
//     products and their sums are exact, and lo's are 2^10 times smaller.  A query's elements may
//     share a grid: their products add up to one score.  The weights of f32 outputs may not: keys
//     behind a dominant one whose value is small make up the result with weights of any size (on a
//     grid it was up to 7e-5 off in norm).  There hi is f16(x), and the values' codes become normal
//     numbers n' by one more instruction a pair (8 slots x 20 heads x 1500 keys 8.2 -> 8.8 us);
//   * S is computed as [keys x columns], O as [dims x columns]; the weights turn from
//     the first product's result into the second's operand by one movmatrix a key group.
//   * ldmatrix brings the codes, as 16-bit elements, straight into the operands' places; its
//     transposing form pairs the values of neighbouring keys.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "internal.h"
#include "kv4.cuh"

namespace cg = cooperative_groups;

namespace madi {
namespace {

constexpr int kMaxNs = 16;                     // CTAs of a cluster (above 8: non-portable size)
constexpr int kMaxStages = 2;                 // a second block in flight; more cost resident warps
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
// Four 8 x 8 matrices of 16-bit elements; lanes 8 i .. 8 i + 7 give the row addresses of matrix i.  Lane
// (g, t) gets elements 2t, 2t + 1 of row g, or (trans) element g of rows 2t, 2t + 1.
MADI_DEV void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
MADI_DEV void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
MADI_DEV uint32_t movm_trans(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
MADI_DEV uint32_t cluster_id_x() {
    uint32_t r;
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
// 1.5 x 2^23 grid steps: adding and subtracting it rounds to the grid.
constexpr float kGrid8 = 12582912.f * 8.f, kGrid4 = 12582912.f * 4.f;
// Exponent that the largest d of the keys so far is brought to in the weights' scale.
template <typename T> constexpr int kTop = sizeof(T) == 4 ? 14 : 12;
// Two weights x < 2^(kTop + 1) as {hi, lo} f16 pairs.  f32 outputs: hi is the nearest f16 and lo the rest
// times 2^11, so that x keeps 22 bits down to 2^-28 of the largest weight (lo as it is, on the grid of
// the f16 form, left weights below 2^-12 of it 11 bits, and some of their results 2^-14 off).  f16
// outputs: hi is a multiple of 4, which below 2^13 is an f16, and lo, at most 2, leaves 2^-24 of
// the largest weight or 2^-12 of x off.
constexpr float kLoUp = 2048.f;
template <typename T>
MADI_DEV void split_weights(float x0, float x1, uint32_t &w0, uint32_t &w1) {
    float l0, l1;
    if constexpr (sizeof(T) == 4) {
        const __half2 h = __floats2half2_rn(x0, x1);
        const float2 hf = __half22float2(h);
        mul2(l0, l1, x0, x1, kLoUp, kLoUp);
        fma2(l0, l1, hf.x, hf.y, -kLoUp, -kLoUp, l0, l1);
        const uint32_t hi = h2_as_u32(h), lo = h2_as_u32(__floats2half2_rn(l0, l1));
        w0 = __byte_perm(hi, lo, 0x5410);
        w1 = __byte_perm(hi, lo, 0x7632);
    } else {
        float h0, h1;
        add2(h0, h1, x0, x1, kGrid4, kGrid4);
        add2(h0, h1, h0, h1, -kGrid4, -kGrid4);
        fma2(l0, l1, h0, h1, -1.f, -1.f, x0, x1);
        w0 = h2_as_u32(__floats2half2_rn(h0, l0));
        w1 = h2_as_u32(__floats2half2_rn(h1, l1));
    }
}
// Two codes of a word under the mask of tile i as f16 numbers: n' of the low nibbles (even i), 16 n' of
// the high ones.
MADI_DEV uint32_t codes_f16(uint32_t w, int i) {
    const uint32_t v = (w & ((i & 1) ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;     // 1024 + z, 1024 + 16 z
    return h2_as_u32(__hsub2(*reinterpret_cast<const __half2 *>(&v), __float2half2_rn((i & 1) ? 1152.f : 1032.f)));
}
// Elements p[0 .. 7] and p[32 .. 39].
MADI_DEV void ld16(const float *p, float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 v = reinterpret_cast<const float4 *>(p + 32 * (i >> 1))[i & 1];
        f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
    }
}
MADI_DEV void ld16(const __half *p, float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p + 32 * i);
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
// floor(log2 x) of a positive normal f32.
MADI_DEV int ilog2f_(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }

// One warp's partial result for a column: running max (base 2), sum, and unnormalised output.
constexpr int kPart = 2 + kKv4Hd;

// NT groups of four query columns per CTA of W warps.  115 to 185 registers; with four groups 255, and 8 to 60 bytes
// (f32) or some 300 to 380 (f16) spilled.
template <int NT, int W, typename T>
__global__ void __launch_bounds__(32 * W, NT > 1 ? 1 : 2) kv4_stream_kernel(const Kv4AttnArgs a, long long slot_bytes,
                                                            long long head_bytes, int group, int ns, int stages) {
    constexpr int kCols = 4 * NT, kThr = 32 * W;
    constexpr bool kF32 = sizeof(T) == 4;
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    __shared__ __align__(8) uint64_t full[W][kMaxStages];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rank = (int)cluster_ctarank(), tile = (int)cluster_id_x(), kvh = blockIdx.y, s = blockIdx.z;
    uint8_t *ring = kv4_smem + (size_t)warp * stages * kKv4Block;
    pdl_trigger();
    if (lane == 0)
        for (int i = 0; i < stages; ++i) mbar_init(&full[warp][i], 1);
    if (tid == 0) abort_flag = 0;
    fence_mbar_init();
    pdl_wait();
    __syncthreads();

    // this CTA's columns: col0 .. col0 + ncol - 1; column x is row x / group, head kvh * group + x % group
    const bool one = a.rows == 1;
    auto row_of = [&](int x) { return one ? 0 : x / group; };
    const int total = kv4_rows(a.n, s, a.rows) * group;
    const int col0 = tile * kCols, ncol = min(total - col0, kCols);
    if (ncol <= 0) return;                                  // padding only (the whole cluster leaves)
    const int lmax = kv4_keys(a.pos, a.lens, s, row_of(col0 + ncol - 1), a.c.max_tok);
    const int lmin = one ? lmax : kv4_keys(a.pos, a.lens, s, row_of(col0), a.c.max_tok);
    const int nblk = (lmax + kKv4Blk - 1) / kKv4Blk, units = ns * W, unit = rank * W + warp;
    const uint8_t *src = a.c.data + s * slot_bytes + kvh * head_bytes;
    auto issue = [&](int blk, int st) {
        mbar_arrive_expect_tx(&full[warp][st], kKv4Block);
        bulk_load(ring + st * kKv4Block, src + (long long)blk * kKv4Block, kKv4Block, &full[warp][st]);
    };
    if (lane == 0)                                          // this warp's blocks: unit, unit + units, ...
        for (int i = 0, blk = unit; i < stages && blk < nblk; ++i, blk += units) issue(blk, i);
    if (ns > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");

    // Per lane: column 4 nt + t.  The query times the power of two 2^e that brings its largest
    // element into [2^13, 2^14).  f32 queries (in base 2 and the softmax scale) are split on a
    // fixed grid: hi a multiple of 8 (11 bits; even columns of the product), lo the rest (odd
    // columns).  hi's products with the codes are then whole multiples of 8 that stay below
    // 2^24 x 8, so the tensor core's sum of them is exact, whatever it does to addends of
    // different size, and lo's, at most 4 each, round 2^11 times finer than q.  f16 queries are
    // hi as they are.  Starting the sums from -8 sum(hi) and -8 sum(lo) turns z = n' + 8 into n'.
    // Lanes with the same g hold column g's dims 8t .. 8t + 7 and 32 + 8t .. 32 + 8t + 7 of their t.
    uint32_t qb[NT][4][2];
    float qsum[NT], qinv[NT], s0[NT][2];
    int len[NT];
    const bool idle = unit >= nblk;                         // no block for this warp
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (idle) break;
        const int col = 4 * nt + (g >> 1);                  // the column whose product operand this lane builds
        float f[16], mx = 0.f, sum = 0.f;
#pragma unroll
        for (int d = 0; d < 16; ++d) f[d] = 0.f;
        if (col < ncol) {
            const int x = col0 + col, i = row_of(x), h = kvh * group + x - i * group;
            ld16(static_cast<const T *>(a.q) + s * a.q_slot + i * a.q_row + h * kKv4Hd + 8 * t, f);
        }
#pragma unroll
        for (int d = 0; d < 16; ++d) {
            if (kF32) f[d] *= 0.125f * kLog2e;
            mx = fmaxf(mx, fabsf(f[d]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = mx > 0.f ? min(max(13 - ilog2f_(mx), -100), 100) : 0;
        const float up = pow2i(e);
        float part = 0.f;
#pragma unroll
        for (int d = 0; d < 16; ++d) {
            const float y = f[d] * up;
            sum += y;
            if (kF32) {
                const float hi = __fsub_rn(__fadd_rn(y, kGrid8), kGrid8);
                f[d] = (g & 1) ? y - hi : hi;
                part += f[d];
            } else {
                f[d] = (g & 1) ? 0.f : y;
            }
        }
        if (!kF32) part = (g & 1) ? 0.f : sum;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        part += __shfl_xor_sync(0xffffffffu, part, 1);
        part += __shfl_xor_sync(0xffffffffu, part, 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // the code operand of step j holds dims b, b + 4 and b + 2, b + 6 (of the lane's 16); its
            // high nibbles (odd j) carry 2^-20, not 2^-24
            const int b = 8 * (j >> 1) + (j & 1);
            const float sc = (j & 1) ? 0.0625f : 1.f;
            qb[nt][j][0] = h2_as_u32(__floats2half2_rn(f[b] * sc, f[b + 4] * sc));
            qb[nt][j][1] = h2_as_u32(__floats2half2_rn(f[b + 2] * sc, f[b + 6] * sc));
        }
        // scores are kept in units of qinv: the products' sums as they are, c sum(q) in their unit
        qinv[nt] = __shfl_sync(0xffffffffu, pow2i(-e) * (kF32 ? kUp24 : kUp24 * 0.125f * kLog2e), 8 * t);
        qsum[nt] = __shfl_sync(0xffffffffu, sum * (1.f / kUp24), 8 * t);
        s0[nt][0] = __shfl_sync(0xffffffffu, part, 8 * t) * (-8.f / kUp24);
        s0[nt][1] = __shfl_sync(0xffffffffu, part, 8 * t + 4) * (-8.f / kUp24);
        const int mycol = 4 * nt + t;
        len[nt] = mycol < ncol ? kv4_keys(a.pos, a.lens, s, row_of(col0 + mycol), a.c.max_tok) : 0;
    }

    // m: running maximum in score units; l, oc: this lane's sums of p and p c over even and odd keys
    float m[NT], l[NT][2], oc[NT][2], o[NT][4][4], o8[NT][4], tot[NT][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -CUDART_INF_F;
        l[nt][0] = l[nt][1] = oc[nt][0] = oc[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nt][i >> 2][i & 3] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o8[nt][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) tot[nt][i] = 0.f;
    }
    // o: sums of z w (w the weights' parts), o8: of 8 w, in every row; z - 8 = n'.  The accumulators'
    // columns 2t, 2t + 1 are this lane's column t; odd tiles are in units of 2^-20.  f32: sums of n' w,
    // odd tiles of 16 n' w.
    auto flush = [&](int nt, float f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = (i & 1) ? -16.f : -1.f;
            float x, y;
            if constexpr (kF32) {
                x = fmaf(o[nt][i][1], 1.f / kLoUp, o[nt][i][0]);
                y = fmaf(o[nt][i][3], 1.f / kLoUp, o[nt][i][2]);
            } else {
                x = fmaf(e, o8[nt][0], o[nt][i][0]) + fmaf(e, o8[nt][1], o[nt][i][1]);
                y = fmaf(e, o8[nt][0], o[nt][i][2]) + fmaf(e, o8[nt][1], o[nt][i][3]);
            }
            tot[nt][2 * i] = (tot[nt][2 * i] + x) * f;
            tot[nt][2 * i + 1] = (tot[nt][2 * i + 1] + y) * f;
            o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
        o8[nt][0] = o8[nt][1] = o8[nt][2] = o8[nt][3] = 0.f;
    };
    // The weights p d enter the second product times 2^we, with d's largest exponent so far
    // brought to kTop.  f16 outputs: the codes are the subnormals z 2^-24, whose products the tensor core
    // aligns as if they were 2^10 larger and cuts there; hi is a multiple of 4 so that the sums of z hi are
    // exact all the same, up to 2^26 = 15 x 2^13 x 546 keys.  f32 outputs: hi has all its bits, so the codes
    // come as the normal numbers n', whose sums lose no more than f32 ones.  After kFlush blocks of 64
    // keys, and when the scale moves, the products' sums are added to f32 totals and start anew: a total that
    // had been scaled by something else than its grid would be cut to the grid by the next product.
    constexpr int kFlush = kF32 ? 2 : 4;
    float dcap = 0.f, wscale = 1.f;                         // largest d the scale allows for; 2^we
    int we = 0, since = 0;                                  // since: blocks since the sums were flushed
    // the rows a lane points ldmatrix at: tile rows 0 .. 7, 8 .. 15 (first 16 bytes), and again (last 16)
    const uint32_t rows_at = smem_u32(ring) + (lane & 15) * 32 + (lane >> 4) * 16;

    bool alive = true;
    int st = 0, blk = unit;
    uint32_t phase = 0;
    for (; blk < nblk; blk += units) {
        if (!warp_wait_all(&full[warp][st], phase, &abort_flag, a.dev_err)) {
            alive = false;
            break;
        }
        const uint8_t *kb = ring + st * kKv4Block, *vb = kb + kKv4Half;
        const int key0 = blk * kKv4Blk;                     // at most 2^30 + 63
        const bool whole = key0 + kKv4Blk <= lmin;          // every column attends every key of the block
        // ------------------------------------------------ scores (rows g and g + 8 of each tile)
        float sc[NT][4][2];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t kw[4];                                 // row g, row g + 8: words t; words 4 + t
            ldmatrix4(kw, rows_at + st * kKv4Block + kt * 512);
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                acc[nt][0] = acc[nt][2] = s0[nt][0];
                acc[nt][1] = acc[nt][3] = kF32 ? s0[nt][1] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t mask = (j & 1) ? 0x00F000F0u : 0x000F000Fu;
                const uint32_t u = kw[j & 2], w = kw[(j & 2) + 1];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma16816(acc[nt], u & mask, w & mask, (u >> 8) & mask, (w >> 8) & mask, qb[nt][j][0], qb[nt][j][1]);
            }
            const float2 pa = __half22float2(*reinterpret_cast<const __half2 *>(kb + kKv4Codes + (16 * kt + g) * 4));
            const float2 pb = __half22float2(*reinterpret_cast<const __half2 *>(kb + kKv4Codes + (16 * kt + 8 + g) * 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // an f16 q has no lo part
                const float x0 = (kF32 ? acc[nt][0] + acc[nt][1] : acc[nt][0]) * pa.y;
                const float x1 = (kF32 ? acc[nt][2] + acc[nt][3] : acc[nt][2]) * pb.y;
                sc[nt][kt][0] = fmaf(pa.x, qsum[nt], x0);
                sc[nt][kt][1] = fmaf(pb.x, qsum[nt], x1);
            }
        }
        // ------------------------------------------------ weights
        float dv[4][2], cv[4][2];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float2 p =
                    __half22float2(*reinterpret_cast<const __half2 *>(vb + kKv4Codes + (16 * kt + 8 * r + g) * 4));
                cv[kt][r] = p.x;
                dv[kt][r] = p.y;
            }
        if (!whole) {
            // masked keys score -inf; rows behind the last key may hold anything, so their c and
            // d are not used at all
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int key = key0 + 16 * kt + 8 * r + g;
                    if (key >= lmax) cv[kt][r] = dv[kt][r] = 0.f;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        if (key >= len[nt]) sc[nt][kt][r] = -CUDART_INF_F;
                }
        }
        float dm = fmaxf(dv[0][0], dv[0][1]);
#pragma unroll
        for (int kt = 1; kt < 4; ++kt) dm = max3f(dm, dv[kt][0], dv[kt][1]);
        bool grow = dm > dcap;
        float mx[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            mx[nt] = fmaxf(sc[nt][0][0], sc[nt][0][1]);
#pragma unroll
            for (int kt = 1; kt < 4; ++kt) mx[nt] = max3f(mx[nt], sc[nt][kt][0], sc[nt][kt][1]);
            grow = grow || mx[nt] > m[nt];
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, x));
            float ds = 1.f;
            if (dm > dcap) {
                const int w2 = kTop<T> - ilog2f_(dm);       // d >= 2^-24, a normal f32
                ds = dcap > 0.f ? pow2i(max(w2 - we, -126)) : 1.f;
                we = w2;
                wscale = pow2i(we);
                dcap = pow2i(kTop<T> + 1 - we) * 0.99609375f;       // the largest 8-bit number below 2^(kTop + 1 - we)
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx[nt] = fmaxf(mx[nt], __shfl_xor_sync(0xffffffffu, mx[nt], x));
                const float mn = fmaxf(m[nt], mx[nt]);
                const float al = mn == m[nt] ? 1.f : ex2_approx((m[nt] - mn) * qinv[nt]);
                m[nt] = mn;
                mul2(l[nt][0], l[nt][1], l[nt][0], l[nt][1], al, al);
                mul2(oc[nt][0], oc[nt][1], oc[nt][0], oc[nt][1], al, al);
                flush(nt, al * ds);
            }
            since = 0;
        } else if (++since == kFlush) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) flush(nt, 1.f);
            since = 0;
        }
        uint32_t pw[NT][4][2];                              // p d 2^we, split
        auto weights = [&](auto masked) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                float d0, d1;
                mul2(d0, d1, dv[kt][0], dv[kt][1], wscale, wscale);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    // no key yet: every score is -inf
                    const float mq = m[nt] == -CUDART_INF_F ? 0.f : -m[nt] * qinv[nt];
                    float p0, p1, x0, x1, c0 = cv[kt][0], c1 = cv[kt][1];
                    fma2(p0, p1, sc[nt][kt][0], sc[nt][kt][1], qinv[nt], qinv[nt], mq, mq);
                    p0 = ex2_approx(p0);
                    p1 = ex2_approx(p1);
                    add2(l[nt][0], l[nt][1], l[nt][0], l[nt][1], p0, p1);
                    if (masked.value) {                     // weight 0, but c may be NaN for this column only
                        if (sc[nt][kt][0] == -CUDART_INF_F) c0 = 0.f;
                        if (sc[nt][kt][1] == -CUDART_INF_F) c1 = 0.f;
                    }
                    fma2(oc[nt][0], oc[nt][1], p0, p1, c0, c1, oc[nt][0], oc[nt][1]);
                    mul2(x0, x1, p0, p1, d0, d1);
                    split_weights<T>(x0, x1, pw[nt][kt][0], pw[nt][kt][1]);
                }
            }
        };
        if (whole) weights(std::false_type{});
        else weights(std::true_type{});
        // ------------------------------------------------ O += V^T p
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            // keys 2t, 2t + 1 side by side; 8 more: dims 4g .. 4g + 3; the same keys, dims 32 + 4g ..
            uint32_t vw[4];
            ldmatrix4_trans(vw, rows_at + st * kKv4Block + kKv4Half + kt * 512);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t b0 = movm_trans(pw[nt][kt][0]), b1 = movm_trans(pw[nt][kt][1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t mask = (i & 1) ? 0x00F000F0u : 0x000F000Fu;
                    const uint32_t u = vw[i & 2], w = vw[(i & 2) + 1];
                    if constexpr (kF32)
                        mma16816(o[nt][i], codes_f16(u, i), codes_f16(u >> 8, i), codes_f16(w, i), codes_f16(w >> 8, i), b0,
                                 b1);
                    else
                        mma16816(o[nt][i], u & mask, (u >> 8) & mask, w & mask, (w >> 8) & mask, b0, b1);
                }
                if constexpr (!kF32) mma16816(o8[nt], 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, b0, b1);
            }
        }
        __syncwarp();                                       // the stage's last reads, before it is filled again
        if (lane == 0 && blk + stages * (long long)units < nblk) issue(blk + stages * units, st);
        if (++st == stages) {
            st = 0;
            phase ^= 1u;
        }
    }

    // ------------------------------------------------ this warp's (m, l, o) per column
    // The ring is free: every copy issued has landed (after an expired wait, the copies still
    // in flight are waited for first, with the same bound).
    if (!alive && lane == 0)
        for (int i = 0; i < stages && blk < nblk; ++i, blk += units) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&full[warp][st], phase))
                if (clock64() - t0 > kWaitBudgetCycles) break;
            if (++st == stages) {
                st = 0;
                phase ^= 1u;
            }
        }
    __syncwarp();
    float *wp = reinterpret_cast<float *>(ring);            // [kCols][kPart]
    if (idle || !alive) {                                   // l = 0: the rest is not read
        if (lane < kCols) {
            wp[lane * kPart] = -CUDART_INF_F;
            wp[lane * kPart + 1] = 0.f;
        }
    } else {
        const float back = pow2i(-we) * (kF32 ? 1.f : kUp24);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float ls = l[nt][0] + l[nt][1], os = oc[nt][0] + oc[nt][1];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                ls += __shfl_xor_sync(0xffffffffu, ls, x);
                os += __shfl_xor_sync(0xffffffffu, os, x);
            }
            flush(nt, 1.f);
            float *p = wp + (4 * nt + t) * kPart;
            if (g == 0) {
                p[0] = m[nt] * qinv[nt];
                p[1] = ls;
            }
            // accumulator i: dims 4g + {0, 2}, {1, 3}, 32 + 4g + {0, 2}, {1, 3}; odd ones in units of 2^-20
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float b = (i & 1) ? back * 0.0625f : back;
                const int d = 32 * (i >> 1) + 4 * g + (i & 1);
                p[2 + d] = fmaf(tot[nt][2 * i], b, os);
                p[2 + d + 2] = fmaf(tot[nt][2 * i + 1], b, os);
            }
        }
    }
    __syncthreads();

    // ------------------------------------------------ join the warps, then the cluster
    // Column x's partials of all CTAs meet in CTA x % ns, at recv[x / ns][rank].
    auto put = [&](int col, int d, float ll, float oo) {
        const int x = col0 + col, i = row_of(x), h = kvh * group + x - i * group;
        stf(static_cast<T *>(a.out) + s * a.o_slot + i * a.o_row + h * kKv4Hd + d, ll == 0.f ? 0.f : oo / ll);
    };
    float *recv = reinterpret_cast<float *>(kv4_smem + (size_t)W * stages * kKv4Block);
    if (ns > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
    const size_t step = (size_t)stages * kKv4Block / sizeof(float);
    for (int x = tid; x < ncol * kKv4Hd; x += kThr) {
        const int col = x / kKv4Hd, d = x % kKv4Hd;
        const float *p = reinterpret_cast<const float *>(kv4_smem) + col * kPart;
        float mm = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < W; ++w) mm = fmaxf(mm, p[w * step]);
        const float ref = mm == -CUDART_INF_F ? 0.f : mm;
        float ll = 0.f, oo = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float lw = p[w * step + 1];
            if (lw == 0.f) continue;                        // no key (a NaN sum is not 0)
            const float f = ex2_approx(p[w * step] - ref);
            ll = fmaf(lw, f, ll);
            oo = fmaf(p[w * step + 2 + d], f, oo);
        }
        if (ns > 1) {
            const int to_rank = col % ns;
            float *to = cg::this_cluster().map_shared_rank(recv, to_rank) + ((col / ns) * ns + rank) * kPart;
            to[2 + d] = oo;
            if (d == 0) {
                to[0] = mm;
                to[1] = ll;
            }
        } else {
            put(col, d, ll, oo);
        }
    }
    if (W == 1 || ns == 1) return;                          // CTAs of one warp come without a cluster
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    for (int col = rank + tid / kKv4Hd * ns; col < ncol; col += kThr / kKv4Hd * ns) {
        const int d = tid % kKv4Hd;
        const float *p = recv + (col / ns) * ns * kPart;
        float mm = -CUDART_INF_F;
        for (int r = 0; r < ns; ++r) mm = fmaxf(mm, p[r * kPart]);
        const float ref = mm == -CUDART_INF_F ? 0.f : mm;
        float ll = 0.f, oo = 0.f;
        for (int r = 0; r < ns; ++r) {
            const float f = ex2_approx(p[r * kPart] - ref);
            ll = fmaf(p[r * kPart + 1], f, ll);
            oo = fmaf(p[r * kPart + 2 + d], f, oo);
        }
        put(col, d, ll, oo);
    }
}

// f16 query columns (rows x query heads per kv head) from which the tensor-core tiles of kv4_flash.cu
// run: 32, or with a (slot, kv head) per SM what no longer fits one tile here.  They round the weights to f16
// where this form keeps 22 bits: 2.6e-4 in norm against the 2.1e-4 of a result rounded once, which is why
// calls that fit one tile here stay here although the crossover of the times lies near.  The rule goes by the number of
// pairs alone; with few pairs of long caches the tiles would be faster from some 20 columns.  Measured (us, here and
// there): 8 slots x 20 heads x 1500 keys 16 columns 24, 33; 17 42, 34; 32 42, 34; 16 x 20 x 448
// 20 columns 31, 24.  Fewer pairs: 1 x 20 x 1500 24 columns 11.0, 14.4; 1 x 20 x 448 32 columns 10.9, 11.3;
// 4 x 8 x 16000 24 columns 59, 50, 4 x 8 x 1000 11.0, 16.3, 2 x 8 x 60000 20 columns 122, 148.
constexpr int kFlashCols = 32;

template <int NT, int W, typename T>
cudaError_t launch_stream(const Kv4AttnArgs &a, long long tiles, int ns, cudaStream_t st) {
    auto fn = kv4_stream_kernel<NT, W, T>;
    const int nblk = (a.c.max_tok + kKv4Blk - 1) / kKv4Blk;
    const long long hb = (long long)nblk * kKv4Block;
    constexpr size_t kMaxSmem = (size_t)W * kMaxStages * kKv4Block + (size_t)(4 * NT + kMaxNs) * kPart * sizeof(float);
    static int max_ns = 1;                               // largest cluster the device schedules
    static std::once_flag once;
    static cudaError_t once_status;
    if (cudaError_t e = run_once(once, once_status, [&] {
            cudaError_t e1 = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
            if (e1 == cudaSuccess) e1 = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = kMaxNs;
            cfg.blockDim = 32 * W;
            cfg.dynamicSmemBytes = kMaxSmem;
            if (e1 == cudaSuccess) e1 = cudaOccupancyMaxPotentialClusterSize(&max_ns, fn, &cfg);
            return e1;
        }))
        return e;
    ns = std::min(ns, max_ns);
    const int stages = nblk > ns * W ? kMaxStages : 1;
    const size_t smem = (size_t)W * stages * kKv4Block +
                        (ns > 1 ? (size_t)((4 * NT + ns - 1) / ns) * ns * kPart * sizeof(float) : 0);
    if (tiles * ns > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_k(fn, dim3((unsigned)(tiles * ns), (unsigned)a.c.kv_heads, (unsigned)a.c.slots), 32 * W, smem, st, ns, a,
                    hb * a.c.kv_heads, hb, a.heads / a.c.kv_heads, ns, stages);
}

// Warps per (slot, kv head, tile), in CTAs of 4 or 8: as many as the SMs hold at once (16 a SM with one
// column group, else 8), none without a block; twice that where each would still have six blocks or
// more (ragged lengths leave warps idle).  CTAs of 8 where they give more warps, and on a tie unless a
// short cache has to be cut up finely.  Measured (us): 8 slots x 20 heads x 1500 keys 8.1 as 3 CTAs of 4
// (8.9 as 1 of 8, 10.3 as 6 of 4), 16 x 20 x 448 ragged 5.7 as 1 of 4 (6.2 as 1 of 8), 8 x 8 x 6000
// 10.2 as 4 of 8 (10.5 as 8 of 4), 1 x 20 x 1500 4.3 as 6 of 4 (4.7 as 3 of 8), 4 x 8 x 65003 ragged
// 28.9 as 16 of 8 (32.9 as 8 of 8).  (f32 figures of choices not taken, here and below, from before the values' codes
// became normal numbers, which adds 0 to 15 %: the chosen ones take 8.7, 6.0, 10.5 and 4.5 now.)
// With more (slot, kv head, tile)s than that, a CTA's idle warps and its join only take room from the
// next one: CTAs of two warps, of one for one or two blocks.  Measured with 4, 2 and 1 warps (us):
// f32, 14 slots x 50 rows x 32 / 4 heads x 52 keys 45.6, 32.4, 28.0 (now 26.1); 8 x 48 x 20 x 1500 46.6, 42.4, 71;
// 32 x 5 x 20 x 448 15.1, 10.9, 14.6; x 100 12.7, 9.5, 8.3; one
// column group: 64 x 1 x 20 x 64 8.5, 6.9, 5.3; 40 x 1 x 20 x 1500 (two sets of warps an SM) 22.3, 25.6, 35.9.
template <int NT, typename T>
cudaError_t launch_stream_n(const Kv4AttnArgs &a, long long cols, cudaStream_t st) {
    const long long tiles = (cols + 4 * NT - 1) / (4 * NT), pairs = tiles * a.c.kv_heads * a.c.slots;
    const int nblk = (a.c.max_tok + kKv4Blk - 1) / kKv4Blk;
    long long room = (NT == 1 ? 16LL : 8LL) * num_sms() / pairs;
    if (room < (NT == 1 ? 2 : 4))
        return room < 2 && nblk <= 2 ? launch_stream<NT, 1, T>(a, tiles, 1, st) : launch_stream<NT, 2, T>(a, tiles, 1, st);
    if (nblk >= 12 * room) room *= 2;
    const bool cut = nblk <= room;                       // a block per warp
    auto ctas = [&](int w) {
        // whole powers of two, or three times one: other cluster sizes pack badly (64 pairs, 48 blocks:
        // 8.1 us as 4 CTAs of 8, 11.2 as 9 of 4)
        const long long n = std::min<long long>((nblk + w - 1) / w, room / w);
        int c = 1;
        for (int i = 2; i <= kMaxNs; ++i)
            if (n >= i && ((i & (i - 1)) == 0 || i == 3 || i == 6 || i == 12)) c = i;
        return c;
    };
    const int n4 = ctas(4);
    if constexpr (NT < 4) {
        const int n8 = ctas(8);
        if (room >= 8 && (8 * n8 > 4 * n4 || (8 * n8 == 4 * n4 && (n8 == 1 || !cut))))
            return launch_stream<NT, 8, T>(a, tiles, n8, st);
    }
    return launch_stream<NT, 4, T>(a, tiles, n4, st);
}

template <typename T>
cudaError_t launch_stream_t(const Kv4AttnArgs &a, long long cols, cudaStream_t st) {
    return cols <= 4 ? launch_stream_n<1, T>(a, cols, st)
                     : cols <= 8 ? launch_stream_n<2, T>(a, cols, st) : launch_stream_n<4, T>(a, cols, st);
}

}  // namespace

cudaError_t launch_kv4_attn(const Kv4AttnArgs &a, bool f16, cudaStream_t st) {
    const long long cols = (long long)a.rows * (a.heads / a.c.kv_heads);
    if (f16 && (cols >= kFlashCols || (cols > 16 && (long long)a.c.slots * a.c.kv_heads >= num_sms())))
        return launch_kv4_flash(a, st);
    return f16 ? launch_stream_t<__half>(a, cols, st) : launch_stream_t<float>(a, cols, st);
}

}  // namespace madi

// kv4_flash.cu -- attention of many query rows over the 4-bit K/V cache (kv4.cuh) on the
// 5th-generation tensor cores: f16 queries and outputs, head_dim 64.
//
// Same mathematics as the streaming form (kv4_attn.cu), as matrix products of 128 x 128 tiles:
//     S = Q K^T,  K = c + d n':   Q (d n')^T + sum(Q) c^T
//     O = P V,    V = c + d n':   P (d n')   + sum_j P_j c_j
// d has 8 significant bits and |n'| <= 8, so d n' is exact in f16 and only P is rounded (2^-11 at
// most, as the output itself is): the keys' c enters S as a fifth K = 16 step with sum(Q) as two
// f16 parts, the values' c as one f32 FMA per score beside the softmax.  Rounding c + d n' to f16
// instead would add two more errors of the output's own size.
//
// One CTA per (256 query columns of one kv head, slot, share of the keys); a column is one
// (query row, query head of the kv head).  13 warps:
//   warps 0-3   one key per thread: read its packed K and V (64 bytes and two (c, d)), write the two
//               f16 rows and the c's into a 3-stage ring, in the SWIZZLE_128B layout; the next
//               tile's bytes are in flight meanwhile;
//   warps 4-11  the softmax of the two 128-column tiles (thread = column = TMEM lane), as in
//               flash_enc.cu: S in TMEM, P written back as f16, O rescaled when a maximum grew;
//   warp 12     issues the products (S: 5 steps, both operands in shared memory; O: P in TMEM as
//               the first operand, V N-contiguous) and owns TMEM.
// Within every 8 dims the shared-memory order is 0 4 1 5 2 6 3 7 -- what one mask of a code word
// gives as a pair of f16 -- for Q and K alike, and for V's columns, which are put back in order
// when O is written.  Each query row is scaled by a power of two so that its largest element lies
// in [8, 16): sum(Q) cannot leave the f16 range, and the softmax scale takes it back.
// When there are fewer CTAs than SMs, a cluster of ns CTAs splits the keys; the partial results
// meet through distributed shared memory (each CTA joins its share of the rows).
// Every wait is bounded.
#include <cooperative_groups.h>
#include <cuda.h>
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

constexpr int kQT = 128;                       // query columns per tile
constexpr int kKT = 128;                       // keys per tile
constexpr int kNS = 3;                         // ring stages
constexpr int kTile = 128 * 64 * 2;            // bytes of one [128][64] f16 tile
constexpr int kDeqThr = 128;                   // warps 0..3
constexpr int kSmWarp0 = 4;                    // warps 4..7: tile 0; 8..11: tile 1
constexpr int kMmaWarp = 12;
constexpr int kThr = 32 * 13;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTileCols = 256, kPCol = 128, kOCol = 192;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kIdescS = idesc_f16_f32(kQT, kKT);
constexpr uint32_t kIdescPV = idesc_f16_f32(kQT, kKv4Hd) | (1u << 16);     // V: N-contiguous
constexpr int kMaxNs = 8;
constexpr int kPartW = kKv4Hd + 2;             // a row's partial: O, m, l

struct __align__(16) FlashShared {
    float cv[kNS][kKT];      // the values' c
    uint64_t q_full;         // 256: both Q tiles and their sums written
    uint64_t kv_full[kNS];   // 128: a stage's keys and values written
    uint64_t kv_empty[kNS];  // its products complete
    uint64_t s_full[2], s_free[2], p_ready[2], o_done[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

// Q tiles 0 and 1 | sums of Q (tile x in 16-byte chunks 2x, 2x + 1 of each row) | stages of
// K, c of K (chunks 0, 1 of each row), V.
constexpr size_t kQBytes = 3 * (size_t)kTile, kStage = 3 * (size_t)kTile;
constexpr size_t kSmem = 1024 + kQBytes + kNS * kStage + sizeof(FlashShared);
static_assert(kSmem <= 227 * 1024, "shared memory");
static_assert(kNS * kStage >= 2 * kQT * kPartW * sizeof(float), "the partials take the ring's place");

MADI_DEV void wait_drain(uint64_t *bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > kWaitBudgetCycles) return;
}
MADI_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
MADI_DEV float max3f(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
MADI_DEV float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// 16-byte chunk c of row r of a [128][64] f16 tile in the SWIZZLE_128B layout.
MADI_DEV uint4 *chunk(uint8_t *tile, int r, int c) {
    return reinterpret_cast<uint4 *>(tile + r * 128 + ((c ^ (r & 7)) << 4));
}
// d n' of one code word's eight elements, in the order 0 4 1 5 2 6 3 7.
MADI_DEV uint4 dequant_word(uint32_t w, __half2 d) {
    const __half2 k1032 = __float2half2_rn(1032.f), k16 = __float2half2_rn(0.0625f), km72 = __float2half2_rn(-72.f);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = i ? w >> 8 : w;
        const uint32_t a = (v & 0x000F000Fu) | 0x64006400u, b = (v & 0x00F000F0u) | 0x64006400u;
        // 1024 + z -> z - 8;  1024 + 16 z -> z - 8 (both exact)
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), k1032);
        const __half2 y = __hfma2(*reinterpret_cast<const __half2 *>(&b), k16, km72);
        o[2 * i] = h2_as_u32(__hmul2(x, d));
        o[2 * i + 1] = h2_as_u32(__hmul2(y, d));
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

struct KeyBytes {
    uint4 k0, k1, v0, v1;
    uint32_t kcd, vcd;
};

__global__ void __launch_bounds__(kThr, 1)
    kv4_flash_kernel(const Kv4AttnArgs a, long long slot_bytes, long long head_bytes, int group, int tiles, int ns) {
    extern __shared__ uint8_t kv4f_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(kv4f_smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *qs = smem, *qx = smem + 2 * kTile, *ring = smem + kQBytes;
    FlashShared *sh = reinterpret_cast<FlashShared *>(ring + kNS * kStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % ns;
    // causal rows: the last tiles have the most keys, so they start first
    const int tile = tiles - 1 - (int)(blockIdx.x / ns) % tiles, kvh = (int)(blockIdx.x / ns) / tiles, s = blockIdx.y;
    pdl_trigger();
    if (threadIdx.x == 0) {
        mbar_init(&sh->q_full, 2 * kQT);
        for (int i = 0; i < kNS; ++i) {
            mbar_init(&sh->kv_full[i], kDeqThr);
            mbar_init(&sh->kv_empty[i], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&sh->s_full[x], 1);
            mbar_init(&sh->s_free[x], kQT);
            mbar_init(&sh->p_ready[x], kQT);
            mbar_init(&sh->o_done[x], 1);
        }
        mbar_init(&sh->drain, 1);
        sh->abort = 0;
        fence_mbar_init();
    }
    pdl_wait();
    const int total = kv4_rows(a.n, s, a.rows) * group, col0 = tile * 2 * kQT;
    if (col0 >= total) return;                               // padding only (the whole cluster leaves)
    // key tiles of column tile x in this CTA's share [j0, j1)
    int top[2], nt[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int last = min(col0 + (x + 1) * kQT, total) - 1;
        top[x] = last >= col0 + x * kQT ? kv4_keys(a.pos, a.lens, s, last / group, a.c.max_tok) : 0;
    }
    const int kmax = max(top[0], top[1]), all = (kmax + kKT - 1) / kKT;
    const int j0 = (int)((long long)all * rank / ns), j1 = (int)((long long)all * (rank + 1) / ns);
#pragma unroll
    for (int x = 0; x < 2; ++x) nt[x] = max(min((top[x] + kKT - 1) / kKT, j1) - j0, 0);
    const int nmax = max(nt[0], nt[1]);

    if (warp == kMmaWarp) {
        tmem_alloc(&sh->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    volatile int *abort_flag = &sh->abort;

    // softmax state, kept to the end of the kernel
    float m = -CUDART_INF_F, l = 0.f, oc = 0.f;
    const int x = warp >= kSmWarp0 + 4 ? 1 : 0;              // column tile of a softmax warp
    const int row = (warp & 3) * 32 + lane;                  // column within the tile
    const uint32_t tb = tmem + ((uint32_t)((warp & 3) * 32) << 16) + x * kTileCols;
    const int col = col0 + x * kQT + row;
    bool alive = true;

    if (warp < 4) {
        // ------------------------------------------------ codes -> f16 tiles, one key per thread
        const int r = threadIdx.x;
        const uint8_t *src = a.c.data + s * slot_bytes + kvh * head_bytes;
        auto fetch = [&](int j, KeyBytes &b) {
            const int key = (j0 + j) * kKT + r;
            b.kcd = b.vcd = 0;
            if (key < kmax) {
                const uint8_t *blk = src + (long long)(key / kKv4Blk) * kKv4Block;
                const int off = key % kKv4Blk;
                const uint4 *kp = reinterpret_cast<const uint4 *>(blk + off * 32);
                const uint4 *vp = reinterpret_cast<const uint4 *>(blk + kKv4Half + off * 32);
                b.k0 = kp[0];
                b.k1 = kp[1];
                b.v0 = vp[0];
                b.v1 = vp[1];
                b.kcd = *reinterpret_cast<const uint32_t *>(blk + kKv4Codes + off * 4);
                b.vcd = *reinterpret_cast<const uint32_t *>(blk + kKv4Half + kKv4Codes + off * 4);
            } else {
                b.k0 = b.k1 = b.v0 = b.v1 = make_uint4(0, 0, 0, 0);      // d = 0: a zero row
            }
        };
        for (int i = 0; i < kNS; ++i) *chunk(ring + i * kStage + kTile, r, 1) = make_uint4(0, 0, 0, 0);
        KeyBytes b;
        if (nmax > 0) fetch(0, b);
        for (int j = 0; j < nmax; ++j) {
            const int st = j % kNS;
            if (!warp_wait_all(&sh->kv_empty[st], ((uint32_t)(j / kNS) & 1u) ^ 1u, abort_flag, a.dev_err)) break;
            const KeyBytes cur = b;
            if (j + 1 < nmax) fetch(j + 1, b);
            uint8_t *kt = ring + st * kStage, *kx = kt + kTile, *vt = kx + kTile;
            __half2 kcd = *reinterpret_cast<const __half2 *>(&cur.kcd), vcd = *reinterpret_cast<const __half2 *>(&cur.vcd);
            // A value row that reads back as NaN must reach the columns that attend it and no
            // other: P = 0 times NaN would reach all.  It makes its key's score NaN instead.
            const float vc = __low2float(vcd), vd = __high2float(vcd);
            if (!(fabsf(vc) <= 65504.f && fabsf(vd) <= 65504.f)) {
                vcd = __float2half2_rn(0.f);
                kcd = __halves2half2(__float2half_rn(CUDART_NAN_F), __high2half(kcd));
            }
            const __half2 kd = __high2half2(kcd), vd2 = __high2half2(vcd);
            const uint32_t kw[8] = {cur.k0.x, cur.k0.y, cur.k0.z, cur.k0.w, cur.k1.x, cur.k1.y, cur.k1.z, cur.k1.w};
            const uint32_t vw[8] = {cur.v0.x, cur.v0.y, cur.v0.z, cur.v0.w, cur.v1.x, cur.v1.y, cur.v1.z, cur.v1.w};
#pragma unroll
            for (int c = 0; c < 8; ++c) *chunk(kt, r, c) = dequant_word(kw[c], kd);
#pragma unroll
            for (int c = 0; c < 8; ++c) *chunk(vt, r, c) = dequant_word(vw[c], vd2);
            *chunk(kx, r, 0) = make_uint4(h2_as_u32(__low2half2(kcd)), 0, 0, 0);
            sh->cv[st][r] = __low2float(vcd);
            fence_proxy_async_smem();
            mbar_arrive(&sh->kv_full[st]);
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------ products
        if (lane == 0) {
            const uint64_t qd = smem_desc_sw128(smem_u32(qs)), qxd = smem_desc_sw128(smem_u32(qx));
            const uint64_t rd = smem_desc_sw128(smem_u32(ring));
            constexpr uint64_t kTileU = kTile >> 4, kStageU = kStage >> 4;
            int seen = -1;                                   // last key tile known to be in the ring
            bool ok = mbar_wait(&sh->q_full, 0, abort_flag, a.dev_err);
            auto issue_s = [&](int y, int j) -> bool {
                const int st = j % kNS;
                if (seen < j) {
                    if (!mbar_wait(&sh->kv_full[st], (uint32_t)(j / kNS) & 1u, abort_flag, a.dev_err)) return false;
                    seen = j;
                }
                tc_fence_after();
                const uint64_t kd = rd + st * kStageU;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_ss(tmem + y * kTileCols, qd + y * kTileU + 2 * k, kd + 2 * k, kIdescS, k != 0);
                mma_ss(tmem + y * kTileCols, qxd + 2 * y, kd + kTileU, kIdescS, 1);
                umma_commit(&sh->s_full[y]);
                return true;
            };
            for (int y = 0; ok && y < 2; ++y)
                if (nt[y] > 0) ok = issue_s(y, 0);
            for (int j = 0; ok && j < nmax; ++j) {
                const int st = j % kNS;
                for (int y = 0; ok && y < 2; ++y) {
                    if (j >= nt[y]) continue;
                    if (j + 1 < nt[y] &&
                        (!mbar_wait(&sh->s_free[y], (uint32_t)j & 1u, abort_flag, a.dev_err) || !issue_s(y, j + 1))) {
                        ok = false;
                        break;
                    }
                    if (!mbar_wait(&sh->p_ready[y], (uint32_t)j & 1u, abort_flag, a.dev_err)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t t0 = tmem + y * kTileCols;
#pragma unroll
                    for (int k = 0; k < kKT / 16; ++k)
                        umma_f16_ts(t0 + kOCol, t0 + kPCol + 8 * k, rd + st * kStageU + 2 * kTileU + 128 * k, kIdescPV,
                                    (j | k) != 0);
                    umma_commit(&sh->o_done[y]);
                }
                if (ok) umma_commit(&sh->kv_empty[st]);
            }
            umma_commit(&sh->drain);
            wait_drain(&sh->drain, 0);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ softmax, one query column per thread
        const int q = col / group;
        const bool real = col < total;
        const int klim = real ? kv4_keys(a.pos, a.lens, s, q, a.c.max_tok) : 0x7fffffff;
        float scale;
        {
            float f[64], mx = 0.f, sum = 0.f;
            if (real) {
                const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const __half *>(a.q) + s * a.q_slot +
                                                                   q * a.q_row + (kvh * group + col % group) * kKv4Hd);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint4 u = src[c];
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                        f[8 * c + 2 * i] = v.x;
                        f[8 * c + 2 * i + 1] = v.y;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 64; ++i) f[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 64; ++i) mx = fmaxf(mx, fabsf(f[i]));
            const int e = mx > 0.f ? 3 - ((int)(__float_as_uint(mx) >> 23) - 127) : 0;     // -12 .. 27
            const float up = pow2i(e);
            scale = 0.125f * kLog2e * pow2i(-e);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __half2 h = __floats2half2_rn(f[8 * c + i] * up, f[8 * c + i + 4] * up);
                    sum += __low2float(h) + __high2float(h);
                    o[i] = h2_as_u32(h);
                }
                *chunk(qs + x * kTile, row, c) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            const float hi = __half2float(__float2half_rn(sum));
            *chunk(qx, row, 2 * x) = make_uint4(h2_as_u32(__floats2half2_rn(sum, sum - hi)), 0, 0, 0);
            *chunk(qx, row, 2 * x + 1) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            mbar_arrive(&sh->q_full);
        }
        const int n = nt[x];
        for (int j = 0; j < n; ++j) {
            const int st = j % kNS;
            alive = warp_wait_all(&sh->s_full[x], (uint32_t)j & 1u, abort_flag, a.dev_err) &&
                    warp_wait_all(&sh->kv_full[st], (uint32_t)(j / kNS) & 1u, abort_flag, a.dev_err);
            if (!alive) break;
            tc_fence_after();
            const int kcur = klim - min((j0 + j) * kKT, klim);           // keys of this tile the column attends
            const bool full = __all_sync(0xffffffffu, kcur >= kKT);
            float mx[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) mx[k] = -CUDART_INF_F;
            uint32_t sv[2][32];
            tmem_ld32(tb, sv[0]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < kKT / 32; ++c) {
                if (c + 1 < kKT / 32) tmem_ld32(tb + 32 * (c + 1), sv[(c + 1) & 1]);
                const uint32_t (&cv)[32] = sv[c & 1];
                if (full) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        mx[(i >> 1) & 7] = max3f(mx[(i >> 1) & 7], __uint_as_float(cv[i]), __uint_as_float(cv[i + 1]));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * c + i < kcur) mx[i & 7] = fmaxf(mx[i & 7], __uint_as_float(cv[i]));
                }
                if (c + 1 < kKT / 32) tmem_wait_ld();
            }
            const float mxr =
                fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
            const float mn = fmaxf(m, mxr * scale);
            const float ml = mn == -CUDART_INF_F ? 0.f : mn;              // no key yet
            const float alpha = mn == m ? 1.f : ex2_approx(m - ml);       // exactly 1 when it did not move
            if (j > 0) {
                alive = warp_wait_all(&sh->o_done[x], (uint32_t)(j - 1) & 1u, abort_flag, a.dev_err);
                if (!alive) break;
                tc_fence_after();
            }
            float bq[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, bc[4] = {0.f, 0.f, 0.f, 0.f};
            tmem_ld32(tb, sv[0]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < kKT / 32; ++c) {
                if (c + 1 < kKT / 32) tmem_ld32(tb + 32 * (c + 1), sv[(c + 1) & 1]);
                const uint32_t (&cv)[32] = sv[c & 1];
                uint32_t pp[16];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 cc = *reinterpret_cast<const float4 *>(&sh->cv[st][32 * c + i]);
                    float e[4];
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        float a0, a1;
                        fma2(a0, a1, __uint_as_float(cv[i + k]), __uint_as_float(cv[i + k + 1]), scale, scale, -ml, -ml);
                        e[k] = ex2_approx(a0);
                        e[k + 1] = ex2_approx(a1);
                    }
                    if (!full) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) e[k] = 32 * c + i + k < kcur ? e[k] : 0.f;
                    }
                    const int g = (i >> 1) & 2;
                    add2(bq[2 * g], bq[2 * g + 1], bq[2 * g], bq[2 * g + 1], e[0], e[1]);
                    add2(bq[2 * g + 2], bq[2 * g + 3], bq[2 * g + 2], bq[2 * g + 3], e[2], e[3]);
                    fma2(bc[0], bc[1], e[0], e[1], cc.x, cc.y, bc[0], bc[1]);
                    fma2(bc[2], bc[3], e[2], e[3], cc.z, cc.w, bc[2], bc[3]);
                    pp[i >> 1] = h2_as_u32(__floats2half2_rn(e[0], e[1]));
                    pp[(i >> 1) + 1] = h2_as_u32(__floats2half2_rn(e[2], e[3]));
                }
                tmem_st16(tb + kPCol + 16 * c, pp);
                if (c + 1 < kKT / 32) {
                    tmem_wait_ld();
                    if (c + 2 == kKT / 32) {
                        tc_fence_before();                   // the last of S is in registers
                        mbar_arrive(&sh->s_free[x]);
                    }
                }
            }
            l = l * alpha + (((bq[0] + bq[1]) + (bq[2] + bq[3])) + ((bq[4] + bq[5]) + (bq[6] + bq[7])));
            oc = oc * alpha + ((bc[0] + bc[1]) + (bc[2] + bc[3]));
            const bool grew = mn != m;
            m = mn;
            if (j > 0 && __any_sync(0xffffffffu, grew)) {
                uint32_t ov[32];
#pragma unroll
                for (int c = 0; c < kKv4Hd / 32; ++c) {
                    tmem_ld32(tb + kOCol + 32 * c, ov);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float o0, o1;
                        mul2(o0, o1, __uint_as_float(ov[i]), __uint_as_float(ov[i + 1]), alpha, alpha);
                        ov[i] = __float_as_uint(o0);
                        ov[i + 1] = __float_as_uint(o1);
                    }
                    tmem_st32(tb + kOCol + 32 * c, ov);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sh->p_ready[x]);
        }
        if (alive && n > 0) alive = warp_wait_all(&sh->o_done[x], (uint32_t)(n - 1) & 1u, abort_flag, a.dev_err);
        if (alive) tc_fence_after();
        if (ns == 1 && alive) {
            // O columns 8 g + 2 r, 8 g + 2 r + 1 are dims 8 g + r, 8 g + r + 4
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            __half *orow = static_cast<__half *>(a.out) + s * a.o_slot + q * a.o_row + (kvh * group + col % group) * kKv4Hd;
#pragma unroll
            for (int c = 0; c < kKv4Hd / 32; ++c) {
                uint32_t ov[32];
                if (n > 0) {
                    tmem_ld32(tb + kOCol + 32 * c, ov);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] = 0;
                }
                if (real) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        float v[8];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            v[r] = (__uint_as_float(ov[8 * g + 2 * r]) + oc) * inv;
                            v[r + 4] = (__uint_as_float(ov[8 * g + 2 * r + 1]) + oc) * inv;
                        }
                        uint4 w;
                        w.x = h2_as_u32(__floats2half2_rn(v[0], v[1]));
                        w.y = h2_as_u32(__floats2half2_rn(v[2], v[3]));
                        w.z = h2_as_u32(__floats2half2_rn(v[4], v[5]));
                        w.w = h2_as_u32(__floats2half2_rn(v[6], v[7]));
                        *reinterpret_cast<uint4 *>(orow + 32 * c + 8 * g) = w;
                    }
                }
            }
        }
    }

    if (ns > 1) {
        // The cluster's partials: this CTA's rows into the ring's place (its products are
        // done), then every CTA joins its share of the rows from all of them.
        __syncthreads();
        float *part = reinterpret_cast<float *>(ring);       // [256][kPartW]
        if (warp >= kSmWarp0 && warp < kMmaWarp) {
            float *p = part + (x * kQT + row) * kPartW;
            const bool have = alive && nt[x] > 0;
            p[kKv4Hd] = have ? m : -CUDART_INF_F;
            p[kKv4Hd + 1] = have ? l : 0.f;
#pragma unroll
            for (int c = 0; c < kKv4Hd / 32; ++c) {
                uint32_t ov[32];
                if (have) {
                    tmem_ld32(tb + kOCol + 32 * c, ov);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] = 0;
                }
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        p[32 * c + 8 * g + r] = __uint_as_float(ov[8 * g + 2 * r]) + oc;
                        p[32 * c + 8 * g + r + 4] = __uint_as_float(ov[8 * g + 2 * r + 1]) + oc;
                    }
            }
        }
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
        const int per = 2 * kQT / ns, r0 = rank * per;
        auto cl = cg::this_cluster();
        for (int i = threadIdx.x; i < per * (kKv4Hd / 4); i += kThr) {
            const int r = r0 + i / (kKv4Hd / 4), d = 4 * (i % (kKv4Hd / 4)), c = col0 + r;
            if (c >= total) continue;
            float mm = -CUDART_INF_F;
            for (int k = 0; k < ns; ++k) mm = fmaxf(mm, cl.map_shared_rank(part, k)[r * kPartW + kKv4Hd]);
            const float ref = mm == -CUDART_INF_F ? 0.f : mm;
            float ll = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < ns; ++k) {
                const float *p = cl.map_shared_rank(part, k) + r * kPartW;
                const float f = ex2_approx(p[kKv4Hd] - ref);
                ll = fmaf(p[kKv4Hd + 1], f, ll);
#pragma unroll
                for (int z = 0; z < 4; ++z) o[z] = fmaf(p[d + z], f, o[z]);
            }
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
            uint2 w;
            w.x = h2_as_u32(__floats2half2_rn(o[0] * inv, o[1] * inv));
            w.y = h2_as_u32(__floats2half2_rn(o[2] * inv, o[3] * inv));
            *reinterpret_cast<uint2 *>(static_cast<__half *>(a.out) + s * a.o_slot + (c / group) * a.o_row +
                                       (kvh * group + c % group) * kKv4Hd + d) = w;
        }
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

}  // namespace

cudaError_t launch_kv4_flash(const Kv4AttnArgs &a, cudaStream_t st) {
    static std::once_flag once;
    static cudaError_t once_status;
    if (cudaError_t e = run_once(once, once_status, [] {
            return cudaFuncSetAttribute(kv4_flash_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
        }))
        return e;
    const int group = a.heads / a.c.kv_heads;
    const long long tiles = ((long long)a.rows * group + 2 * kQT - 1) / (2 * kQT);
    const int nblk = (a.c.max_tok + kKv4Blk - 1) / kKv4Blk;
    const long long hb = (long long)nblk * kKv4Block, ctas = tiles * a.c.kv_heads * a.c.slots;
    int ns = 1;
    while (ns < kMaxNs && ctas * ns < num_sms() && nblk >= 8 * ns) ns *= 2;
    if (tiles * a.c.kv_heads * ns > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_k(kv4_flash_kernel, dim3((unsigned)(tiles * a.c.kv_heads * ns), (unsigned)a.c.slots), kThr, kSmem, st, ns,
                    a, hb * a.c.kv_heads, hb, group, (int)tiles, ns);
}

}  // namespace madi

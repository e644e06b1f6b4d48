// kv4_flash.cu -- attention of many query rows over the 4-bit K/V cache (kv4.cuh) on the
// 5th-generation tensor cores: f16 queries and outputs, head_dim 64.
//
// Same mathematics as the streaming form (kv4_attn.cu), as matrix products of 128 x 96 tiles:
//     S = Q K^T,  K = c + d n':   Q (d n')^T + sum(Q) c^T
//     O = P V,    V = c + d n':   P (d n')   + sum_j P_j c_j
// d has 8 significant bits and |n'| <= 8, so d n' is exact in f16 and only P is rounded (by 2^-11 of
// itself, as the output is, and by 2^-38 of the row's largest where it is below 2^-27 of that; the
// streaming form keeps 22 bits of it): the keys' c enters S as a fifth K = 16 step with sum(Q) as two
// f16 parts, the values' c as one more column of V, beside a column of ones that gives the sum of
// the weights.  Rounding c + d n' to f16 instead would add two more errors of the output's own size.
//
// One CTA per (128 or 256 query columns of one kv head, slot, share of the keys); a column is one
// (query row, query head of the kv head).  Warps:
//   warps 0-2   read the packed K and V rows (32 bytes and (c, d) each), write the f16 rows and the
//               c's into a ring of stages, in the SWIZZLE_128B layout; the next tile's bytes are in
//               flight meanwhile;
//   warp 3      issues the products (S: 5 steps, both operands in shared memory; O: P in TMEM as
//               the first operand, V N-contiguous) and owns TMEM;
//   warps 4-11  (4-7) the softmax of the 128-column tiles (thread = column = TMEM lane), as in
//               flash_enc.cu: S in TMEM, P written back as f16, O rescaled when a maximum grew.
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

#include <mutex>
#include <type_traits>

#include "internal.h"
#include "kv4.cuh"

namespace cg = cooperative_groups;

namespace madi {
namespace {

constexpr int kQT = 128;                       // query columns per tile
constexpr int kKT = 96;                        // keys per tile: S, P and O of two tiles fit TMEM, a row of S registers
constexpr int kTile = 128 * 64 * 2;            // bytes of one [128][64] f16 tile (Q)
constexpr int kKTile = kKT * 64 * 2;           // bytes of one [96][64] f16 tile (K, V)
constexpr int kDeqThr = 96;                    // warps 0..2
constexpr int kMmaWarp = 3;
constexpr int kSmWarp0 = 4;                    // warps 4..7: tile 0; 8..11: tile 1
constexpr uint32_t kTileCols = 256, kPCol = 96, kOCol = 144, kSumCol = kOCol + kKv4Hd;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kIdescS = idesc_f16_f32(kQT, kKT);
constexpr uint32_t kIdescPV = idesc_f16_f32(kQT, kKv4Hd + 16) | (1u << 16);      // V: N-contiguous
constexpr int kMaxNs = 8;
// A weight is 2^kPOff times 2^(score - reference); the reference lies at most 2^kSlack below the largest score so
// far, so the largest weight is between 2^13 and 2^15 and f16 holds weights down to 2^-27 of it with all its bits
// (those behind a dominant key count as much as any when that key's value is small; with the largest at 1
// to 2^8, half of a result was lost at 2^-22).  Slack 2 for 8 costs about 1 %: 2 x 1024 rows x 32 heads,
// 16640 keys 351.8 us, 348.4 with 8, 349.6 with 4, 356.0 with 0.
constexpr float kSlack = 2.f, kPOff = 13.f;
constexpr int kPartW = kKv4Hd + 2;             // a row's partial: O, m, l

template <int kX, int kNS> struct __align__(16) FlashShared {
    uint64_t q_full;         // kX * 128: the Q tiles and their sums written
    uint64_t kv_full[kNS];   // 96: a stage's keys and values written
    uint64_t kv_empty[kNS];  // its products complete
    uint64_t s_full[kX], s_free[kX], p_ready[kX], o_done[kX];
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

// A CTA with kX query tiles: two with a ring of three stages, one CTA per SM; or one with two stages,
// two CTAs per SM.  Shared memory: Q tiles | sums of Q (tile x in 16-byte chunks 2x, 2x + 1 of each row)
// | stages of K | V | a key's extra columns, in one row: chunks 0, 1 the columns 64.. of V (the value's
// c, then 1: their products with P are sum p c and sum p), chunks 2, 3 the fifth step of K (c twice).
constexpr size_t kStage = 3 * (size_t)kKTile;
template <int kX> struct FlashCfg {
    static constexpr int kNS = kX == 2 ? 3 : 2, kPerSm = kX == 2 ? 1 : 2, kThr = 32 * (4 + 4 * kX);
    static constexpr uint32_t kTmemCols = 256 * kX;
    using Shared = FlashShared<kX, kNS>;
    static constexpr size_t kQBytes = (kX + 1) * (size_t)kTile;
    static constexpr size_t kSmem = 1024 + kQBytes + kNS * kStage + sizeof(Shared);
    static_assert(kPerSm * (kSmem + 1024) <= 227 * 1024, "shared memory");
    static_assert(kNS * kStage >= kX * kQT * kPartW * sizeof(float), "the partials take the ring's place");
};

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
// Two consecutive 32-bit columns.
MADI_DEV void tmem_ld2(uint32_t taddr, uint32_t &r0, uint32_t &r1) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(taddr));
}
MADI_DEV void tmem_st2(uint32_t taddr, uint32_t r0, uint32_t r1) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(taddr), "r"(r0), "r"(r1) : "memory");
}

// 16-byte chunk c of row r of a [..][64] f16 tile in the SWIZZLE_128B layout.
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

MADI_DEV __half2 as_h2(uint32_t w) { return *reinterpret_cast<__half2 *>(&w); }
struct RowBytes {
    uint4 lo, hi;       // code words
    uint32_t cd;
};

template <int kX>
__global__ void __launch_bounds__(FlashCfg<kX>::kThr, FlashCfg<kX>::kPerSm)
    kv4_flash_kernel(const Kv4AttnArgs a, long long slot_bytes, long long head_bytes, int group, int tiles, int ns) {
    using Cfg = FlashCfg<kX>;
    using Shared = typename Cfg::Shared;
    constexpr int kNS = Cfg::kNS, kThr = Cfg::kThr;
    constexpr size_t kQBytes = Cfg::kQBytes;
    extern __shared__ uint8_t kv4f_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(kv4f_smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *qs = smem, *qx = smem + kX * kTile, *ring = smem + kQBytes;
    Shared *sh = reinterpret_cast<Shared *>(ring + kNS * kStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % ns;
    // causal rows: the last tiles have the most keys, so they start first
    const int tile = tiles - 1 - (int)(blockIdx.x / ns) % tiles, kvh = (int)(blockIdx.x / ns) / tiles, s = blockIdx.y;
    pdl_trigger();
    if (threadIdx.x == 0) {
        mbar_init(&sh->q_full, kX * kQT);
        for (int i = 0; i < kNS; ++i) {
            mbar_init(&sh->kv_full[i], kDeqThr);
            mbar_init(&sh->kv_empty[i], 1);
        }
        for (int x = 0; x < kX; ++x) {
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
    const int total = kv4_rows(a.n, s, a.rows) * group, col0 = tile * kX * kQT;
    if (col0 >= total) return;                               // padding only (the whole cluster leaves)
    // key tiles of column tile x in this CTA's share [j0, j1)
    int top[kX], nt[kX], kmax = 0, nmax = 0;
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        const int last = min(col0 + (x + 1) * kQT, total) - 1;
        top[x] = last >= col0 + x * kQT ? kv4_keys(a.pos, a.lens, s, last / group, a.c.max_tok) : 0;
    }
#pragma unroll
    for (int x = 0; x < kX; ++x) kmax = max(kmax, top[x]);
    const int all = (kmax + kKT - 1) / kKT;
    const int j0 = (int)((long long)all * rank / ns), j1 = (int)((long long)all * (rank + 1) / ns);
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        nt[x] = max(min((top[x] + kKT - 1) / kKT, j1) - j0, 0);
        nmax = max(nmax, nt[x]);
    }

    if (warp == kMmaWarp) {
        tmem_alloc(&sh->tmem_base, Cfg::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    volatile int *abort_flag = &sh->abort;

    if (warp < kMmaWarp) {
        // ------------------------------------------------ codes -> f16 tiles
        // One key per thread: its K and V rows, fetched a tile ahead as soon as the ones before are
        // written, so that one set of registers serves.
        const int r = threadIdx.x;
        const uint8_t *src = a.c.data + s * slot_bytes + kvh * head_bytes;
        RowBytes kb, vb;
        auto fetch = [&](int j, int half, RowBytes &b) {
            const int key = (j0 + j) * kKT + r;
            b.lo = b.hi = make_uint4(0, 0, 0, 0);
            b.cd = 0;                                        // d = 0: a zero row
            if (j < nmax && key < kmax) {
                const uint8_t *blk = src + (long long)(key / kKv4Blk) * kKv4Block + half;
                const int off = key % kKv4Blk;
                b.lo = reinterpret_cast<const uint4 *>(blk + off * 32)[0];
                b.hi = reinterpret_cast<const uint4 *>(blk + off * 32)[1];
                b.cd = *reinterpret_cast<const uint32_t *>(blk + kKv4Codes + off * 4);
            }
        };
        auto write = [&](uint8_t *rows, const RowBytes &b, __half2 d) {
            const uint32_t w[8] = {b.lo.x, b.lo.y, b.lo.z, b.lo.w, b.hi.x, b.hi.y, b.hi.z, b.hi.w};
#pragma unroll
            for (int c = 0; c < 8; ++c) *chunk(rows, r, c) = dequant_word(w[c], d);
        };
        for (int i = 0; i < kNS; ++i) {
            *chunk(ring + i * kStage + 2 * kKTile, r, 1) = make_uint4(0, 0, 0, 0);
            *chunk(ring + i * kStage + 2 * kKTile, r, 3) = make_uint4(0, 0, 0, 0);
        }
        fetch(0, 0, kb);
        fetch(0, kKv4Half, vb);
        for (int j = 0; j < nmax; ++j) {
            const int st = j % kNS;
            if (!warp_wait_all(&sh->kv_empty[st], ((uint32_t)(j / kNS) & 1u) ^ 1u, abort_flag, a.dev_err)) break;
            uint8_t *kt = ring + st * kStage, *xt = kt + 2 * kKTile;
            __half2 kcd = as_h2(kb.cd), vcd = as_h2(vb.cd);
            // A value row that reads back as NaN must reach the columns that attend it and no
            // other: P = 0 times NaN would reach all.  It makes its key's score NaN instead.
            if (!(fabsf(__low2float(vcd)) <= 65504.f && fabsf(__high2float(vcd)) <= 65504.f)) {
                vcd = __float2half2_rn(0.f);
                kcd = __halves2half2(__float2half_rn(CUDART_NAN_F), __high2half(kcd));
            }
            write(kt, kb, __high2half2(kcd));
            fetch(j + 1, 0, kb);
            write(kt + kKTile, vb, __high2half2(vcd));
            fetch(j + 1, kKv4Half, vb);
            *chunk(xt, r, 0) = make_uint4(h2_as_u32(__halves2half2(__low2half(vcd), __float2half_rn(1.f))), 0, 0, 0);
            *chunk(xt, r, 2) = make_uint4(h2_as_u32(__low2half2(kcd)), 0, 0, 0);
            fence_proxy_async_smem();
            mbar_arrive(&sh->kv_full[st]);
        }
        if (ns > 1) {                                        // the softmax warps' join
            named_bar_sync(0, kThr);
            cluster_sync_all();
            cluster_sync_all();
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------ products
        if (lane == 0) {
            const uint64_t qd = smem_desc_sw128(smem_u32(qs)), qxd = smem_desc_sw128(smem_u32(qx));
            const uint64_t rd = smem_desc_sw128(smem_u32(ring));
            constexpr uint64_t kTileU = kTile >> 4, kKTileU = kKTile >> 4, kStageU = kStage >> 4;
            // V N-contiguous: its columns 64.. lie one [96][64] tile further on (the descriptor's leading
            // offset, bits 16..29, which K-major operands do not use)
            const uint64_t vd = (rd & ~((uint64_t)0x3FFF << 16)) + kKTileU + (kKTileU << 16);
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
                mma_ss(tmem + y * kTileCols, qxd + 2 * y, kd + 2 * kKTileU + 2, kIdescS, 1);
                umma_commit(&sh->s_full[y]);
                return true;
            };
            for (int y = 0; ok && y < kX; ++y)
                if (nt[y] > 0) ok = issue_s(y, 0);
            for (int j = 0; ok && j < nmax; ++j) {
                const int st = j % kNS;
                for (int y = 0; ok && y < kX; ++y) {
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
                        umma_f16_ts(t0 + kOCol, t0 + kPCol + 8 * k, vd + st * kStageU + 128 * k, kIdescPV,
                                    (j | k) != 0);
                    umma_commit(&sh->o_done[y]);
                }
                if (ok) umma_commit(&sh->kv_empty[st]);
            }
            umma_commit(&sh->drain);
            wait_drain(&sh->drain, 0);
        }
        __syncwarp();
        if (ns > 1) {                                        // the softmax warps' join
            named_bar_sync(0, kThr);
            cluster_sync_all();
            cluster_sync_all();
        }
    } else {
        // ------------------------------------------------ softmax, one query column per thread
        float m = -CUDART_INF_F;
        const int x = (warp - kSmWarp0) >> 2;                // column tile of this warp
        const int row = (warp & 3) * 32 + lane;              // column within the tile
        const uint32_t tb = tmem + ((uint32_t)((warp & 3) * 32) << 16) + x * kTileCols;
        const int col = col0 + x * kQT + row;
        bool alive = true;
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
            alive = warp_wait_all(&sh->s_full[x], (uint32_t)j & 1u, abort_flag, a.dev_err);
            if (!alive) break;
            tc_fence_after();
            const int kcur = klim - min((j0 + j) * kKT, klim);           // keys of this tile the column attends
            const bool full = __all_sync(0xffffffffu, kcur >= kKT);
            float mn = m, alpha = 1.f;
            // One row of S through the softmax.  Only the last tiles of a column mask keys: their own
            // copy of the code, so that the others carry no selects.
            auto tile_softmax = [&](auto whole) -> bool {
                uint32_t sv[kKT / 32][32];
#pragma unroll
                for (int c = 0; c < kKT / 32; ++c) tmem_ld32(tb + 32 * c, sv[c]);
                tmem_wait_ld();
                tc_fence_before();                           // S is in registers: the next S may take its place
                mbar_arrive(&sh->s_free[x]);
                auto score = [&](int c, int i) {
                    const float v = __uint_as_float(sv[c][i]);
                    return whole.value || 32 * c + i < kcur ? v : -CUDART_INF_F;
                };
                float mx[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) mx[k] = -CUDART_INF_F;
#pragma unroll
                for (int c = 0; c < kKT / 32; ++c)
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        mx[(i >> 1) & 7] = max3f(mx[(i >> 1) & 7], score(c, i), score(c, i + 1));
                const float mxr = max3f(max3f(mx[0], mx[1], mx[2]), max3f(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
                // The reference moves only when a maximum passes it by more than 2^kSlack, so O is rescaled in
                // few tiles instead of most.
                const float mt = mxr * scale;
                mn = mt > m + kSlack ? mt : m;
                const float ml = mn == -CUDART_INF_F ? 0.f : mn;          // no key yet
                const float off = kPOff - ml;
                alpha = mn == m ? 1.f : ex2_approx(m - ml);               // exactly 1 when it did not move
                if (j > 0) {
                    if (!warp_wait_all(&sh->o_done[x], (uint32_t)(j - 1) & 1u, abort_flag, a.dev_err)) return false;
                    tc_fence_after();
                }
#pragma unroll
                for (int c = 0; c < kKT / 32; ++c) {
                    uint32_t pp[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float a0, a1;
                        fma2(a0, a1, score(c, i), score(c, i + 1), scale, scale, off, off);
                        pp[i >> 1] = h2_as_u32(__floats2half2_rn(ex2_approx(a0), ex2_approx(a1)));
                    }
                    tmem_st16(tb + kPCol + 16 * c, pp);
                }
                return true;
            };
            alive = full ? tile_softmax(std::true_type{}) : tile_softmax(std::false_type{});
            if (!alive) break;
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
                uint32_t c0, c1;
                tmem_ld2(tb + kSumCol, c0, c1);
                tmem_wait_ld();
                tmem_st2(tb + kSumCol, __float_as_uint(__uint_as_float(c0) * alpha), __float_as_uint(__uint_as_float(c1) * alpha));
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sh->p_ready[x]);
        }
        if (alive && n > 0) alive = warp_wait_all(&sh->o_done[x], (uint32_t)(n - 1) & 1u, abort_flag, a.dev_err);
        float l = 0.f, oc = 0.f;                             // sums of p and of p c
        if (alive) {
            tc_fence_after();
            if (n > 0) {
                uint32_t c0, c1;
                tmem_ld2(tb + kSumCol, c0, c1);
                tmem_wait_ld();
                oc = __uint_as_float(c0);
                l = __uint_as_float(c1);
            }
        }
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
        if (ns > 1) {
            // The cluster's partials: this CTA's rows into the ring's place (its products are
            // done), then every CTA joins its share of the rows from all of them.
            named_bar_sync(0, kThr);
            float *part = reinterpret_cast<float *>(ring);   // [kX * kQT][kPartW]
            float *p = part + (x * kQT + row) * kPartW;
            const bool have = alive && n > 0;
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
            cluster_sync_all();
            const int r0 = kX * kQT * rank / ns, per = kX * kQT * (rank + 1) / ns - r0;
            auto cl = cg::this_cluster();
            for (int i = threadIdx.x - 32 * kSmWarp0; i < per * (kKv4Hd / 4); i += kX * kQT) {
                const int r = r0 + i / (kKv4Hd / 4), d = 4 * (i % (kKv4Hd / 4)), c = col0 + r;
                if (c >= total) continue;
                float mm = -CUDART_INF_F;
                for (int k = 0; k < ns; ++k) mm = fmaxf(mm, cl.map_shared_rank(part, k)[r * kPartW + kKv4Hd]);
                const float ref = mm == -CUDART_INF_F ? 0.f : mm;
                float ll = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
                for (int k = 0; k < ns; ++k) {
                    const float *pk = cl.map_shared_rank(part, k) + r * kPartW;
                    const float f = ex2_approx(pk[kKv4Hd] - ref);
                    ll = fmaf(pk[kKv4Hd + 1], f, ll);
#pragma unroll
                    for (int z = 0; z < 4; ++z) o[z] = fmaf(pk[d + z], f, o[z]);
                }
                const float inv = ll == 0.f ? 0.f : 1.0f / ll;
                uint2 w;
                w.x = h2_as_u32(__floats2half2_rn(o[0] * inv, o[1] * inv));
                w.y = h2_as_u32(__floats2half2_rn(o[2] * inv, o[3] * inv));
                *reinterpret_cast<uint2 *>(static_cast<__half *>(a.out) + s * a.o_slot + (c / group) * a.o_row +
                                           (kvh * group + c % group) * kKv4Hd + d) = w;
            }
            cluster_sync_all();
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

template <int kX>
cudaError_t launch_flash(const Kv4AttnArgs &a, cudaStream_t st) {
    using Cfg = FlashCfg<kX>;
    static std::once_flag once;
    static cudaError_t once_status;
    if (cudaError_t e = run_once(once, once_status, [] {
            return cudaFuncSetAttribute(kv4_flash_kernel<kX>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::kSmem);
        }))
        return e;
    const int group = a.heads / a.c.kv_heads;
    const long long tiles = ((long long)a.rows * group + kX * kQT - 1) / (kX * kQT);
    const int nblk = (a.c.max_tok + kKv4Blk - 1) / kKv4Blk;
    const long long hb = (long long)nblk * kKv4Block, ctas = tiles * a.c.kv_heads * a.c.slots;
    const long long room = (long long)num_sms() * Cfg::kPerSm;
    // Cluster size.  A CTA costs about 7 us beside its key tiles of 1.7 us each (4 tiles' time),
    // one of a cluster 16 us (9 tiles'); take the size with the least rounds x time.  Two or three rounds of
    // long shares are cut once more where slots may differ in length, which would leave the rounds unbalanced: 2 x
    // 1024 rows x 32 / 8 heads, 16640 keys, at 1 and 2 CTAs: ragged pos 379, 351 us, ragged lens 390, 359; equal pos
    // 506, 547.  Whole caches (515, 558) and what fits one round are not: 2 x 128 rows x 32 / 8 heads x 60000 at 4
    // and 8: 243, 400, ragged lens 244, 266; 1 x 2000 x 8 / 2 x 30000 at 2 and 4: 240, 252.
    const long long ktiles = (a.c.max_tok + kKT - 1) / kKT;
    int ns = 1;
    long long best = 0;
    for (int c = 1; c <= kMaxNs; ++c) {
        const long long rounds = (ctas * c + room - 1) / room;
        const long long cost = rounds * (ktiles / c + (c > 1 ? 9 : 4));
        if (c == 1 || cost < best) {
            best = cost;
            ns = c;
        }
    }
    const bool unequal = a.c.slots > 1 && (a.pos || a.lens || a.n);
    while (unequal && ns * 2 <= kMaxNs && ctas * ns > room && ctas * ns < 4 * room && ktiles / (ns * 2) >= 64) ns *= 2;
    if (tiles * a.c.kv_heads * ns > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_k(kv4_flash_kernel<kX>, dim3((unsigned)(tiles * a.c.kv_heads * ns), (unsigned)a.c.slots), Cfg::kThr,
                    Cfg::kSmem, st, ns, a, hb * a.c.kv_heads, hb, group, (int)tiles, ns);
}

}  // namespace

// One query tile per CTA where the columns fit one (8 slots x 20 heads x 1500 keys: 64 columns 35 us, with
// two 43; 128: 36, 44; 128 registers, some 60 bytes spilled, for two CTAs an SM), else two, which share the keys they unpack (2 x 1024 rows x 32 heads, 16640 keys:
// 352 us; 349 and 363 with one at an earlier state).
cudaError_t launch_kv4_flash(const Kv4AttnArgs &a, cudaStream_t st) {
    return (long long)a.rows * (a.heads / a.c.kv_heads) <= kQT ? launch_flash<1>(a, st) : launch_flash<2>(a, st);
}

}  // namespace madi

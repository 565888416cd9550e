// gemm8.hip -- products of two matrices in 8 bits, out = a . b^T (+ bias).
//
//   out[m][n] = sum_k a[m][k] 2^ea[m][k / 128] b[n][k] 2^eb[n][k / 128]
//
// Codes are widened to bf16 on their way from LDS or memory into the matrix cores,
// their block's scale folded in by the same instruction (both exact: a code has
// four significant bits), and multiplied by v_mfma_f32_32x32x16_bf16 or
// v_mfma_f32_16x16x32_bf16 into 32-bit sums.  The matrix cores also take e4m3
// itself, at twice the rate, but add eight neighbouring products aligned to the
// largest of them with 13 bits below it, the rest cut off (probe_mfma_e4m3.hip): 1.5e-5
// off on normal data, 7e-5 and always low on positive data, where these sums are 1e-7
// and 3e-7 off at k = 4096.
#include <algorithm>
#include <cmath>

#include "bf16x3.h"
#include "gemm_common.h"
#include "linear8.h"

namespace clove {
namespace k {

namespace {

// Eight codes (two dwords) times 2^e (scale) as bf16.
__device__ __forceinline__ bf8 widen8(unsigned lo, unsigned hi, float scale) {
    union {
        bf8 v;
        bf2 p[4];
    } r;
    r.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    r.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    r.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    r.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return r.v;
}

// Workgroups are dealt to the eight XCDs in turn, each with its own L2: workgroup L
// takes the L / 8-th tile of its XCD's eighth of an order that goes through groups
// of eight tile rows column by column, so that an XCD's workgroups share operands.
__device__ __forceinline__ bool tile_of(int L, int tiles_m, int tiles_n, int *tm, int *tn) {
    const int tiles = tiles_m * tiles_n, xcd = L % 8;
    const int V = (int)((int64_t)xcd * tiles / 8) + L / 8;
    if (V >= (int)((int64_t)(xcd + 1) * tiles / 8)) return false;
    const int group = 8 * tiles_n, first = V / group * 8, rows = min(8, tiles_m - first);
    const int r = V % group;
    *tm = first + r % rows;
    *tn = r / rows;
    return true;
}

// One operand's buffer from row r0 on, `rows` rows at most: a row past the matrix's
// end lies past the buffer, where reads give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t codes_from(const uint8_t *p, int r0, int rows,
                                                             int all, uint32_t kp) {
    return make_rsrc(p + (size_t)r0 * kp, (uint32_t)min(rows, all - r0) * kp);
}

// Where row r's exponents lie, in bytes behind those of row r0's line.
__device__ __forceinline__ uint32_t exps_at(int r, int r0, bool tiles, int blocks) {
    return (uint32_t)((tiles ? r >> 7 : r) - (tiles ? r0 >> 7 : r0)) * (uint32_t)blocks * 4u;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t exps_from(const int32_t *p, int r0, int rows,
                                                            bool tiles, int blocks) {
    return make_rsrc(p + (size_t)(tiles ? r0 >> 7 : r0) * blocks,
                     (uint32_t)rows * (uint32_t)blocks * 4u);
}

// In LDS a row of a block is 128 bytes, its eight 16-byte slots permuted by the
// row: eight lanes that read one slot of eight rows meet every bank, and a DMA of
// eight rows (lane l: slot l % 8 of row l / 8) still reads whole lines.
__device__ __forceinline__ int slot_of(int row, int k16) { return 16 * (k16 ^ (row & 7)); }

// BM x BN tiles in KG groups of waves of 64 x 64 each; group k takes the chunks k,
// k + KG, ... (32 codes) of every block, and the groups' sums are added at the end:
// more waves a CU without smaller tiles for each, whose operands would be widened
// more often (four conversions an MFMA here, eight with waves of 32 x 32).  Blocks of
// both operands and their exponents move by buffer->LDS DMA into two stages, one
// filling while the other is multiplied (in registers the exponents would make every
// block wait for all DMAs in flight).
//
// What bounds it: 4096^3 in 256 x 256 tiles of sixteen waves 111-115 us, 1190-1240
// TFLOP/s, of which the 64 MiB of results are some 13 us at the end; a large bf16
// library product runs at 1208 on the same card, at its power limit.  Four waves
// of 128 x 64 on 256 x 128 tiles 134 us, of 64 x 64 on 128 x 128 124-134.  Results
// stored with the non-temporal policy: 8192 x 4096 x 1024 86 us, 92 without.  Small
// products are bound by a block's chain of barrier, reads, conversions and MFMAs
// (0.5-0.65 us with a workgroup a CU; three to six stages no quicker): 768 x 768 x
// 1554 9.2 us, waves of 32 x 32 on 64 x 64 tiles 9.2-10.5.
template <int BM, int BN, int KG, int MINW>
__global__ void __launch_bounds__(BM / 64 * (BN / 64) * KG * 64)
    __attribute__((amdgpu_waves_per_eu(MINW))) gemm8_kernel(Gemm8Args g, Gemm8Plan p) {
    constexpr int WG = BM / 64 * (BN / 64), NW = WG * KG;  // waves of a group, and all
    constexpr int IB = 2, JB = 2;                          // a wave's 32 x 32 blocks
    constexpr int OWN = IB * JB * 4 / KG;                  // quarter blocks that a group stores
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int ND = (BM + BN) / 8, IW = (ND + NW - 1) / NW;   // DMAs a block, and a wave's
    constexpr int XD = (BM + BN) / 64, XW = (XD + NW - 1) / NW;  // of exponents
    static_assert(BM % 64 == 0 && BN % 64 == 0, "whole DMAs of exponents");
    static_assert(IB * JB * 4 % KG == 0 && 4 % KG == 0, "equal shares");
    static_assert(KG == 1 || NW * OWN * 1024 <= 2 * STAGE, "a round of sums fits");
    __shared__ __attribute__((aligned(16))) char smem[2 * (STAGE + XD * 256)];
    int tm, tn;
    if (!tile_of(blockIdx.x, p.tiles_m, p.tiles_n, &tm, &tn)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int kb0 = blockIdx.y * p.per_split;
    const int blocks = min(p.per_split, g.blocks - kb0);
    const uint32_t kp = (uint32_t)g.blocks * 128u;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, h = lane >> 5;
    const int kg = wave / WG;
    const int wm0 = wave % WG / (BN / 64) * 64, wn0 = wave % (BN / 64) * 64;
    const __amdgpu_buffer_rsrc_t ra = codes_from(g.a, m0, BM, g.m, kp);
    const __amdgpu_buffer_rsrc_t rb = codes_from(g.b, n0, BN, g.n, kp);
    const __amdgpu_buffer_rsrc_t rxa = exps_from(g.a_exps, m0, BM, g.a_tiles, g.blocks);
    const __amdgpu_buffer_rsrc_t rxb = exps_from(g.b_exps, n0, BN, g.b_tiles, g.blocks);
    // DMA d moves eight rows, those of a first
    uint32_t off[IW], xoff[XW];
#pragma unroll
    for (int u = 0; u < IW; ++u) {
        const int d = u * NW + wave, r = (d < BM / 8 ? d : d - BM / 8) * 8 + lane / 8;
        off[u] = (uint32_t)r * kp + (uint32_t)slot_of(r, lane % 8) + (uint32_t)kb0 * 128u;
    }
    // DMA d of exponents has those of 64 rows (past the end: the last one's)
#pragma unroll
    for (int u = 0; u < XW; ++u) {
        const int at = (u * NW + wave) * 64 + lane;
        xoff[u] = (at < BM ? exps_at(min(m0 + at, g.m - 1), m0, g.a_tiles, g.blocks)
                           : exps_at(min(n0 + at - BM, g.n - 1), n0, g.b_tiles, g.blocks)) +
                  (uint32_t)kb0 * 4u;
    }
    const auto stage = [&](int kb) { return smem + (kb & 1) * (STAGE + XD * 256); };
    const auto dma = [&](int kb) {
        char *st = stage(kb);
#pragma unroll
        for (int u = 0; u < XW; ++u) {
            const int d = u * NW + wave;
            if (d < BM / 64)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rxa, (lds_void *)(st + STAGE + d * 256), 4,
                                                         (int)xoff[u], kb * 4, 0, 0);
            else if (d < XD)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rxb, (lds_void *)(st + STAGE + d * 256), 4,
                                                         (int)xoff[u], kb * 4, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < IW; ++u) {
            const int d = u * NW + wave;
            if ((u + 1) * NW <= BM / 8 || (u * NW < BM / 8 && d < BM / 8))
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void *)(st + d * 1024), 16,
                                                         (int)off[u], kb * 128, 0, 0);
            else if ((u + 1) * NW <= ND || d < ND)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void *)(st + d * 1024), 16,
                                                         (int)off[u], kb * 128, 0, 0);
        }
    };
    f16v acc[IB][JB];
#pragma unroll
    for (int i = 0; i < IB; ++i)
#pragma unroll
        for (int j = 0; j < JB; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    if (blocks > 0) dma(0);
    for (int kb = 0; kb < blocks; ++kb) {
        // this wave's DMAs of the block have landed and its reads of the stage
        // before are done; past the barrier, every wave's
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        if (kb + 1 < blocks) dma(kb + 1);
        const char *sA = stage(kb), *sB = sA + BM * 128;
        const int *x = reinterpret_cast<const int *>(sA + STAGE);
        float sa[IB], sb[JB];
#pragma unroll
        for (int i = 0; i < IB; ++i) sa[i] = lin8_pow2(x[wm0 + 32 * i + l32]);
#pragma unroll
        for (int j = 0; j < JB; ++j) sb[j] = lin8_pow2(x[BM + wn0 + 32 * j + l32]);
        __builtin_amdgcn_s_setprio(1);
        // chunk c: lanes 0-31 hold its codes 0-15, lanes 32-63 16-31, of both operands
#pragma unroll
        for (int u = 0; u < 4 / KG; ++u) {
            const int c = u * KG + kg, slot = slot_of(l32, 2 * c + h);
            bf8 fa[IB][2], fb[JB][2];
#pragma unroll
            for (int i = 0; i < IB; ++i) {
                const u4 v = *reinterpret_cast<const u4 *>(sA + (wm0 + 32 * i + l32) * 128 + slot);
                fa[i][0] = widen8(v[0], v[1], sa[i]);
                fa[i][1] = widen8(v[2], v[3], sa[i]);
            }
#pragma unroll
            for (int j = 0; j < JB; ++j) {
                const u4 v = *reinterpret_cast<const u4 *>(sB + (wn0 + 32 * j + l32) * 128 + slot);
                fb[j][0] = widen8(v[0], v[1], sb[j]);
                fb[j][1] = widen8(v[2], v[3], sb[j]);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < IB; ++i)
#pragma unroll
                    for (int j = 0; j < JB; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][q], fb[j][q],
                                                                            acc[i][j], 0, 0, 0);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    // group o stores quarter blocks o OWN .. o OWN + OWN - 1 of its waves' tiles: in
    // round t it gets them from group o - t, so their sums are added in one order
    const auto quarter = [&](int o, int u, auto f) {
        const int q = o * OWN + u;
        f(acc[q / 4 / JB][q / 4 % JB], q % 4);
    };
#pragma unroll
    for (int t = 1; t < KG; ++t) {
        f4 *const sums = reinterpret_cast<f4 *>(smem);
        lds_barrier();
#pragma unroll
        for (int o = 0; o < KG; ++o)
            if (kg == (o + KG - t) % KG)
#pragma unroll
                for (int u = 0; u < OWN; ++u)
                    quarter(o, u, [&](f16v &v, int e) {
                        sums[(wave * OWN + u) * 64 + lane] =
                            (f4){v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
                    });
        lds_barrier();
#pragma unroll
        for (int o = 0; o < KG; ++o)
            if (kg == o)
#pragma unroll
                for (int u = 0; u < OWN; ++u)
                    quarter(o, u, [&](f16v &v, int e) {
                        const int from = (o + KG - t) % KG * WG + wave % WG;
                        const f4 w = sums[(from * OWN + u) * 64 + lane];
#pragma unroll
                        for (int q = 0; q < 4; ++q) v[4 * e + q] += w[q];
                    });
    }
    // element e of block (i, j): row 32 i + 8 (e / 4) + 4 h + e % 4, column 32 j + l % 32
    const int row0 = m0 + wm0 + 4 * h, col0 = n0 + wn0 + l32;
    const size_t n = (size_t)g.n;
    float *const out = (p.splits > 1 ? g.ws + (size_t)blockIdx.y * g.m * n : g.out) +
                       (size_t)row0 * n + col0;
    float bias[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j)
        bias[j] = g.bias && p.splits == 1 && col0 + 32 * j < g.n ? g.bias[col0 + 32 * j] : 0.0f;
    // (the loads are waited for here: behind a branch they are taken to be on their way
    // still, and every store would wait for the store before it)
#pragma unroll
    for (int j = 0; j < JB; ++j) asm volatile("" : "+v"(bias[j]));
    const auto store = [&](auto whole) {
#pragma unroll
        for (int o = 0; o < KG; ++o)
            if (kg == o)
#pragma unroll
                for (int u = 0; u < OWN; ++u) {
                    const int q = o * OWN + u, i = q / 4 / JB, j = q / 4 % JB;
                    if (!decltype(whole)::value && col0 + 32 * j >= g.n) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int down = 32 * i + 8 * (q % 4) + e;
                        if (decltype(whole)::value || row0 + down < g.m)
                            __builtin_nontemporal_store(acc[i][j][4 * (q % 4) + e] + bias[j],
                                                        out + down * n + 32 * j);
                    }
                }
    };
    // (a check for each element costs more than its store)
    if (m0 + BM <= g.m && n0 + BN <= g.n)
        store(std::true_type());
    else
        store(std::false_type());
}

// The splits' sums (up to kMaxSplits), in their order, and the bias; four elements a
// thread (the last ones one by one), at any 4 bytes, all loads on their way first.
constexpr int kMaxSplits = 8;
__global__ void __launch_bounds__(256) join_kernel(Gemm8Args g, int splits) {
    const size_t n = (size_t)g.m * g.n;
    for (size_t i = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x); i < n;
         i += (size_t)gridDim.x * 1024) {
        if (i + 4 <= n) {
            lin8_f4u v[kMaxSplits];
#pragma unroll
            for (int j = 0; j < kMaxSplits; ++j)
                if (j < splits) v[j] = *reinterpret_cast<const lin8_f4u *>(g.ws + j * n + i);
            lin8_f4u s = v[0];
#pragma unroll
            for (int j = 1; j < kMaxSplits; ++j)
                if (j < splits) s += v[j];
            if (g.bias) {
                int col = (int)(i % (size_t)g.n);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[e] += g.bias[col];
                    if (++col == g.n) col = 0;
                }
            }
            *reinterpret_cast<lin8_f4u *>(g.out + i) = s;
        } else {
            for (size_t e = i; e < n; ++e) {
                float s = g.ws[e];
                for (int j = 1; j < splits; ++j) s += g.ws[j * n + e];
                g.out[e] = s + (g.bias ? g.bias[e % g.n] : 0.0f);
            }
        }
    }
}

// Up to MB rows of a: a workgroup of W waves takes RB rows of b and the waves share
// out the blocks of k (w, w + W, ...).  Each streams its blocks of both operands
// through two stages of its own in LDS, by DMA of whole 128-byte lines,
// so no wave waits for another until their sums are added, in wave order.  One
// operand's exponents to a DMA: lanes of both in one take a loop over the two buffers
// (1 x 64 x 14336 10.2 us, 9.2 without).  A third stage of 16 rows: 9.6 for 9.0.
template <int RB, int MB, int W>
__global__ void __launch_bounds__(64 * W) stream_kernel(Gemm8Args g) {
    constexpr int IB = (RB + 31) / 32, JB = MB / 32, Q = RB < 32 ? RB / 8 : 4;  // Q: quarters
    constexpr int STAGE = (RB + MB) * 128, ND = (RB + MB) / 8;
    constexpr int XB = (RB + 63) / 64, XA = (MB + 63) / 64;  // DMAs of exponents
    constexpr int RING = STAGE + (XB + XA) * 256;
    static_assert(W * IB * JB * Q * 1024 <= W * 2 * RING, "the sums fit");
    __shared__ __attribute__((aligned(16))) char smem[W * 2 * RING];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, h = lane >> 5;
    const int rb32 = RB < 32 ? l32 % RB : l32;  // (16 rows of b fill an operand twice)
    const int n0 = blockIdx.x * RB;
    const uint32_t kp = (uint32_t)g.blocks * 128u;
    const __amdgpu_buffer_rsrc_t rb = codes_from(g.b, n0, RB, g.n, kp);
    const __amdgpu_buffer_rsrc_t ra = codes_from(g.a, 0, MB, g.m, kp);
    const __amdgpu_buffer_rsrc_t rxb = exps_from(g.b_exps, n0, RB, g.b_tiles, g.blocks);
    const __amdgpu_buffer_rsrc_t rxa = exps_from(g.a_exps, 0, MB, g.a_tiles, g.blocks);
    // DMA d moves eight rows, those of b first
    const uint32_t off = (uint32_t)(lane / 8) * kp + (uint32_t)slot_of(lane / 8, lane % 8);
    uint32_t xb[XB], xa[XA];  // where this lane's rows have their exponents
#pragma unroll
    for (int u = 0; u < XB; ++u)
        xb[u] = exps_at(min(n0 + min(u * 64 + lane, RB - 1), g.n - 1), n0, g.b_tiles, g.blocks);
#pragma unroll
    for (int u = 0; u < XA; ++u)
        xa[u] = exps_at(min(min(u * 64 + lane, MB - 1), g.m - 1), 0, g.a_tiles, g.blocks);
    char *const ring = smem + wave * (2 * RING);
    const int a_dmas = min(MB / 8, (g.m + 7) / 8);  // (rows past g.m are not stored)
    const auto dma = [&](int i) {
        char *st = ring + (i & 1) * RING;
        const int kb = wave + i * W;
#pragma unroll
        for (int u = 0; u < XB; ++u)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rxb, (lds_void *)(st + STAGE + u * 256), 4,
                                                     (int)xb[u], kb * 4, 0, 0);
#pragma unroll
        for (int u = 0; u < XA; ++u)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rxa, (lds_void *)(st + STAGE + (XB + u) * 256), 4, (int)xa[u], kb * 4, 0, 0);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (d < RB / 8)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void *)(st + d * 1024), 16,
                                                         (int)(off + d * 8 * kp), kb * 128, 0, 0);
            else if (d - RB / 8 < a_dmas)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    ra, (lds_void *)(st + d * 1024), 16, (int)(off + (d - RB / 8) * 8 * kp),
                    kb * 128, 0, 0);
        }
    };
    f16v acc[IB][JB];
#pragma unroll
    for (int i = 0; i < IB; ++i)
#pragma unroll
        for (int j = 0; j < JB; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int count = (g.blocks - wave + W - 1) / W;  // (0 or less: none)
    if (count > 0) dma(0);
    for (int i = 0; i < count; ++i) {
        // the block has landed, and the one before it is read
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (i + 1 < count) dma(i + 1);
        const char *st = ring + (i & 1) * RING;
        const int *x = reinterpret_cast<const int *>(st + STAGE);
        float sb[IB], sa[JB];
#pragma unroll
        for (int r = 0; r < IB; ++r) sb[r] = lin8_pow2(x[32 * r + rb32]);
#pragma unroll
        for (int t = 0; t < JB; ++t) sa[t] = lin8_pow2(x[XB * 64 + 32 * t + l32]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int slot = slot_of(l32, 2 * c + h);
            bf8 fb[IB][2], fa[JB][2];
#pragma unroll
            for (int r = 0; r < IB; ++r) {
                const u4 v = *reinterpret_cast<const u4 *>(st + (32 * r + rb32) * 128 + slot);
                fb[r][0] = widen8(v[0], v[1], sb[r]);
                fb[r][1] = widen8(v[2], v[3], sb[r]);
            }
#pragma unroll
            for (int t = 0; t < JB; ++t) {
                const u4 v = *reinterpret_cast<const u4 *>(st + (RB + 32 * t + l32) * 128 + slot);
                fa[t][0] = widen8(v[0], v[1], sa[t]);
                fa[t][1] = widen8(v[2], v[3], sa[t]);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int r = 0; r < IB; ++r)
#pragma unroll
                    for (int t = 0; t < JB; ++t)
                        acc[r][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[r][q], fa[t][q],
                                                                            acc[r][t], 0, 0, 0);
        }
    }
    __syncthreads();
    f4 *const sums = reinterpret_cast<f4 *>(smem);
#pragma unroll
    for (int r = 0; r < IB; ++r)
#pragma unroll
        for (int t = 0; t < JB; ++t)
#pragma unroll
            for (int e = 0; e < Q; ++e)
                sums[((wave * IB * JB + r * JB + t) * Q + e) * 64 + lane] =
                    (f4){acc[r][t][4 * e], acc[r][t][4 * e + 1], acc[r][t][4 * e + 2],
                         acc[r][t][4 * e + 3]};
    __syncthreads();
    // quarter e of block (r, t): rows 32 r + 8 e + 4 h .. of b, row 32 t + l % 32 of a
    for (int u = wave; u < IB * JB * Q; u += W) {
        f4 s = sums[u * 64 + lane];
#pragma unroll
        for (int w = 1; w < W; ++w) s += sums[(w * IB * JB * Q + u) * 64 + lane];
        const int m = u / Q % JB * 32 + l32, n = n0 + u / Q / JB * 32 + 8 * (u % Q) + 4 * h;
        if (g.bias) s += lin8_load4<true>(g.bias, n / 4, g.n);
        if (m < g.m) lin8_store4<true>(g.out + (size_t)m * g.n, n / 4, g.n, s);
    }
}

// ---- which kernel ------------------------------------------------------------
//
// Up to 32 rows of a go to the streaming kernel.  No tiles did them faster, whole or cut
// along k (32 x 1024 x 14336 17.2 us from memory and 9.8 from the last-level cache, 18.2 and
// 12.0 in tiles; 32 x 128 x 16384 16.3 and 10.9, 19.1 and 12.2; 32 x 14336 x 4096 16.2 and
// 10.7, 19.6 and 16.4), though it does not cut k over workgroups: such a long k with so few
// rows of b leaves most CUs idle, three times the time of its bytes.
//
// More rows are priced in microseconds, every kernel with what it measured: a start, so
// much for a step along k of the workgroups that share a CU (step[i] with i + 1 of them),
// the results on their way out at 5.5 TB/s, and for products cut along k a second
// launch that joins them.  The cheapest runs.

struct Tiles {
    int bm, bn, per_cu;
    double start, step[4];
};
constexpr Tiles kTiles[] = {
    {64, 64, 4, 2.3, {0.50, 0.59, 0.82, 1.16}},
    {64, 128, 3, 1.8, {0.64, 0.98, 1.45}},
    {128, 128, 2, 2.0, {1.05, 1.85}},
    {256, 256, 1, 3.0, {3.10}},
};

double tiles_us(const Gemm8Args &g, const Tiles &t, int splits, int num_cus, Gemm8Plan *p) {
    p->bm = t.bm;
    p->bn = t.bn;
    p->tiles_m = (int)(((int64_t)g.m + t.bm - 1) / t.bm);
    p->tiles_n = (int)(((int64_t)g.n + t.bn - 1) / t.bn);
    p->per_split = g.blocks ? (g.blocks + splits - 1) / splits : 0;
    p->splits = g.blocks ? (g.blocks + p->per_split - 1) / p->per_split : 1;
    const double out = 4e-6 * g.m * (double)g.n;  // MB
    double left = (double)p->tiles_m * p->tiles_n * p->splits / num_cus;
    const double full = std::floor(left / t.per_cu);
    double step = full * t.step[t.per_cu - 1];
    left -= full * t.per_cu;
    if (left > 0) {  // between so many workgroups on every CU and one more on some
        const int most = (int)std::ceil(left);
        const double fewer = most > 1 ? t.step[most - 2] : t.step[0];
        step += fewer + (t.step[most - 1] - fewer) * (left - (most - 1));
    }
    double us = t.start + p->per_split * step + p->splits * out / 5.5;
    if (p->splits > 1) us += 3.0 + (p->splits + 1) * out / 4.5;
    return us;
}

// The streaming kernel for up to 32 or 64 rows of a.  One workgroup a CU has eight
// waves (six with 64 rows), more of them four, so that two (for 64 rows: twice the
// rows of b) share a CU: with b from memory (copies in turn, more than the last-level
// cache holds) 32 x 14336 x 4096 16.1 us, 17.7 with eight; 32 x 4096 x 4096 in 32 rows of
// b 8.6 us, 9.7 with four; 64 x 14336 x 4096 18.7 us, 24.3 with 32 rows of b; 64 x 8000 x
// 4096 13.6, 16.7 with 64.  Sixteen rows of b to a workgroup read a more often, but leave no
// CU idle and are quicker by the block, as long as one round of them is enough (32 x
// 14336 x 4096 23.5 us).  From memory and from the last-level cache, for 32 rows of b:
//   32 x 4096 x 14336 19.2 us for 23.8, 12.6 for 15.0; 32 x 4096 x 8192 11.6 for 14.5, 9.0 for 12.5
//   32 x 4096 x 4096 7.4 for 8.7, 5.8 for 6.2; 1 x 4096 x 4096 6.3 for 6.7, 5.6 for 5.6
//   32 x 1024 x 14336 17.0 for 21.7, 9.8 for 11.2; 32 x 4096 x 512 3.8 for 3.8 (the launch)
void stream_form(const Gemm8Args &g, int num_cus, Gemm8Plan *p) {
    const bool one = ((int64_t)g.n + 31) / 32 <= num_cus;
    p->rows_a = g.m <= 32 ? 32 : 64;
    const bool half = p->rows_a == 32 && ((int64_t)g.n + 15) / 16 <= num_cus;
    p->rows_b = p->rows_a == 64 && !one ? 64 : half ? 16 : 32;
    p->waves = !one ? 4 : p->rows_a == 32 ? 8 : 6;
    p->splits = 1;
}
// What it takes for 33 to 64 rows, where tiles can be quicker.
double stream_us(const Gemm8Args &g, int num_cus, const Gemm8Plan &p) {
    const double turns = std::ceil(std::ceil((double)g.n / p.rows_b) / num_cus);
    return 2.5 + turns * ((g.blocks + p.waves - 1) / p.waves) * (p.rows_b == 64 ? 1.75 : 1.3);
}

template <int BM, int BN, int KG, int MINW>
void run_tiles(const Gemm8Args &g, const Gemm8Plan &p, hipStream_t s) {
    const dim3 grid((unsigned)((p.tiles_m * p.tiles_n + 7) / 8 * 8), (unsigned)p.splits);
    gemm8_kernel<BM, BN, KG, MINW><<<grid, BM / 64 * (BN / 64) * KG * 64, 0, s>>>(g, p);
}

template <int RB, int MB, int W>
void run_stream(const Gemm8Args &g, hipStream_t s) {
    stream_kernel<RB, MB, W><<<(unsigned)(((int64_t)g.n + RB - 1) / RB), 64 * W, 0, s>>>(g);
}

}  // namespace

Gemm8Plan gemm8_plan(const Gemm8Args &g, int num_cus) {
    Gemm8Plan best{};
    if (g.m == 0 || g.n == 0) return best;
    if (g.m <= 64) stream_form(g, num_cus, &best);
    if (g.m <= 32) return best;
    double best_us = g.m <= 64 ? stream_us(g, num_cus, best) : 0.0;
    for (const Tiles &t : kTiles)
        for (int splits = 1; splits <= kMaxSplits; splits *= 2) {
            if (splits > 1 && g.blocks < 2 * splits) break;
            Gemm8Plan p{};
            const double us = tiles_us(g, t, splits, num_cus, &p);
            if (best.splits == 0 || us < best_us) {
                best_us = us;
                best = p;
            }
        }
    return best;
}

size_t gemm8_workspace(const Gemm8Args &a, const Gemm8Plan &p) {
    return p.splits > 1 ? (size_t)p.splits * a.m * a.n : 0;
}

void gemm8(const Gemm8Args &a, const Gemm8Plan &p, int num_cus, hipStream_t s) {
    if (a.m == 0 || a.n == 0) return;
    if (p.waves) {
        if (p.rows_b == 16) run_stream<16, 32, 8>(a, s);
        else if (p.rows_a == 32) p.waves == 8 ? run_stream<32, 32, 8>(a, s) : run_stream<32, 32, 4>(a, s);
        else p.rows_b == 32 ? run_stream<32, 64, 6>(a, s) : run_stream<64, 64, 4>(a, s);
        return;
    }
    if (p.bm == 256) run_tiles<256, 256, 1, 4>(a, p, s);
    else if (p.bm == 128) run_tiles<128, 128, 2, 2>(a, p, s);
    else if (p.bn == 128) run_tiles<64, 128, 2, 2>(a, p, s);
    else run_tiles<64, 64, 4, 4>(a, p, s);
    if (p.splits > 1) {
        const size_t work = ((size_t)a.m * a.n + 1023) / 1024;
        join_kernel<<<(unsigned)std::min(work, (size_t)num_cus * 16), 256, 0, s>>>(a, p.splits);
    }
}

}  // namespace k
}  // namespace clove

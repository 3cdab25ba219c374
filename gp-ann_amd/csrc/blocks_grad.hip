// blocks_grad.hip — gradients of the attention over probed cache blocks (include/gpann_blocks.h).
//
// Two passes recompute the weights p = 2^(x log2 e - lse log2 e), each stationary in what it sums: the query side walks the blocks that neighbouring query
// rows probe, as the forward does, and leaves {lse, delta} of every row; the key side has one workgroup per block, past whose keys the rows that
// probe it stream.  No sum crosses workgroups but the parts of blocks that very many rows probe, which are joined in their order: results repeat.
#include "blocks_walk.h"

#include <algorithm>

namespace gpann {

// ---- gradient of the queries ----------------------------------------------------------------------------------------------------------------
// delta = <dout, out> is what every dp is measured against; `out` was rounded, so it is off by e, the same for all of a row's keys.  The walk therefore sums
// ds' = p (dp - delta'), which is e in all, and w = sum p k beside dq' = sum ds' k: the gradient at the true delta is dq' - e w (the weights sum to 1).  Taken
// with the sum of the ds' as they were rounded for the product, that is sum ds' (k - w): the roundings then weigh k - w, not k.  The key side gets delta' + e.
// Where ds' sums to more than rounding can have done, `out` and `lse` are not of these keys alone (attention joined over several calls, whose gradients are taken
// from the joined ones): there is no such e, and nothing is corrected.
// (8192 rows of 128 dimensions in bf16, relative error of dq: 0.0017 is its own rounding, 0.0023 this, 0.0025 with the sum before the rounding, 0.0032
// uncorrected.  The products for w took 63 us when the query side took 720.)
//
// 8192 query rows of 32 heads, 8 key/value heads of 128 dimensions, 16 probes of 64 rows, by the profiler: the query side takes 563 us (three products, 188
// GFLOP: 334 TFLOP/s; with the one for w, and the columns that look at nothing, 395 are issued and the matrix cores are busy for 32 % of the cycles) and the key
// side 472 us (four products, 250 GFLOP: 530 TFLOP/s, 26 %); joining 18, counting and marking rows 8 each.  Both are bound as the forward is: two wavefronts a
// SIMD, whose reads, products and weights overlap little.  In scratch: 5 to 8 registers of the query side up to 192 dimensions, 73 to 76 at 256; 2 to 6 of the key side at 256.

// What the key side needs of a (query row, head) row: lse * log2 e (+inf: it weighs nothing) and delta.  Both arrays end with an entry of a row that weighs nothing.
struct BlocksRowInfo {
    float* lse2;
    float* delta;
};

// <dout, out>, and 1.25 times the most that rounding `out` to its type can have moved it by: half a step of every term, in binary16 at least that of its smallest numbers
template <bool BF16, int DC>
__device__ __forceinline__ float BlocksDelta(const uint16_t* out, const u32x4_t (&go)[DC / 2], float& slack) {
    u32x4_t y[DC / 2];
    BlocksLoadRows<DC / 2>(out, y);
    float delta = 0.f, size = 0.f;
#pragma unroll
    for (int s = 0; s < DC / 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = BlocksToFloat((uint16_t)y[s][i], BF16) * BlocksToFloat((uint16_t)go[s][i], BF16);
            const float hi = BlocksToFloat((uint16_t)(y[s][i] >> 16), BF16) * BlocksToFloat((uint16_t)(go[s][i] >> 16), BF16);
            delta += lo;
            delta += hi;
            size += fabsf(lo) + fabsf(hi);
            if (!BF16) size += (fabsf(BlocksToFloat((uint16_t)go[s][i], BF16)) + fabsf(BlocksToFloat((uint16_t)(go[s][i] >> 16), BF16))) * 0x1p-14f;   // 2^-25 / 2^-11
        }
    slack = BlocksSumOver4(size) * (BF16 ? 1.25f / 256.f : 1.25f / 2048.f);
    return BlocksSumOver4(delta);
}

// One query row's heads (columns r < heads), its probed rows straight from memory: the way out for rows whose neighbours' values are not finite, and for those with
// a ds that binary16 cannot hold (above 65504, where the gradients may well be in range): a column's ds are taken in units of a power of two that follows their
// largest, as the sums are when it grows.
template <bool BF16, int DC>
__device__ __forceinline__ void BlocksQueryGradRow(const BlocksArgs& a, uint32_t b, uint32_t h, uint32_t t, uint32_t head, bool live, int visible, uint32_t lane,
                                                   uint32_t* scratch, const uint16_t* out, const uint16_t* dout, const float* lse, uint16_t* dq, BlocksRowInfo rows) {
    constexpr int KS = DC / 2, N = DC / 2;
    const uint32_t r = lane & 15, g = lane >> 4;
    int block;
    int64_t ko, vo;
    const uint32_t count = BlocksGatherProbes(a, a.probes + (((int64_t)b * a.Tq + t) * a.Hkv + h) * a.P, b, visible, scratch, lane, block, ko, vo);
    u32x4_t q[KS], go[KS];
    BlocksLoadRows<KS>(a.q + b * a.qs[0] + t * a.qs[1] + head * a.qs[2] + g * 8, q);
    BlocksLoadRows<KS>(dout + b * a.os[0] + t * a.os[1] + head * a.os[2] + g * 8, go);
    float slack;
    const float delta = BlocksDelta<BF16, DC>(out + b * a.os[0] + t * a.os[1] + head * a.os[2] + g * 8, go, slack);
    const int64_t row = ((int64_t)b * a.Tq + t) * a.Hq + head;
    const float l = lse[row], lse2 = l == -__builtin_inff() ? __builtin_inff() : l * kLog2e;
    f32x4_t acc[DC];
#pragma unroll
    for (int d = 0; d < DC; ++d) acc[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float down = 1.f;   // units of the column's ds and sums: 1 / down
    const uint32_t tpb = a.bs / 16, units = count * tpb;
    BlocksCursor c(0, tpb);
    for (uint32_t u = 0; u < units; u += 2) {
        f32x4_t s[2];
        uint32_t kc[8][N];
        const bool second = u + 1 < units;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int blk = __builtin_amdgcn_readlane(block, (int)c.slot), base = (int)c.sub * 16, most = visible - 1 - blk * (int)a.bs;
            const uint16_t* k = a.k + BlocksReadLane64(ko, c.slot) + h * a.ks[2];
            const uint16_t* v = a.v + BlocksReadLane64(vo, c.slot) + h * a.vs[2] + min(base + (int)r, most) * a.vs[1] + g * 8;
            const uint16_t* kr = k + min(base + (int)r, most) * a.ks[1] + g * 8;
            f32x4_t dp = {0.f, 0.f, 0.f, 0.f};
            s[x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                s[x] = BlocksMfma<BF16>(*reinterpret_cast<const u32x4_t*>(kr + j * 32), q[j], s[x]);
                dp = BlocksMfma<BF16>(*reinterpret_cast<const u32x4_t*>(v + j * 32), go[j], dp);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                BlocksLoadColumns<N>(k + min(base + (int)g * 4 + i, most) * a.ks[1] + r * DC, kc[x * 4 + i]);
                const bool ok = (x == 0 || second) && blk * (int)a.bs + base + (int)g * 4 + i < visible;
                const float p = BlocksExp2(s[x][i] * a.scale2 - lse2);
                s[x][i] = ok ? p * (dp[i] - delta) : 0.f;
                if (!ok)
#pragma unroll
                    for (int w = 0; w < N; ++w) kc[x * 4 + i][w] = 0u;
            }
            if (x == 0 && second) c.Next();
        }
        c.Next();
        if constexpr (!BF16) {
            float most = 0.f;   // (a NaN is passed over)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(fabsf(s[0][i]), fabsf(s[1][i])));
            most = BlocksMaxOver4(most);
            if (__ballot(most * down >= 32768.f)) {
                const uint32_t e = __float_as_uint(most) >> 23;   // 2^(e - 127) <= most < 2^(e - 126)
                const float to = most * down >= 32768.f && e < 255 ? __uint_as_float((268 - e) << 23) : down, f = to / down;   // most * to: 2^14 .. 2^15
                down = to;
#pragma unroll
                for (int d = 0; d < DC; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[d][i] *= f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[0][i] *= down;
                s[1][i] *= down;
            }
        }
        const u32x4_t ds = BlocksPackOperand<BF16>(s[0], s[1]);
#pragma unroll
        for (int d = 0; d < DC; ++d) acc[d] = BlocksMfma<BF16>(BlocksColumn<N>(kc, d), ds, acc[d]);
    }
    if (!live) return;
    uint16_t* dst = dq + b * a.qs[0] + (int64_t)t * a.qs[1] + head * a.qs[2];
    const float scale = a.scale / down;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[N];
#pragma unroll
        for (int x = 0; x < N; ++x) w[x] = BlocksPack<BF16>(acc[2 * x][i] * scale, acc[2 * x + 1][i] * scale);
        BlocksStoreColumns<N>(dst + (g * 4 + i) * DC, w);
    }
    if (g == 0) {
        rows.lse2[row] = lse2;
        rows.delta[row] = delta;
    }
}

// NT tiles of 16 keys, the first at LDS byte `at`, against a wavefront's 16 columns, in pairs: a pair's logits are on the matrix cores while the weights of the one
// before are computed, and its part of the sums while those of the one behind are.  `less_delta`: minus the column's delta, four times over.
template <bool BF16, int DC, int NT, int NM, typename F>
__device__ __forceinline__ void BlocksWalkQueryGrad(float scale2, const BlocksWalkAddresses<DC>& ad, uint32_t at, const int (&start)[NM], const uint32_t (&mask)[NM],
                                                    const BlocksWalkColumns<1>& col, uint32_t g4, const u32x4_t (&q)[DC / 2], const u32x4_t (&go)[DC / 2], float lse2,
                                                    const f32x4_t& less_delta, f32x4_t (&acc)[DC], f32x4_t (&wk)[DC], f32x4_t& sds, float& off, F&& meanwhile) {
    using S = BlocksWalkShape<DC>;
    constexpr uint32_t TILE = S::D * 32;
    constexpr int KS = DC / 2, NP = NT / 2, PER = NT / NM;
    f32x4_t x[NT], y[NT];
    u32x4_t k[2][KS], v[2][KS], p, ds;
    u32x2_t kt[DC][2];
    uint32_t step[KS], turned[DC];
    auto read_rows = [&](int z, u32x4_t(&f)[2][KS], uint32_t tensor) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) f[i][s] = BlocksReadRow(step[s] + tensor + (2 * z + i) * TILE);
    };
    auto read_dimension = [&](int z, int d) {
#pragma unroll
        for (int i = 0; i < 2; ++i) kt[d][i] = BlocksReadTransposed(turned[d] + (2 * z + i) * TILE);
    };
    auto read_turned = [&](int z) {
#pragma unroll
        for (int d = 0; d < DC; ++d) read_dimension(z, d);
    };
    auto logit_step = [&](int z, int n) {   // of 4 KS: logits, then dp
        const int i = n % 2, s = n / 2 % KS;
        f32x4_t& to = n < 2 * KS ? x[2 * z + i] : y[2 * z + i];
        if (s == 0) to = n < 2 * KS ? f32x4_t{0.f, 0.f, 0.f, 0.f} : less_delta;
        to = n < 2 * KS ? BlocksMfma<BF16>(k[i][s], q[s], to) : BlocksMfma<BF16>(v[i][s], go[s], to);
    };
    auto sum_step = [&](int n) {   // of 2 DC
        const int d = n / 2;
        const u32x4_t kk = {kt[d][0][0], kt[d][0][1], kt[d][1][0], kt[d][1][1]};
        if (n % 2 == 0)
            acc[d] = BlocksMfma<BF16>(kk, ds, acc[d]);
        else
            wk[d] = BlocksMfma<BF16>(kk, p, wk[d]);
    };
    ad.RowSteps(at, step);
    read_rows(0, k, 0);
    __builtin_amdgcn_sched_barrier(0);
    read_rows(0, v, S::TENSOR);
    ad.template Dimensions<DC>(at, turned);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 2 * KS; ++n) logit_step(0, n);
    __builtin_amdgcn_sched_barrier(0);
    if (NP > 1) read_rows(1, k, 0);   // operands are read as soon as their registers are free: a full LDS latency ahead of the products
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 2 * KS; n < 4 * KS; ++n) logit_step(0, n);
    __builtin_amdgcn_sched_barrier(0);
    if (NP > 1) read_rows(1, v, S::TENSOR);
    meanwhile();   // the next stage is asked for under the products' cover
    if (NP == 1) read_turned(0);
    static_assert(NP <= 2);
#pragma unroll
    for (int z = 0; z < NP; ++z) {
        __builtin_amdgcn_sched_barrier(0);
        float less[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = (2 * z + i) / PER;
            if (i == 0 || PER == 1) {
                if (start[e] + (PER == 1 ? 16 : 32) + (PER == 4 ? 32 * z : 0) > col.seen_by_all) {
                    const int limit = col.visible[0] - start[e] - (PER == 4 ? 32 * z : 0) - (int)g4;
#pragma unroll
                    for (int j = 0; j < (PER == 1 ? 4 : 8); ++j)
                        x[2 * z + i + j / 4][j % 4] = (j / 4) * 16 + j % 4 < limit ? x[2 * z + i + j / 4][j % 4] : -__builtin_inff();
                }
            }
            less[i] = ((mask[e] >> col.in[0]) & 1) ? -lse2 : -__builtin_inff();
        }
        __builtin_amdgcn_sched_barrier(0);
        // One matrix instruction, then a step of the weights, and so on: a wavefront's vector instructions run beside its matrix instructions where they alternate
        // (64 products and 192 additions in a loop, two wavefronts a SIMD: 1326 ticks taking turns, 2353 one block after the other; this kernel 613 -> 601 us when it was changed to it).
        constexpr int STEPS = 2 * DC > 16 ? 2 * DC : 16;   // 2 DC = 4 KS products, 16 steps of the weights
#pragma unroll
        for (int n = 0; n < STEPS; ++n) {
            if (z > 0 && n < 2 * DC) sum_step(n);
            if (z > 0 && n % 2 == 1 && n < 2 * DC) read_dimension(z, n / 2);
            if (z + 1 < NP && n >= 2 * KS && n < 4 * KS) read_dimension(0, n - 2 * KS);
            if (z + 1 < NP && n < 4 * KS) logit_step(z + 1, n);
            if (n < 16) {
                const int e = n / 2, i = 2 * z + e / 4, j = e % 4;
                if (n % 2 == 0)
                    x[i][j] = __builtin_fmaf(x[i][j], scale2, less[i - 2 * z]);
                else
                    x[i][j] = BlocksExp2(x[i][j]);
                if (n % 2 == 0 && e > 0) y[2 * z + (e - 1) / 4][(e - 1) % 4] *= x[2 * z + (e - 1) / 4][(e - 1) % 4];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        y[2 * z + 1][3] *= x[2 * z + 1][3];
#pragma unroll
        for (int i = 2 * z; i < 2 * z + 2; ++i) off += (y[i][0] + y[i][1]) + (y[i][2] + y[i][3]);
        if (z > 0) sds = BlocksMfma<BF16>(BlocksOnes<BF16>(), ds, sds);
        // one rounding of p and ds to the tensors' type, as of p in the forward
        p = BlocksPackOperand<BF16>(x[2 * z], x[2 * z + 1]);
        ds = BlocksPackOperand<BF16>(y[2 * z], y[2 * z + 1]);
    }
#pragma unroll
    for (int n = 0; n < 2 * DC; ++n) sum_step(n);
    sds = BlocksMfma<BF16>(BlocksOnes<BF16>(), ds, sds);
}

// ... where the sums and the operands of a row leave too few registers for that: one pair of tiles, operands in batches
template <bool BF16, int DC, int NM, typename F>
__device__ __forceinline__ void BlocksWalkQueryGradTight(float scale2, const BlocksWalkAddresses<DC>& ad, uint32_t at, const int (&start)[NM], const uint32_t (&mask)[NM],
                                                         const BlocksWalkColumns<1>& col, uint32_t g4, const u32x4_t (&q)[DC / 2], const u32x4_t (&go)[DC / 2],
                                                         float lse2, float delta, f32x4_t (&acc)[DC], f32x4_t (&wk)[DC], f32x4_t& sds, float& off, F&& meanwhile) {
    using S = BlocksWalkShape<DC>;
    constexpr uint32_t TILE = S::D * 32;
    constexpr int KS = DC / 2, SOME = DC > 12 ? KS / 4 : KS / 2, TURNED = DC > 12 ? 2 : 4;
    f32x4_t x[2], y[2];
    meanwhile();
    auto product = [&](uint32_t tensor, const u32x4_t(&with)[KS], f32x4_t(&to)[2]) {
        uint32_t step[KS];
        ad.RowSteps(at, step);
#pragma unroll
        for (int s0 = 0; s0 < KS; s0 += SOME) {
            u32x4_t f[2][SOME];
#pragma unroll
            for (int s = 0; s < SOME; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) f[i][s] = BlocksReadRow(step[s0 + s] + tensor + i * TILE);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < SOME; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) to[i] = BlocksMfma<BF16>(f[i][s], with[s0 + s], to[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = y[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    product(0, q, x);
    product(S::TENSOR, go, y);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int first = start[i * NM / 2] + (NM == 1 ? i * 16 : 0);
        if (first + 16 > col.seen_by_all) {
            const int limit = col.visible[0] - first - (int)g4;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = j < limit ? x[i][j] : -__builtin_inff();
        }
        const float less = ((mask[i * NM / 2] >> col.in[0]) & 1) ? -lse2 : -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[i][j] = BlocksExp2(__builtin_fmaf(x[i][j], scale2, less));
            y[i][j] = x[i][j] * (y[i][j] - delta);
        }
        off += (y[i][0] + y[i][1]) + (y[i][2] + y[i][3]);
    }
    const u32x4_t p = BlocksPackOperand<BF16>(x[0], x[1]), ds = BlocksPackOperand<BF16>(y[0], y[1]);   // rounded as above
    sds = BlocksMfma<BF16>(BlocksOnes<BF16>(), ds, sds);
    uint32_t turned[DC];
    ad.template Dimensions<DC>(at, turned);
#pragma unroll
    for (int d0 = 0; d0 < DC; d0 += TURNED) {
        u32x2_t kt[TURNED][2];
#pragma unroll
        for (int d = 0; d < TURNED; ++d)
#pragma unroll
            for (int i = 0; i < 2; ++i) kt[d][i] = BlocksReadTransposed(turned[d0 + d] + i * TILE);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < TURNED; ++d) {
            const u32x4_t kk = {kt[d][0][0], kt[d][0][1], kt[d][1][0], kt[d][1][1]};
            acc[d0 + d] = BlocksMfma<BF16>(kk, ds, acc[d0 + d]);
            wk[d0 + d] = BlocksMfma<BF16>(kk, p, wk[d0 + d]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// NT: tiles taken at a time; NM: of how many blocks they may be
template <bool BF16, int DC, int NT, int NM>
__global__ void __launch_bounds__(512) BlocksQueryGradKernel(BlocksArgs a, uint32_t tpw, uint32_t mtiles, uint32_t tiles, const uint16_t* __restrict__ out,
                                                             const uint16_t* __restrict__ dout, const float* __restrict__ lse, uint16_t* __restrict__ dq,
                                                             BlocksRowInfo info) {
    TakeWholeRegisterFile();
    using S = BlocksWalkShape<DC>;
    constexpr int KS = DC / 2;
    extern __shared__ __attribute__((aligned(1024))) char s_walk[];
    __shared__ uint32_t s_count, s_scratch[8][64];
    __shared__ float s_slack[8][16];
    const BlocksWalkTables<DC> tab(s_walk);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t pair, tile;
    if (!BlocksPairOf(blockIdx.x, a.B * a.Hkv, tiles, pair, tile)) return;
    BlocksWalkRows w;
    w.b = pair / a.Hkv;
    w.h = pair % a.Hkv;
    w.wt0 = (tiles - 1 - tile) * 8;
    w.tpw = tpw;
    w.mtiles = mtiles;
    w.n = BlocksKvLen(a, w.b);
    w.m = BlocksQLen(a, w.b);
    const BlocksWalkColumns<1> col(a, w, wave, r);
    {   // rows behind the sequence's last
        const uint32_t t = col.t0 + (mtiles > 1 ? 0 : min(r, col.cols - 1) / a.G);
        if ((int)t >= w.m && t < a.Tq && r < col.cols) {
            uint16_t* dst = dq + w.b * a.qs[0] + (int64_t)t * a.qs[1] + (w.h * a.G + (mtiles > 1 ? col.mt * 16 + r : r % a.G)) * a.qs[2] + g * 4;
#pragma unroll
            for (int d = 0; d < DC; ++d) *reinterpret_cast<u32x2_t*>(dst + d * 16) = u32x2_t{0u, 0u};
        }
    }
    if ((int)w.FirstRow(w.wt0) >= w.m) return;
    const uint32_t blocks = ((uint32_t)BlocksVisible(a, w.n, w.m, (int)w.EndRow() - 1) + a.bs - 1) / a.bs, tpb = a.bs / 16;

    const float scale2 = a.scale2 == 0.f ? 1.f : fabsf(a.scale2);
    u32x4_t q[KS], go[KS];
    const int64_t at_q = w.b * a.qs[0] + (int64_t)col.Row(w, 0) * a.qs[1] + col.head[0] * a.qs[2] + g * 8;
    const int64_t at_o = w.b * a.os[0] + (int64_t)col.Row(w, 0) * a.os[1] + col.head[0] * a.os[2] + g * 8;
    BlocksLoadRows<KS>(a.q + at_q, q);
    BlocksLoadRows<KS>(dout + at_o, go);
    if (a.scale2 <= 0.f)
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] = a.scale2 == 0.f ? u32x4_t{0u, 0u, 0u, 0u} : q[s] ^ 0x80008000u;
    float slack;
    float delta = BlocksDelta<BF16, DC>(out + at_o, go, slack);
    if (g == 0) s_slack[wave][r] = slack;   // (wanted after the walk: a register less in it)
    const int64_t row = ((int64_t)w.b * a.Tq + col.Row(w, 0)) * a.Hq + col.head[0];
    const float l = lse[row], lse2 = l == -__builtin_inff() ? __builtin_inff() : l * kLog2e;   // an empty row weighs nothing
    const BlocksWalkAddresses<DC> ad(lane);
    f32x4_t acc[DC], wk[DC], sds = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DC; ++d) acc[d] = wk[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float off = 0.f;
    f32x4_t less_delta = {-delta, -delta, -delta, -delta};   // (where the products start from it)
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[s]), "+v"(go[s]));
    if (DC <= 8) asm volatile("" : "+v"(less_delta));
    const BlocksWalker<DC> walk(a, wave, lane);
    const uint32_t lds = BlocksLdsAddress(s_walk);

    for (uint32_t window = 0; window < blocks; window += S::WINDOW) {
        const uint32_t in_window = min(S::WINDOW, blocks - window);
        const uint32_t units = BlocksWalkList<DC>(a, w, window, in_window, tab, &s_count) * tpb, stages = (units + 3) / 4;
        BlocksWalkStage now = {}, next = {};   // of the stages that are multiplied and loaded now
        BlocksWalkSource from = {};
        if (stages) from = walk.Describe(a, w, tab, window, 0, units, col.seen_by_any, next);
        for (uint32_t s = 0; s < S::GROUP && s < stages; ++s) walk.Load(from, s, lds + s * S::STAGE);
        for (uint32_t s = 0; s < stages; ++s) {
            const uint32_t ahead = s + S::GROUP, at = lds + s % S::BUFFERS * S::STAGE;
            if (s % S::GROUP == 0) {
                if (s % kDescribed == 0) now = next;
                if (ahead % kDescribed == 0 && ahead < stages) from = walk.Describe(a, w, tab, window, ahead, units, col.seen_by_any, next);
                BlocksDmaWait<0>();
                BlocksStageBarrier();   // this group has landed, and nobody reads the one before any more
            }
            bool asked = false;
            auto load = [&]() {
                if (ahead < stages && !asked) walk.Load(from, ahead, lds + ahead % S::BUFFERS * S::STAGE);
                asked = true;
            };
#pragma unroll 1
            for (uint32_t z = 0; z < 4; z += NT) {
                const uint32_t first = s % kDescribed * 4 + z;
                int start[NM];
                uint32_t mask[NM], any = 0;
#pragma unroll
                for (uint32_t y = 0; y < NM; ++y) {
                    start[y] = __builtin_amdgcn_readlane(now.start, (int)(first + y * (NT / NM)));
                    mask[y] = (uint32_t)__builtin_amdgcn_readlane((int)now.mask, (int)(first + y * (NT / NM)));
                    any |= mask[y];
                }
                if (any) {
                    if constexpr (DC > 8)
                        BlocksWalkQueryGradTight<BF16, DC>(scale2, ad, at + z * S::D * 32, start, mask, col, g * 4, q, go, lse2, delta, acc, wk, sds, off, load);
                    else
                        BlocksWalkQueryGrad<BF16, DC, NT>(scale2, ad, at + z * S::D * 32, start, mask, col, g * 4, q, go, lse2, less_delta, acc, wk, sds, off, load);
                }
            }
            load();
        }
        __syncthreads();
    }
    off = BlocksSumOver4(off);
    float bad = off * 0.f;
    BlocksWaveSync();
    const bool own = fabsf(off) <= s_slack[wave][r];   // what the rounding of `out` explains; else `out` and `lse` are of more keys than these
    const float e = own ? sds[0] : 0.f;
#pragma unroll
    for (int d = 0; d < DC; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[d][i] -= e * wk[d][i];
            bad += acc[d][i] * 0.f;
        }
    if (__ballot(bad != 0.f)) {   // as in the forward: a value that is not finite may have met a weight 0
        const uint32_t heads = mtiles > 1 ? col.cols : a.G, head = w.h * a.G + col.mt * 16 + min(r, heads - 1);
        for (uint32_t x = 0; x < col.rows; ++x)
            BlocksQueryGradRow<BF16, DC>(a, w.b, w.h, col.t0 + x, head, r < heads, BlocksVisible(a, w.n, w.m, (int)(col.t0 + x)), lane, s_scratch[wave], out, dout, lse,
                                         dq, info);
        return;
    }
    if (!col.live[0]) return;
    uint16_t* dst = dq + w.b * a.qs[0] + (int64_t)(col.t0 + col.in[0]) * a.qs[1] + col.head[0] * a.qs[2] + g * 4;
#pragma unroll
    for (int d = 0; d < DC; ++d)
        *reinterpret_cast<u32x2_t*>(dst + d * 16) =
            u32x2_t{BlocksPack<BF16>(acc[d][0] * a.scale, acc[d][1] * a.scale), BlocksPack<BF16>(acc[d][2] * a.scale, acc[d][3] * a.scale)};
    if (g == 0) {
        info.lse2[row] = lse2;
        info.delta[row] = own ? delta + off : delta;
    }
}

// ---- which query rows probe a block -------------------------------------------------------------------------------------------------------------
// One workgroup per pair, kMarkRows query rows and kMarkBlocks blocks: bits are set in LDS and every word is written, so nothing has to be cleared
__global__ void __launch_bounds__(256) BlocksBitsKernel(BlocksArgs a, uint32_t words, uint32_t* __restrict__ bits) {
    __shared__ uint32_t s_bits[kMarkBlocks * (kMarkRows / 32)];
    constexpr uint32_t W = kMarkRows / 32;
    const uint32_t pair = blockIdx.x, b = pair / a.Hkv, h = pair % a.Hkv, t0 = blockIdx.y * kMarkRows, window = blockIdx.z * kMarkBlocks, tid = threadIdx.x;
    const uint32_t in_window = min(kMarkBlocks, a.nblk - window);
    const int n = BlocksKvLen(a, b), m = BlocksQLen(a, b);
    for (uint32_t i = tid; i < in_window * W; i += 256) s_bits[i] = 0;
    __syncthreads();
    const uint32_t rows = min(kMarkRows, a.Tq - t0);
    for (uint32_t i = tid; i < rows * a.P; i += 256) {
        const uint32_t in = i / a.P, t = t0 + in;
        const int p = a.probes[(((int64_t)b * a.Tq + t) * a.Hkv + h) * a.P + i % a.P];
        if (p < (int)window || (uint32_t)p >= window + in_window || (int64_t)p * a.bs >= BlocksVisible(a, n, m, (int)t)) continue;
        atomicOr(s_bits + ((uint32_t)p - window) * W + in / 32, 1u << (in & 31));
    }
    __syncthreads();
    for (uint32_t i = tid; i < in_window * W; i += 256) {
        const uint32_t block = window + i / W, word = t0 / 32 + i % W;
        uint32_t x = s_bits[i];
        int64_t ko, vo;
        if (x && a.table && !BlocksBase(a, b, (int)block, ko, vo)) x = 0;
        if (word < words) bits[((uint64_t)pair * a.nblk + block) * words + word] = x;
    }
}

gpann_status BlocksMarkProbes(const BlocksArgs& a, uint32_t words, uint32_t* bits, hipStream_t st) {
    const dim3 grid(a.B * a.Hkv, (a.Tq + kMarkRows - 1) / kMarkRows, (a.nblk + kMarkBlocks - 1) / kMarkBlocks);
    hipLaunchKernelGGL(BlocksBitsKernel, grid, dim3(256), 0, st, a, words, bits);
    GPANN_HIP_TRY(hipGetLastError());
    return GPANN_OK;
}

// ---- gradients of the keys and values -------------------------------------------------------------------------------------------------------
// A block's query rows are taken in parts of `part`: every block has one part, whose workgroup writes the gradients, unless more rows probe it; then every
// part leaves its sums in a slot of its own and they are added afterwards, in order.
struct BlocksPart {
    uint32_t block, index;
    int slot;   // -1: the block's only part
};
// one workgroup per pair: counts[pair][block] of its query rows, parts[pair][capacity], used[pair], first_slot[pair][block]
__global__ void __launch_bounds__(1024) BlocksPartsKernel(BlocksArgs a, uint32_t words, uint32_t part, uint32_t capacity, const uint32_t* __restrict__ bits,
                                                          uint32_t* __restrict__ counts, BlocksPart* __restrict__ parts, uint32_t* __restrict__ used,
                                                          int* __restrict__ first_slot, BlocksRowInfo info) {
    __shared__ uint32_t s_n[1024], s_sum[16], s_slots[16];
    const uint32_t pair = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    uint32_t base = 0, slots = 0;
    for (uint32_t j0 = 0; j0 < a.nblk; j0 += 1024) {
        const uint32_t in = min(1024u, a.nblk - j0);
        for (uint32_t j = wave; j < in; j += 16 * 8) {   // eight blocks' words on their way at a time
            const uint32_t* row[8];
            uint32_t c[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                row[i] = bits + ((uint64_t)pair * a.nblk + j0 + min(j + 16 * i, in - 1)) * words;
                c[i] = 0;
            }
            for (uint32_t w = lane; w < words; w += 64)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) c[i] += (uint32_t)__popc(row[i][w]);
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                for (int s = 32; s > 0; s >>= 1) c[i] += __shfl_xor(c[i], s);
                if (lane == 0 && j + 16 * i < in) s_n[j + 16 * i] = c[i];
            }
        }
        __syncthreads();
        const uint32_t j = j0 + tid, rows = tid < in ? s_n[tid] : 0, n = tid < in ? max(1u, (rows + part - 1) / part) : 0, m = n > 1 ? n : 0;
        uint32_t x = n, y = m;   // inclusive sums over the wavefront, then over the workgroup
        for (int s = 1; s < 64; s <<= 1) {
            const uint32_t x1 = __shfl_up(x, s), y1 = __shfl_up(y, s);
            if ((int)lane >= s) {
                x += x1;
                y += y1;
            }
        }
        if (lane == 63) {
            s_sum[wave] = x;
            s_slots[wave] = y;
        }
        __syncthreads();
        uint32_t at = base + x - n, slot = slots + y - m;
        for (uint32_t w = 0; w < 16; ++w) {
            if (w < wave) {
                at += s_sum[w];
                slot += s_slots[w];
            }
            base += s_sum[w];
            slots += s_slots[w];
        }
        for (uint32_t i = 0; i < n; ++i) parts[(uint64_t)pair * capacity + at + i] = BlocksPart{j, i, n > 1 ? (int)(slot + i) : -1};
        if (tid < in) {
            counts[(uint64_t)pair * a.nblk + j] = rows;
            first_slot[(uint64_t)pair * a.nblk + j] = n > 1 ? (int)slot : -1;
        }
        __syncthreads();
    }
    if (tid == 0) used[pair] = base;
    if (tid == 0 && pair == 0) {
        info.lse2[(uint64_t)a.B * a.Tq * a.Hq] = __builtin_inff();
        info.delta[(uint64_t)a.B * a.Tq * a.Hq] = 0.f;
    }
}

// Shape of the key side: a workgroup holds 64 keys (four 16-key tiles), ND wavefronts a tile each take 1 / ND of the dimensions of its sums (where both would
// not fit a wavefront's registers, or a block has fewer tiles than there are wavefronts), and RGS groups of wavefronts take 32 of a stage's 32 RGS rows each.
// Four stages: one being read transposed, the next by rows, one in flight, one being asked for.
template <int DC, int RGS>
struct BlocksKeyShape {
    static constexpr uint32_t D = DC * 16, CPR = D / 8, ROWS = 32 * RGS, TENSOR = ROWS * D * 2, STAGE = 2 * TENSOR + 1024, BUFFERS = 4;
};

// A wavefront's sums once more, 16 keys (a lane's own: `key`, as its column of the products) and dimensions dim0 .. of the rows first .. first + 31, first + step ..:
// in binary32, row by row, and only of rows that see the key.  In the products a row that does not is a weight 0, and 0 times a value that is not finite is none
// that belongs there; and a ds above 65504 is an infinity in binary16.  So a wavefront whose sums are not finite comes here.  (8192 rows of 32 heads of 128 dimensions, the whole training step: 1.4 ms, with an
// infinity in one row's dout 3.6 ms, in every row's 12.1 ms.)
template <bool BF16, int DC, int OD>
__device__ __forceinline__ void BlocksKeyGradAgain(const BlocksArgs& a, uint32_t b, uint32_t h, int n, int m, const uint32_t* list, uint32_t rows, uint32_t first, uint32_t step,
                                                   int key, uint32_t dim0, uint32_t lane, const u32x4_t (&kf)[DC / 2], const u32x4_t (&vf)[DC / 2], float scale2,
                                                   const uint16_t* dout, BlocksRowInfo info, f32x4_t (&ak)[OD], f32x4_t (&av)[OD]) {
    const uint32_t r = lane & 15, g = lane >> 4;
    const uint16_t* q0 = a.q + b * a.qs[0] + (int64_t)h * a.G * a.qs[2];
    const uint16_t* o0 = dout + b * a.os[0] + (int64_t)h * a.G * a.os[2];
#pragma unroll
    for (int d = 0; d < OD; ++d) ak[d] = av[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (uint32_t at = first; at < rows; at += at % 32 == 16 ? step - 16 : 16) {
        const uint32_t row = min(at + r, rows - 1), mine = list[row / a.G];
        const uint16_t* q = q0 + (int64_t)mine * a.qs[1] + (int64_t)(row % a.G) * a.qs[2] + g * 8;
        const uint16_t* o = o0 + (int64_t)mine * a.os[1] + (int64_t)(row % a.G) * a.os[2] + g * 8;
        f32x4_t x = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < DC / 2; ++j) {
            x = BlocksMfma<BF16>(*reinterpret_cast<const u32x4_t*>(q + j * 32), kf[j], x);
            dp = BlocksMfma<BF16>(*reinterpret_cast<const u32x4_t*>(o + j * 32), vf[j], dp);
        }
        float p[4], ds[4];   // of rows at + 4 g + i and the lane's key; a weight -1: the row does not see it
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t y = min(at + g * 4 + i, rows - 1), t = list[y / a.G], which = (b * a.Tq + t) * a.Hq + h * a.G + y % a.G;   // (checked: below 2^32)
            p[i] = at + g * 4 + i < rows && key < BlocksVisible(a, n, m, (int)t) ? BlocksExp2(__builtin_fmaf(x[i], scale2, -info.lse2[which])) : -1.f;
            ds[i] = p[i] * (dp[i] - info.delta[which]);
        }
        for (uint32_t y = 0; y < 16 && at + y < rows; y += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t z = min(at + y + i, rows - 1), t = list[z / a.G];
                const uint16_t* qz = q0 + (int64_t)t * a.qs[1] + (int64_t)(z % a.G) * a.qs[2] + dim0 + r;
                const uint16_t* oz = o0 + (int64_t)t * a.os[1] + (int64_t)(z % a.G) * a.os[2] + dim0 + r;
                float weight[4], slope[4];   // of keys 4 g + k: the sums' rows
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    weight[k] = __shfl(p[i], (int)(y * 4 + g * 4) + k);
                    slope[k] = __shfl(ds[i], (int)(y * 4 + g * 4) + k);
                }
#pragma unroll
                for (int d = 0; d < OD; ++d) {
                    const float qd = BlocksToFloat(qz[d * 16], BF16), od = BlocksToFloat(oz[d * 16], BF16);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        ak[d][k] = weight[k] == -1.f ? ak[d][k] : __builtin_fmaf(slope[k], qd, ak[d][k]);
                        av[d][k] = weight[k] == -1.f ? av[d][k] : __builtin_fmaf(weight[k], od, av[d][k]);
                    }
                }
            }
    }
}

template <bool BF16, int DC, int ND, int RGS>
__global__ void __launch_bounds__(512) BlocksKeyGradKernel(BlocksArgs a, uint32_t words, uint32_t part_rows, uint32_t capacity, uint32_t slots, uint32_t groups,
                                                           uint32_t per_pair, const uint32_t* __restrict__ bits, const BlocksPart* __restrict__ parts,
                                                           const uint32_t* __restrict__ used, const uint16_t* __restrict__ dout, BlocksRowInfo info,
                                                           uint16_t* __restrict__ dk, uint16_t* __restrict__ dv, float* __restrict__ partial) {
    TakeWholeRegisterFile();
    using W = BlocksWalkShape<DC>;
    using S = BlocksKeyShape<DC, RGS>;
    constexpr int KS = DC / 2, D = DC * 16, OD = DC / ND;
    constexpr bool TIGHT = DC > 8;   // too few registers for operands of two products at a time: every one is read right before its use
    extern __shared__ __attribute__((aligned(1024))) char s_keys[];   // stages {Q rows, dO rows, lse2, delta}; afterwards the sums of the row groups; the row list behind
    uint32_t* s_list = reinterpret_cast<uint32_t*>(s_keys + S::BUFFERS * S::STAGE);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t pair, x;
    if (!BlocksPairOf(blockIdx.x, a.B * a.Hkv, per_pair, pair, x)) return;
    const uint32_t group = x % groups, item = x / groups;
    if (item >= used[pair]) return;
    const BlocksPart part = parts[(uint64_t)pair * capacity + item];
    const uint32_t b = pair / a.Hkv, h = pair % a.Hkv, tpb = a.bs / 16, kts = min(4u, tpb - group * 4);
    const int n = BlocksKvLen(a, b), m = BlocksQLen(a, b);
    const uint32_t kt = wave % kts, hd = wave / kts % ND, group_of = wave / (kts * ND);
    const bool works = group_of < RGS;   // wavefronts beyond kts * ND * RGS load, and repeat another's products for nothing
    const uint32_t rg = group_of % RGS;
    const uint32_t in_block = (group * 4 + kt) * 16;
    const int key = (int)(part.block * a.bs + in_block + r);

    u32x4_t kf[KS], vf[KS];
    const int last_row = n - 1 - (int)(part.block * a.bs);
    if (last_row >= 0) {   // (a block behind the sequence's end has no query rows either)
        int64_t ko, vo;
        (void)BlocksBase(a, b, (int)part.block, ko, vo);
        const int row = min((int)(in_block + r), last_row);
        BlocksLoadRows<KS>(a.k + ko + h * a.ks[2] + row * a.ks[1] + g * 8, kf);
        BlocksLoadRows<KS>(a.v + vo + h * a.vs[2] + row * a.vs[1] + g * 8, vf);
    }
    // the rows of this part: ranks [index * part_rows, ...) among the set bits, 512 words at a time
    __shared__ uint32_t s_words[8];
    uint32_t listed;
    {
        const uint32_t* row_bits = bits + ((uint64_t)pair * a.nblk + part.block) * words;
        const uint32_t lo = part.index * part_rows, hi = lo + part_rows;
        uint32_t before = 0;
        for (uint32_t w0 = 0; w0 < words && before < hi; w0 += 512) {
            uint32_t w = w0 + threadIdx.x < words ? row_bits[w0 + threadIdx.x] : 0u;
            const uint32_t c = (uint32_t)__popc(w);
            uint32_t sum = c;
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t y = __shfl_up(sum, s);
                if ((int)lane >= s) sum += y;
            }
            if (lane == 63) s_words[wave] = sum;
            __syncthreads();
            uint32_t rank = before + sum - c;
            for (uint32_t y = 0; y < 8; ++y) {
                if (y < wave) rank += s_words[y];
                before += s_words[y];
            }
            while (w) {
                if (rank >= lo && rank < hi) s_list[rank - lo] = (w0 + threadIdx.x) * 32 + (uint32_t)__ffs(w) - 1;
                ++rank;
                w &= w - 1;
            }
            __syncthreads();
        }
        listed = before > lo ? min(before, hi) - lo : 0;
    }
    const uint32_t rows = listed * a.G, stages = (rows + S::ROWS - 1) / S::ROWS;

    f32x4_t ak[OD], av[OD];
#pragma unroll
    for (int d = 0; d < OD; ++d) ak[d] = av[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (stages > 0) {
        const float scale2 = a.scale2 == 0.f ? 1.f : fabsf(a.scale2);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (a.scale2 <= 0.f) kf[s] = a.scale2 == 0.f ? u32x4_t{0u, 0u, 0u, 0u} : kf[s] ^ 0x80008000u;   // the scale's sign, on the keys' side here
            asm volatile("" : "+v"(kf[s]), "+v"(vf[s]));
        }
        const BlocksWalkAddresses<DC> ad(lane, hd * OD);
        const uint32_t lds = BlocksLdsAddress(s_keys);
        // Row i of the part: query row list[i / G], head i % G of the group.  A wavefront asks for PER / 8 pieces of 64 / CPR rows of both tensors a stage,
        // the last one for the rows' numbers too; `place`: what a lane adds to a row's address.  Offsets are in units of 16 bytes: a head's stride, of up to 2^31
        // elements, then fits 32 bits (in bytes it would not), and the shift is part of the addition to the base.
        constexpr uint32_t PER = S::ROWS * S::CPR / 64, PIECES = (PER + 7) / 8;
        const uint32_t inverse = a.G > 1 ? 0xFFFFFFFFu / a.G + 1 : 0;
        const char* q0 = reinterpret_cast<const char*>(a.q + b * a.qs[0] + (int64_t)h * a.G * a.qs[2]);
        const char* o0 = reinterpret_cast<const char*>(dout + b * a.os[0] + (int64_t)h * a.G * a.os[2]);
        const uint32_t qrow = (uint32_t)(a.qs[1] / 8), orow = (uint32_t)(a.os[1] / 8), qhead = (uint32_t)(a.qs[2] / 8), ohead = (uint32_t)(a.os[2] / 8);
        uint32_t piece_row[PIECES], place[PIECES];
#pragma unroll
        for (uint32_t y = 0; y < PIECES; ++y) {
            const uint32_t at = (wave + 8 * y) * 64 + lane;
            piece_row[y] = at / S::CPR;
            place[y] = W::Slot(at % S::CPR, piece_row[y] % 16);
        }
        auto row_of = [&](uint32_t i, uint32_t& t, uint32_t& head) {
            const uint32_t in = inverse ? __umulhi(i, inverse) : i;   // i / G, exact below 2^16
            t = s_list[in];
            head = i - in * a.G;
        };
        auto load_rows = [&](uint32_t s, uint32_t y, uint32_t to) {
            const uint32_t j = wave + 8 * y;
            if (PER % 8 != 0 && j >= PER) return;
            uint32_t t, head;
            row_of(min(s * S::ROWS + piece_row[y], rows - 1), t, head);
            const uint64_t q_at = (uint64_t)head * qhead + place[y], o_at = (uint64_t)head * ohead + place[y];
            BlocksDmaFrom(q0 + (((uint64_t)t * qrow + q_at) << 4), to + j * 1024);
            BlocksDmaFrom(o0 + (((uint64_t)t * orow + o_at) << 4), to + S::TENSOR + j * 1024);
        };
        auto load_info = [&](uint32_t s, uint32_t to) {
            if (wave != 7) return;
            const uint32_t i = s * S::ROWS + lane;
            uint32_t t, head;
            row_of(min(i, rows - 1), t, head);
            const uint32_t at = i < rows ? ((b * a.Tq + t) * a.Hq + h * a.G + head) : a.B * a.Tq * a.Hq;   // a row that weighs nothing (checked: below 2^32)
            if (lane < S::ROWS) {
                BlocksDmaWordFrom(info.lse2 + at, to + 2 * S::TENSOR);
                BlocksDmaWordFrom(info.delta + at, to + 2 * S::TENSOR + 256);
            }
        };
        const uint32_t mine = 2 * (PER / 8 + (wave < PER % 8 ? 1 : 0)) + (wave == 7 ? 2 : 0);   // DMA instructions of this wavefront per stage
        for (uint32_t s = 0; s + 1 < S::BUFFERS && s < stages; ++s) {
            for (uint32_t y = 0; y < (PER + 7) / 8; ++y) load_rows(s, y, lds + s * S::STAGE);
            load_info(s, lds + s * S::STAGE);
        }
        auto wait = [&](uint32_t s, uint32_t behind) {   // until stage s has landed, with `behind` stages after it in flight (if there are as many)
            BlocksDmaWaitFor(mine * min(behind, stages - 1 - min(s, stages - 1)));
            BlocksStageBarrier();
        };
        const uint32_t by_info = lds + 2 * S::TENSOR + (rg * 32 + g * 4) * 4, by_row = lds + rg * 2 * D * 32;
        auto rows_of = [&](uint32_t stage, uint32_t tensor, u32x4_t(&f)[2][KS]) {
            uint32_t step[KS];
            ad.RowSteps(by_row + stage, step);
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int y = 0; y < 2; ++y) f[y][j] = BlocksReadRow(step[j] + tensor + y * D * 32);
        };
        auto turned_of = [&](uint32_t stage, uint32_t tensor, u32x2_t(&f)[OD][2]) {
            uint32_t turned[OD];
            ad.template Dimensions<OD>(by_row + stage, turned);
#pragma unroll
            for (int d = 0; d < OD; ++d)
#pragma unroll
                for (int y = 0; y < 2; ++y) f[d][y] = BlocksReadTransposed(turned[d] + tensor + y * D * 32);
        };
        auto product = [&](const u32x4_t(&f)[2][KS], const u32x4_t(&keys)[KS], f32x4_t(&x)[2]) {
#pragma unroll
            for (int y = 0; y < 2; ++y) x[y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int y = 0; y < 2; ++y) x[y] = BlocksMfma<BF16>(f[y][j], keys[j], x[y]);
        };
        // The four products of a stage in a pipeline: while stage s's weights are computed, stage s + 1's logits are on the matrix cores.  LDS reads go out a
        // phase before the products that use them; the scheduling barriers keep the phases, inside one the compiler interleaves.
        // rows of this part that do not see the whole block: at most a block's query rows, the first of the list (and none but partly visible keys: the end)
        const int block_end = min((int)((part.block + 1) * a.bs), n);
        const bool tail = (int)((part.block + 1) * a.bs) > n;
        uint32_t partly = tail ? rows : 0;
        if (a.causal && !tail) partly = BlocksVisible(a, n, m, (int)s_list[0]) < block_end ? min(rows, a.bs * a.G) : 0;
        f32x4_t p[2], ds[2];
        u32x4_t dso = {0u, 0u, 0u, 0u};   // of the stage before: its part of the keys' sums is added behind the next barrier, while the first reads are on their way
        u32x2_t qt[OD][2];
#pragma unroll
        for (int d = 0; d < OD; ++d) qt[d][0] = qt[d][1] = u32x2_t{0u, 0u};
        auto add_keys = [&]() {
#pragma unroll
            for (int d = 0; d < OD; ++d) ak[d] = BlocksMfma<BF16>(dso, u32x4_t{qt[d][0][0], qt[d][0][1], qt[d][1][0], qt[d][1][1]}, ak[d]);
        };
        wait(0, 2);
        {
            u32x4_t f[2][KS];
            rows_of(0, 0, f);
            product(f, kf, p);
            rows_of(0, S::TENSOR, f);
            product(f, vf, ds);
        }
        for (uint32_t s = 0; s < stages; ++s) {
            const uint32_t stage = (s & 3) * S::STAGE, next = ((s + 1) & 3) * S::STAGE, to = lds + ((s + 3) & 3) * S::STAGE;
            const bool more = s + 3 < stages;
            wait(s + 1, 1);   // (behind the last stage: rows of an earlier one, whose products nobody uses)
            u32x4_t f[2][KS], f1[2][KS], about[2][2];   // lse2 and delta of the lane's eight rows
            u32x2_t ot[OD][2];
            f32x4_t p1[2], ds1[2];
            rows_of(next, 0, f);
            {
                uint32_t at = by_info + stage;
                asm volatile("" : "+v"(at));
#pragma unroll
                for (int i = 0; i < 4; ++i) about[i >> 1][i & 1] = BlocksReadRow(at + (i >> 1) * 256 + (i & 1) * 64);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!TIGHT) add_keys();
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!TIGHT) rows_of(next, S::TENSOR, f1);
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_rows(s + 3, 0, to);
            __builtin_amdgcn_sched_barrier(0);
            product(f, kf, p1);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[y][i] = BlocksExp2(__builtin_fmaf(p[y][i], scale2, -__uint_as_float(about[0][y][i])));
                    ds[y][i] = p[y][i] * (ds[y][i] - __uint_as_float(about[1][y][i]));
                }
            // the first rows of the list may see only a part of the block
            if (s * S::ROWS < partly) {
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t row = min(s * S::ROWS + rg * 32 + y * 16 + g * 4 + i, rows - 1), in = inverse ? __umulhi(row, inverse) : row;
                        const bool ok = key < BlocksVisible(a, n, m, (int)s_list[in]);
                        p[y][i] = ok ? p[y][i] : 0.f;
                        ds[y][i] = ok ? ds[y][i] : 0.f;
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (TIGHT)
                rows_of(next, S::TENSOR, f1);
            else
                turned_of(stage, S::TENSOR, ot);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!BF16)   // a weight is at most 1 and 2^-14 is the least that binary16 holds in full: as it is, those of a few thousand rows would be lost
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[y][i] *= 32768.f;
            const u32x4_t po = BlocksPackOperand<BF16>(p[0], p[1]);
            dso = BlocksPackOperand<BF16>(ds[0], ds[1]);
            product(f1, vf, ds1);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (TIGHT) turned_of(stage, S::TENSOR, ot);
            if (more) {
#pragma unroll
                for (uint32_t y = 1; y < (PER + 7) / 8; ++y) load_rows(s + 3, y, to);
                load_info(s + 3, to);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!TIGHT) turned_of(stage, 0, qt);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < OD; ++d) av[d] = BlocksMfma<BF16>(po, u32x4_t{ot[d][0][0], ot[d][0][1], ot[d][1][0], ot[d][1][1]}, av[d]);
            if constexpr (TIGHT) {
                __builtin_amdgcn_sched_barrier(0);
                turned_of(stage, 0, qt);
                __builtin_amdgcn_sched_barrier(0);
                add_keys();
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                p[y] = p1[y];
                ds[y] = ds1[y];
            }
        }
        if constexpr (!TIGHT) add_keys();
        if constexpr (!BF16)
#pragma unroll
            for (int d = 0; d < OD; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) av[d][i] *= 1.f / 32768.f;
    }
    if (works) {
        float bad = 0.f;
#pragma unroll
        for (int d = 0; d < OD; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) bad += (ak[d][i] + av[d][i]) * 0.f;
        if (__ballot(bad != 0.f))
            BlocksKeyGradAgain<BF16, DC, OD>(a, b, h, n, m, s_list, rows, rg * 32, S::ROWS, key, hd * OD * 16, lane, kf, vf, a.scale2 == 0.f ? 1.f : fabsf(a.scale2), dout, info,
                                             ak, av);
    }
    // the second row group's sums are added to the first's
    if (RGS > 1) {
        f32x4_t* s_add = reinterpret_cast<f32x4_t*>(s_keys) + (wave % (kts * ND)) * 2 * OD * 64 + lane;
        __syncthreads();
        if (works && rg == 1)
#pragma unroll
            for (int d = 0; d < OD; ++d) {
                s_add[d * 64] = ak[d];
                s_add[(OD + d) * 64] = av[d];
            }
        __syncthreads();
        if (works && rg == 0)
#pragma unroll
            for (int d = 0; d < OD; ++d) {
                ak[d] += s_add[d * 64];
                av[d] += s_add[(OD + d) * 64];
            }
    }
    if (!works || rg != 0) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t in = in_block + g * 4 + i, row = part.block * a.bs + in;
        if (row >= a.Tk) continue;
        if (part.slot >= 0) {
            float* pk = partial + (((uint64_t)pair * slots + part.slot) * a.bs + in) * 2 * D + hd * OD * 16 + r;
#pragma unroll
            for (int d = 0; d < OD; ++d) {
                pk[d * 16] = ak[d][i];
                pk[D + d * 16] = av[d][i];
            }
        } else {
            uint16_t* pk = dk + b * a.ks[0] + row * a.ks[1] + h * a.ks[2] + hd * OD * 16 + r;
            uint16_t* pv = dv + b * a.vs[0] + row * a.vs[1] + h * a.vs[2] + hd * OD * 16 + r;
#pragma unroll
            for (int d = 0; d < OD; ++d) {
                pk[d * 16] = (uint16_t)BlocksPack<BF16>(ak[d][i] * a.scale, 0.f);
                pv[d * 16] = (uint16_t)BlocksPack<BF16>(av[d][i], 0.f);
            }
        }
    }
}

// adds the parts of a block, in order; four dimensions a thread
template <bool BF16>
__global__ void __launch_bounds__(256) BlocksKeyGradJoinKernel(BlocksArgs a, uint32_t d, uint32_t part_rows, uint32_t slots, const uint32_t* __restrict__ counts,
                                                               const int* __restrict__ first_slot, const float* __restrict__ partial, uint16_t* __restrict__ dk,
                                                               uint16_t* __restrict__ dv) {
    const uint32_t block = blockIdx.x, pair = blockIdx.y, b = pair / a.Hkv, h = pair % a.Hkv;
    const int slot = first_slot[(uint64_t)pair * a.nblk + block];
    if (slot < 0) return;
    const uint32_t n = (counts[(uint64_t)pair * a.nblk + block] + part_rows - 1) / part_rows;
    const uint64_t step = (uint64_t)a.bs * 2 * d;
    const uint32_t i = (blockIdx.z * 256 + threadIdx.x) * 4, row = block * a.bs + i / (2 * d), value = i / d % 2, c = i % d;
    if (i >= a.bs * 2 * d || row >= a.Tk) return;
    const float* from = partial + ((uint64_t)pair * slots + slot) * step + i;
    float4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t p = 0; p < n; ++p) {
        const float4 y = *reinterpret_cast<const float4*>(from + p * step);
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
    }
    const float f = value ? 1.f : a.scale;
    uint16_t* to = value ? dv + b * a.vs[0] + row * a.vs[1] + h * a.vs[2] + c : dk + b * a.ks[0] + row * a.ks[1] + h * a.ks[2] + c;
    *reinterpret_cast<u32x2_t*>(to) = u32x2_t{BlocksPack<BF16>(x.x * f, x.y * f), BlocksPack<BF16>(x.z * f, x.w * f)};
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------
namespace {
struct BackwardSpace {
    size_t bits, counts, info, parts, used, first_slot, partial, total;
    uint32_t words, part_rows, capacity, slots;
};
BackwardSpace BackwardLayout(const BlocksArgs& a, uint32_t d) {
    BackwardSpace s{};
    const uint64_t pairs = (uint64_t)a.B * a.Hkv, blocks = pairs * a.nblk;
    s.words = (a.Tq + 31) / 32;
    // 4096 (row, head) rows a part: a workgroup's work then is a few times the longest ordinary block's, and few blocks are divided (32 heads of 128 dimensions,
    // 16 probes of 64 rows, 2048, 4096 and 8192 rows a part: 8192 query rows 1418, 1375 and 1360 us, 2048 query rows 262, 282 and 317)
    s.part_rows = std::max(1u, 4096 / a.G);
    const uint64_t most = (a.Tq + (uint64_t)s.part_rows - 1) / s.part_rows, marks = (uint64_t)a.Tq * a.P;
    s.capacity = (uint32_t)std::min<uint64_t>(a.nblk * std::max<uint64_t>(1, most), a.nblk + marks / s.part_rows);
    s.slots = (uint32_t)std::min<uint64_t>(most > 1 ? a.nblk * most : 0, 2 * marks / s.part_rows);
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t x = at;
        at += BlocksAlign(n);
        return x;
    };
    s.bits = take(blocks * s.words * 4);
    s.counts = take(blocks * 4);
    s.info = take(((size_t)a.B * a.Tq * a.Hq + 1) * 8);
    s.parts = take(pairs * s.capacity * sizeof(BlocksPart));
    s.used = take(pairs * 4);
    s.first_slot = take(blocks * 4);
    s.partial = take(pairs * s.slots * a.bs * 2 * d * 4);
    s.total = at;
    return s;
}

uint32_t KeyGroups(const BlocksArgs& a) { return (a.bs / 16 + 3) / 4; }   // workgroups of 64 keys that a block has

template <bool BF16, int DC, int ND, int RGS>
gpann_status KeyGrad(const BlocksArgs& a, const BackwardSpace& s, const uint16_t* dout, BlocksRowInfo info, uint16_t* dk, uint16_t* dv, char* ws, hipStream_t st) {
    using S = BlocksKeyShape<DC, RGS>;
    const uint32_t groups = KeyGroups(a);
    const uint64_t per_pair = (uint64_t)s.capacity * groups;
    const size_t lds = std::max<size_t>(S::BUFFERS * S::STAGE, RGS > 1 ? (size_t)64 * S::D * 8 : 0) + (size_t)std::min(s.part_rows, a.Tq) * 4;
    return BlocksLaunch(BlocksKeyGradKernel<BF16, DC, ND, RGS>, BlocksPairGrid((uint64_t)a.B * a.Hkv, per_pair), lds, st, a, s.words, s.part_rows, s.capacity, s.slots, groups,
                        (uint32_t)per_pair, reinterpret_cast<const uint32_t*>(ws + s.bits), reinterpret_cast<const BlocksPart*>(ws + s.parts),
                        reinterpret_cast<const uint32_t*>(ws + s.used), dout, info, dk, dv,
                        reinterpret_cast<float*>(ws + s.partial));
}

template <bool BF16, int DC>
gpann_status Backward(const BlocksArgs& a, const uint16_t* out, const float* lse, const uint16_t* dout, uint16_t* dq, uint16_t* dk, uint16_t* dv, char* ws,
                      hipStream_t st) {
    const BackwardSpace s = BackwardLayout(a, DC * 16);
    uint32_t* counts = reinterpret_cast<uint32_t*>(ws + s.counts);
    int* first_slot = reinterpret_cast<int*>(ws + s.first_slot);
    const uint64_t pairs = (uint64_t)a.B * a.Hkv;
    BlocksRowInfo info;
    info.lse2 = reinterpret_cast<float*>(ws + s.info);
    info.delta = info.lse2 + (uint64_t)a.B * a.Tq * a.Hq + 1;
    if (a.Tq > 0) {
        const uint32_t mtiles = (a.G + 15) / 16, tpw = std::max(1u, 16 / a.G);
        const uint64_t waves = mtiles > 1 ? (uint64_t)a.Tq * mtiles : (a.Tq + tpw - 1) / tpw, tiles = (waves + 7) / 8;
        auto kernel = a.bs % 32 == 0 ? BlocksQueryGradKernel<BF16, DC, 2, 1> : BlocksQueryGradKernel<BF16, DC, 2, 2>;
        if constexpr (DC <= 8)
            if (a.bs % 32 == 0) kernel = a.bs % 64 == 0 ? BlocksQueryGradKernel<BF16, DC, 4, 1> : BlocksQueryGradKernel<BF16, DC, 4, 2>;
        GPANN_TRY(BlocksLaunch(kernel, BlocksPairGrid(pairs, tiles), BlocksWalkShape<DC>::LDS, st, a, tpw, mtiles, (uint32_t)tiles, out, dout, lse,
                               dq, info));
    }
    if (a.Tk == 0) return GPANN_OK;
    uint32_t* bits = reinterpret_cast<uint32_t*>(ws + s.bits);
    if (a.Tq > 0) GPANN_TRY(BlocksMarkProbes(a, s.words, bits, st));
    hipLaunchKernelGGL(BlocksPartsKernel, dim3((uint32_t)pairs), dim3(1024), 0, st, a, s.words, s.part_rows, s.capacity, bits, counts,
                       reinterpret_cast<BlocksPart*>(ws + s.parts), reinterpret_cast<uint32_t*>(ws + s.used), first_slot, info);
    GPANN_HIP_TRY(hipGetLastError());
    if constexpr (DC > 8)
        GPANN_TRY((KeyGrad<BF16, DC, 2, 1>(a, s, dout, info, dk, dv, ws, st)));
    else if (a.bs <= 32)
        GPANN_TRY((KeyGrad<BF16, DC, 2, 2>(a, s, dout, info, dk, dv, ws, st)));
    else
        GPANN_TRY((KeyGrad<BF16, DC, 1, 2>(a, s, dout, info, dk, dv, ws, st)));
    if (s.slots > 0) {
        hipLaunchKernelGGL(BlocksKeyGradJoinKernel<BF16>, dim3(a.nblk, (uint32_t)pairs, (a.bs * 2 * DC * 16 + 1023) / 1024), dim3(256), 0, st, a, DC * 16, s.part_rows,
                           s.slots, counts, first_slot, reinterpret_cast<const float*>(ws + s.partial), dk, dv);
        GPANN_HIP_TRY(hipGetLastError());
    }
    return GPANN_OK;
}
}  // namespace

size_t BlocksBackwardSpace(const BlocksArgs& a, uint32_t d) { return BackwardLayout(a, d).total; }

}  // namespace gpann

using namespace gpann;

extern "C" gpann_status gpann_blocks_attend_backward(const gpann_blocks_layout* L, const void* q, const void* k, const void* v, const int32_t* probes, uint32_t nprobe,
                                                     const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv, void* workspace,
                                                     size_t workspace_bytes, void* stream) {
    GPANN_TRY(BlocksCheckLayout(L));
    GPANN_REQUIRE(q && k && v && probes && out && lse && dout && dq && dk && dv, "a tensor is null");
    GPANN_REQUIRE(BlocksAligned(16, q) && BlocksAligned(16, k) && BlocksAligned(16, v) && BlocksAligned(16, out) && BlocksAligned(16, dout) && BlocksAligned(16, dq) &&
                      BlocksAligned(16, dk) && BlocksAligned(16, dv),
                  "q, k, v, out and the gradients must be 16-byte aligned");
    GPANN_REQUIRE(BlocksAligned(4, probes) && BlocksAligned(4, lse), "probes and lse must be 4-byte aligned");
    GPANN_REQUIRE(nprobe >= 1 && nprobe <= GPANN_BLOCKS_MAX_PROBE, "nprobe must be 1 .. GPANN_BLOCKS_MAX_PROBE");
    if (L->page_table) {
        SetLastError("gradients of a paged cache are not supported: pages may be shared between sequences");
        return GPANN_ERR_UNSUPPORTED;
    }
    GPANN_REQUIRE(BlocksDisjoint(L->q_stride, L->batch, L->q_rows, L->q_heads, L->head_dim), "dq overlaps itself");
    GPANN_REQUIRE(BlocksDisjoint(L->k_stride, L->batch, L->kv_rows, L->kv_heads, L->head_dim), "dk overlaps itself");
    GPANN_REQUIRE(BlocksDisjoint(L->v_stride, L->batch, L->kv_rows, L->kv_heads, L->head_dim), "dv overlaps itself");
    GPANN_TRY(BlocksCheckMarks(L));
    GPANN_REQUIRE((uint64_t)L->batch * L->q_rows * L->q_heads < 0xFFFFFFFFull, "2^32 - 1 (query row, head) rows or more");
    const BlocksArgs a = BlocksMakeArgs(L, q, k, v, probes, nprobe);
    const BackwardSpace space = BackwardLayout(a, L->head_dim);
    GPANN_TRY(BlocksCheckGrid(BlocksPairGrid((uint64_t)a.B * a.Hkv, (uint64_t)space.capacity * KeyGroups(a))));   // before the query side is enqueued
    GPANN_TRY(BlocksCheckWorkspace(workspace, workspace_bytes, space.total));
    GPANN_BLOCKS_ENTER(L, stream);
    if (a.B == 0) return GPANN_OK;
    GPANN_BLOCKS_DISPATCH(L, Backward, a, static_cast<const uint16_t*>(out), lse, static_cast<const uint16_t*>(dout), static_cast<uint16_t*>(dq),
                          static_cast<uint16_t*>(dk), static_cast<uint16_t*>(dv), static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
}

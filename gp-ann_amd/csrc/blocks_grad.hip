// blocks_grad.hip — gradients of the attention over probed cache blocks (include/gpann_blocks.h).
//
// Two passes recompute the weights p = 2^(x log2 e - lse log2 e), each stationary in what it sums: the query side walks the blocks that neighbouring query
// rows probe, as the forward does, and leaves {lse, delta, visible} of every row; the key side has one workgroup per block, past whose keys the rows that
// probe it stream.  No sum crosses workgroups but the parts of blocks that very many rows probe, which are joined in their order: results repeat.
#include "blocks_walk.h"

#include <algorithm>

namespace gpann {

// ---- gradient of the queries ----------------------------------------------------------------------------------------------------------------
// delta = <dout, out> is what every dp is measured against; `out` was rounded, so it is off by e, the same for all of a row's keys.  The walk therefore sums
// ds' = p (dp - delta'), which is e in all, and w = sum p k beside dq' = sum ds' k: the gradient at the true delta is dq' - e w (the weights sum to 1).

// What a query row is to the key side
struct BlocksRowInfo {
    float lse2, delta;
    int visible, pad;
};

template <bool BF16, int DC>
__device__ __forceinline__ float BlocksDelta(const uint16_t* out, const u32x4_t (&go)[DC / 2]) {
    u32x4_t y[DC / 2];
    BlocksLoadRows<DC / 2>(out, y);
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < DC / 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            delta += BlocksToFloat((uint16_t)y[s][i], BF16) * BlocksToFloat((uint16_t)go[s][i], BF16);
            delta += BlocksToFloat((uint16_t)(y[s][i] >> 16), BF16) * BlocksToFloat((uint16_t)(go[s][i] >> 16), BF16);
        }
    return BlocksSumOver4(delta);
}

// One query row's heads (columns r < heads), its probed rows straight from memory: the way out for rows whose neighbours' values are not finite.
template <bool BF16, int DC>
__device__ __forceinline__ void BlocksQueryGradRow(const BlocksArgs& a, uint32_t b, uint32_t h, uint32_t t, uint32_t head, bool live, int visible, uint32_t lane,
                                                   uint32_t* scratch, const uint16_t* out, const uint16_t* dout, const float* lse, uint16_t* dq, BlocksRowInfo* rows) {
    constexpr int KS = DC / 2, N = DC / 2;
    const uint32_t r = lane & 15, g = lane >> 4;
    int block;
    int64_t ko, vo;
    const uint32_t count = BlocksGatherProbes(a, a.probes + (((int64_t)b * a.Tq + t) * a.Hkv + h) * a.P, b, visible, scratch, lane, block, ko, vo);
    u32x4_t q[KS], go[KS];
    BlocksLoadRows<KS>(a.q + b * a.qs[0] + t * a.qs[1] + head * a.qs[2] + g * 8, q);
    BlocksLoadRows<KS>(dout + b * a.os[0] + t * a.os[1] + head * a.os[2] + g * 8, go);
    const float delta = BlocksDelta<BF16, DC>(out + b * a.os[0] + t * a.os[1] + head * a.os[2] + g * 8, go);
    const int64_t row = ((int64_t)b * a.Tq + t) * a.Hq + head;
    const float l = lse[row], lse2 = l == -__builtin_inff() ? __builtin_inff() : l * kLog2e;
    f32x4_t acc[DC];
#pragma unroll
    for (int d = 0; d < DC; ++d) acc[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
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
        const u32x4_t ds = BlocksPackOperand<BF16>(s[0], s[1]);
#pragma unroll
        for (int d = 0; d < DC; ++d) acc[d] = BlocksMfma<BF16>(BlocksColumn<N>(kc, d), ds, acc[d]);
    }
    if (!live) return;
    uint16_t* dst = dq + b * a.qs[0] + (int64_t)t * a.qs[1] + head * a.qs[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[N];
#pragma unroll
        for (int x = 0; x < N; ++x) w[x] = BlocksPack<BF16>(acc[2 * x][i] * a.scale, acc[2 * x + 1][i] * a.scale);
        BlocksStoreColumns<N>(dst + (g * 4 + i) * DC, w);
    }
    if (g == 0) rows[row] = BlocksRowInfo{lse2, delta, visible, 0};
}

// NT tiles of 16 keys of the stage at LDS byte `at` against a wavefront's 16 columns
template <bool BF16, int DC, int NT>
__device__ __forceinline__ void BlocksWalkQueryGrad(float scale2, uint32_t tile0, const BlocksWalkAddresses<DC>& ad, uint32_t at, const int (&start)[4],
                                                    const uint32_t (&mask)[4], const BlocksWalkColumns<1>& col, uint32_t g4, const u32x4_t (&q)[DC / 2],
                                                    const u32x4_t (&go)[DC / 2], float lse2, float delta, f32x4_t (&acc)[DC], f32x4_t (&wk)[DC], float& off) {
    using S = BlocksWalkShape<DC>;
    constexpr uint32_t TILE = S::D * 32;
    constexpr int KS = DC / 2;
#pragma unroll
    for (int z = 0; z < NT / 2; ++z) {
        const uint32_t t0 = tile0 + 2 * z;
        f32x4_t x[2], y[2];
        {
            u32x4_t k[2][KS], v[2][KS];
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) k[i][s] = BlocksReadRow(at + ad.rows[s] + (t0 + i) * TILE);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) v[i][s] = BlocksReadRow(at + ad.rows[s] + S::TENSOR + (t0 + i) * TILE);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 2; ++i) x[i] = y[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) x[i] = BlocksMfma<BF16>(k[i][s], q[s], x[i]);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) y[i] = BlocksMfma<BF16>(v[i][s], go[s], y[i]);
        }
        u32x2_t kt[DC][2];
#pragma unroll
        for (int d = 0; d < DC; ++d)
#pragma unroll
            for (int i = 0; i < 2; ++i) kt[d][i] = BlocksReadTransposed(at + ad.turned[d] + (t0 + i) * TILE);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool member = (mask[t0 + i] >> col.in[0]) & 1;
            const float less = member ? -lse2 : -__builtin_inff();
            if (start[t0 + i] + 16 > col.seen_by_all) {
                const int limit = col.visible[0] - start[t0 + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = (int)g4 + j < limit ? x[i][j] : -__builtin_inff();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i][j] = BlocksExp2(__builtin_fmaf(x[i][j], scale2, less));
                y[i][j] = x[i][j] * (y[i][j] - delta);
                off += y[i][j];
            }
        }
        // one rounding of p and ds to the tensors' type, as of p in the forward
        const u32x4_t p = BlocksPackOperand<BF16>(x[0], x[1]), ds = BlocksPackOperand<BF16>(y[0], y[1]);
#pragma unroll
        for (int d = 0; d < DC; ++d) {
            const u32x4_t kk = {kt[d][0][0], kt[d][0][1], kt[d][1][0], kt[d][1][1]};
            acc[d] = BlocksMfma<BF16>(kk, ds, acc[d]);
            wk[d] = BlocksMfma<BF16>(kk, p, wk[d]);
        }
    }
}

template <bool BF16, int DC>
__global__ void __launch_bounds__(512) BlocksQueryGradKernel(BlocksArgs a, uint32_t tpw, uint32_t mtiles, uint32_t tiles, const uint16_t* __restrict__ out,
                                                             const uint16_t* __restrict__ dout, const float* __restrict__ lse, uint16_t* __restrict__ dq,
                                                             BlocksRowInfo* __restrict__ info) {
    TakeWholeRegisterFile();
    using S = BlocksWalkShape<DC>;
    constexpr int KS = DC / 2;
    extern __shared__ __attribute__((aligned(16))) char s_walk[];
    __shared__ uint32_t s_count, s_scratch[8][64];
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
    float delta = BlocksDelta<BF16, DC>(out + at_o, go);
    const int64_t row = ((int64_t)w.b * a.Tq + col.Row(w, 0)) * a.Hq + col.head[0];
    const float l = lse[row], lse2 = l == -__builtin_inff() ? __builtin_inff() : l * kLog2e;   // an empty row weighs nothing
    const BlocksWalkAddresses<DC> ad(lane);
    f32x4_t acc[DC], wk[DC];
#pragma unroll
    for (int d = 0; d < DC; ++d) acc[d] = wk[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float off = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[s]), "+v"(go[s]));
    const BlocksWalker<DC> walk(a, wave, lane);
    const uint32_t lds = BlocksLdsAddress(s_walk);

    for (uint32_t window = 0; window < blocks; window += S::WINDOW) {
        const uint32_t in_window = min(S::WINDOW, blocks - window);
        const uint32_t units = BlocksWalkList<DC>(a, w, window, in_window, tab, &s_count) * tpb, stages = (units + 3) / 4;
        BlocksWalkStage d[S::BUFFERS];
#pragma unroll
        for (uint32_t s = 0; s + 1 < S::BUFFERS; ++s)
            if (s < stages) {
                d[s] = walk.Describe(a, w, tab, window, s, units, col.seen_by_any);
                walk.Load(d[s], lds + s * S::STAGE);
            }
        uint32_t buf = 0;
        for (uint32_t s = 0; s < stages; ++s) {
            const bool more = s + S::BUFFERS - 1 < stages;
            if (more) d[S::BUFFERS - 1] = walk.Describe(a, w, tab, window, s + S::BUFFERS - 1, units, col.seen_by_any);
            if (S::BUFFERS > 2 && s + 1 < stages)
                BlocksDmaWait<(S::BUFFERS - 2) * S::LOADS>();
            else
                BlocksDmaWait<0>();
            BlocksStageBarrier();
            if (more) walk.Load(d[S::BUFFERS - 1], lds + (buf == 0 ? S::BUFFERS - 1 : buf - 1) * S::STAGE);
            int start[4];
            uint32_t mask[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                start[y] = __builtin_amdgcn_readlane(d[0].start, y);
                mask[y] = (uint32_t)__builtin_amdgcn_readlane((int)d[0].mask, y);
            }
            const uint32_t at = lds + buf * S::STAGE;
            if (mask[0] | mask[1]) BlocksWalkQueryGrad<BF16, DC, 2>(scale2, 0, ad, at, start, mask, col, g * 4, q, go, lse2, delta, acc, wk, off);
            if (mask[2] | mask[3]) BlocksWalkQueryGrad<BF16, DC, 2>(scale2, 2, ad, at, start, mask, col, g * 4, q, go, lse2, delta, acc, wk, off);
#pragma unroll
            for (uint32_t y = 0; y + 1 < S::BUFFERS; ++y) d[y] = d[y + 1];
            buf = buf + 1 == S::BUFFERS ? 0 : buf + 1;
        }
        __syncthreads();
    }
    off = BlocksSumOver4(off);
    float bad = off * 0.f;
#pragma unroll
    for (int d = 0; d < DC; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[d][i] -= off * wk[d][i];
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
    if (g == 0) info[row] = BlocksRowInfo{lse2, delta + off, col.visible[0], 0};
}

// ---- which query rows probe a block -------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) BlocksClearKernel(uint32_t* __restrict__ p, uint64_t n) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) p[i] = 0;
}
// set bits and counts are the same whatever their order
__global__ void __launch_bounds__(256) BlocksBitsKernel(BlocksArgs a, uint32_t words, uint32_t* __restrict__ bits, uint32_t* __restrict__ counts) {
    const uint64_t all = (uint64_t)a.B * a.Tq * a.Hkv * a.P;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < all; i += gridDim.x * 256ull) {
        const int p = a.probes[i];
        const uint64_t row = i / a.P;
        const uint32_t h = (uint32_t)(row % a.Hkv), t = (uint32_t)(row / a.Hkv % a.Tq), b = (uint32_t)(row / a.Hkv / a.Tq);
        const int visible = BlocksVisible(a, BlocksKvLen(a, b), BlocksQLen(a, b), (int)t);
        int64_t ko, vo;
        if (p < 0 || (uint32_t)p >= a.nblk || (int64_t)p * a.bs >= visible || !BlocksBase(a, b, p, ko, vo)) continue;
        const uint64_t at = ((uint64_t)b * a.Hkv + h) * a.nblk + p;
        const uint32_t bit = 1u << (t & 31);
        if (counts && !(atomicOr(bits + at * words + t / 32, bit) & bit)) atomicAdd(counts + at, 1u);
        if (!counts) atomicOr(bits + at * words + t / 32, bit);
    }
}

gpann_status BlocksMarkProbes(const BlocksArgs& a, uint32_t words, uint32_t* bits, uint32_t* counts, hipStream_t st) {
    const uint64_t blocks = (uint64_t)a.B * a.Hkv * a.nblk, n = blocks * words, all = (uint64_t)a.B * a.Tq * a.Hkv * a.P;
    hipLaunchKernelGGL(BlocksClearKernel, dim3((uint32_t)std::min<uint64_t>(n / 256 + 1, 8192)), dim3(256), 0, st, bits, n);
    GPANN_HIP_TRY(hipGetLastError());
    if (counts) {
        hipLaunchKernelGGL(BlocksClearKernel, dim3((uint32_t)std::min<uint64_t>(blocks / 256 + 1, 8192)), dim3(256), 0, st, counts, blocks);
        GPANN_HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(BlocksBitsKernel, dim3((uint32_t)std::min<uint64_t>(all / 256 + 1, 16384)), dim3(256), 0, st, a, words, bits, counts);
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
// one workgroup per pair: parts[pair][capacity], used[pair], first_slot[pair][block]
__global__ void __launch_bounds__(256) BlocksPartsKernel(BlocksArgs a, uint32_t part, uint32_t capacity, const uint32_t* __restrict__ counts, BlocksPart* __restrict__ parts,
                                                         uint32_t* __restrict__ used, int* __restrict__ first_slot) {
    __shared__ uint32_t s_sum[2][256];
    const uint32_t pair = blockIdx.x, tid = threadIdx.x;
    uint32_t base = 0, slots = 0;
    for (uint32_t j0 = 0; j0 < a.nblk; j0 += 256) {
        const uint32_t j = j0 + tid;
        const uint32_t n = j < a.nblk ? max(1u, (counts[(uint64_t)pair * a.nblk + j] + part - 1) / part) : 0, m = n > 1 ? n : 0;
        s_sum[0][tid] = n;
        s_sum[1][tid] = m;
        __syncthreads();
        for (uint32_t s = 1; s < 256; s <<= 1) {
            const uint32_t x = tid >= s ? s_sum[0][tid - s] : 0, y = tid >= s ? s_sum[1][tid - s] : 0;
            __syncthreads();
            s_sum[0][tid] += x;
            s_sum[1][tid] += y;
            __syncthreads();
        }
        const uint32_t at = base + s_sum[0][tid] - n, slot = slots + s_sum[1][tid] - m;
        for (uint32_t i = 0; i < n; ++i) parts[(uint64_t)pair * capacity + at + i] = BlocksPart{j, i, n > 1 ? (int)(slot + i) : -1};
        if (j < a.nblk) first_slot[(uint64_t)pair * a.nblk + j] = n > 1 ? (int)slot : -1;
        base += s_sum[0][255];
        slots += s_sum[1][255];
        __syncthreads();
    }
    if (tid == 0) used[pair] = base;
}

// Shape of the key side: a workgroup holds 64 keys (four 16-key tiles; halves of the dimensions apart where both sums would not fit a wavefront's
// registers) and RGS groups of wavefronts take 32 of a stage's 32 RGS rows each.
template <int DC, int RGS>
struct BlocksKeyShape {
    static constexpr uint32_t D = DC * 16, CPR = D / 8, ROWS = 32 * RGS, TENSOR = ROWS * D * 2, STAGE = 2 * TENSOR + ROWS * 16, LOADS = ROWS * D / 2048;
    static constexpr uint32_t BUFFERS = 2 * TENSOR <= 32768 ? 3 : 2;
};

template <bool BF16, int DC, int RGS>
__global__ void __launch_bounds__(512) BlocksKeyGradKernel(BlocksArgs a, uint32_t words, uint32_t part_rows, uint32_t capacity, uint32_t slots, uint32_t groups,
                                                           uint32_t per_pair, const uint32_t* __restrict__ bits, const BlocksPart* __restrict__ parts,
                                                           const uint32_t* __restrict__ used, const uint16_t* __restrict__ dout, const BlocksRowInfo* __restrict__ info,
                                                           uint16_t* __restrict__ dk, uint16_t* __restrict__ dv, float* __restrict__ partial) {
    TakeWholeRegisterFile();
    using W = BlocksWalkShape<DC>;
    using S = BlocksKeyShape<DC, RGS>;
    constexpr int KS = DC / 2, D = DC * 16, ND = DC > 8 ? 2 : 1, OD = DC / ND;
    extern __shared__ __attribute__((aligned(16))) char s_keys[];   // stages {Q rows, dO rows, row info}; afterwards the sums of the row groups; the row list behind
    uint32_t* s_list = reinterpret_cast<uint32_t*>(s_keys + S::BUFFERS * S::STAGE);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t pair, x;
    if (!BlocksPairOf(blockIdx.x, a.B * a.Hkv, per_pair, pair, x)) return;
    const uint32_t group = x % groups, item = x / groups;
    if (item >= used[pair]) return;
    const BlocksPart part = parts[(uint64_t)pair * capacity + item];
    const uint32_t b = pair / a.Hkv, h = pair % a.Hkv, tpb = a.bs / 16, kts = min(4u, tpb - group * 4);
    const int n = BlocksKvLen(a, b);
    const uint32_t kt = wave % kts, hd = ND == 1 ? 0 : wave / kts % ND, rg = wave / (kts * ND);
    const bool works = rg < RGS;   // wavefronts beyond kts * ND * RGS only load
    const uint32_t in_block = (group * 4 + kt) * 16;
    const int key = (int)(part.block * a.bs + in_block + r);

    // the rows of this part: ranks [index * part_rows, ...) among the set bits; one wavefront counts its way there
    __shared__ uint32_t s_rows;
    if (threadIdx.x < 64) {
        const uint32_t* row_bits = bits + ((uint64_t)pair * a.nblk + part.block) * words;
        const uint32_t lo = part.index * part_rows, hi = lo + part_rows;
        uint32_t before = 0;
        for (uint32_t w0 = 0; w0 < words && before < hi; w0 += 64) {
            uint32_t w = w0 + lane < words ? row_bits[w0 + lane] : 0u;
            const uint32_t c = (uint32_t)__popc(w);
            uint32_t sum = c;
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t y = __shfl_up(sum, s);
                if ((int)lane >= s) sum += y;
            }
            uint32_t rank = before + sum - c;
            while (w) {
                if (rank >= lo && rank < hi) s_list[rank - lo] = (w0 + lane) * 32 + (uint32_t)__ffs(w) - 1;
                ++rank;
                w &= w - 1;
            }
            before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        }
        if (lane == 0) s_rows = before > lo ? min(before, hi) - lo : 0;
    }
    __syncthreads();
    const uint32_t rows = s_rows * a.G, stages = (rows + S::ROWS - 1) / S::ROWS;

    f32x4_t ak[OD], av[OD];
#pragma unroll
    for (int d = 0; d < OD; ++d) ak[d] = av[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (stages > 0) {
        u32x4_t kf[KS], vf[KS];
        {
            int64_t ko, vo;
            (void)BlocksBase(a, b, (int)part.block, ko, vo);
            const int row = min((int)(in_block + r), n - 1 - (int)(part.block * a.bs));   // a probed block holds a visible row
            BlocksLoadRows<KS>(a.k + ko + h * a.ks[2] + row * a.ks[1] + g * 8, kf);
            BlocksLoadRows<KS>(a.v + vo + h * a.vs[2] + row * a.vs[1] + g * 8, vf);
        }
        const float scale2 = a.scale2 == 0.f ? 1.f : fabsf(a.scale2);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (a.scale2 <= 0.f) kf[s] = a.scale2 == 0.f ? u32x4_t{0u, 0u, 0u, 0u} : kf[s] ^ 0x80008000u;   // the scale's sign, on the keys' side here
            asm volatile("" : "+v"(kf[s]), "+v"(vf[s]));
        }
        const BlocksWalkAddresses<DC> ad(lane);
        const uint32_t lds = BlocksLdsAddress(s_keys);
        auto row_of = [&](uint32_t s, uint32_t row, uint32_t& t, uint32_t& head) {
            const uint32_t rr = min(s * S::ROWS + row, rows - 1);
            t = s_list[rr / a.G];
            head = h * a.G + rr % a.G;
        };
        auto load = [&](uint32_t s, uint32_t to) {
#pragma unroll
            for (uint32_t y = 0; y < S::LOADS; ++y) {
                const uint32_t j = wave + 8 * y, per = S::ROWS * S::CPR / 64, at = j % per * 64 + lane, row = at / S::CPR;
                uint32_t t, head;
                row_of(s, row, t, head);
                const bool grad = j >= per;
                const uint16_t* src = grad ? dout + b * a.os[0] + t * a.os[1] + head * a.os[2] : a.q + b * a.qs[0] + t * a.qs[1] + head * a.qs[2];
                BlocksDmaFrom(src + W::Chunk(at % S::CPR, row % 16) * 8, to + (grad ? S::TENSOR : 0) + j % per * 1024);
            }
            if (wave < (S::ROWS + 63) / 64) {   // the rows' info, 16 bytes a lane
                uint32_t t, head;
                row_of(s, min(wave * 64 + lane, S::ROWS - 1), t, head);
                if (S::ROWS >= 64 || lane < S::ROWS) BlocksDmaFrom(info + ((int64_t)b * a.Tq + t) * a.Hq + head, to + 2 * S::TENSOR + wave * 1024);
            }
        };
        const bool extra = wave < (S::ROWS + 63) / 64;
        for (uint32_t s = 0; s + 1 < S::BUFFERS && s < stages; ++s) load(s, lds + s * S::STAGE);
        uint32_t buf = 0;
        for (uint32_t s = 0; s < stages; ++s) {
            if (S::BUFFERS > 2 && s + 1 < stages) {
                if (extra)
                    BlocksDmaWait<(S::BUFFERS - 2) * (S::LOADS + 1)>();
                else
                    BlocksDmaWait<(S::BUFFERS - 2) * S::LOADS>();
            } else {
                BlocksDmaWait<0>();
            }
            BlocksStageBarrier();
            if (s + S::BUFFERS - 1 < stages) load(s + S::BUFFERS - 1, lds + (buf == 0 ? S::BUFFERS - 1 : buf - 1) * S::STAGE);
            if (works && s * S::ROWS + rg * 32 < rows) {
                constexpr uint32_t TILE = D * 32;
                const uint32_t at = lds + buf * S::STAGE + rg * 2 * TILE;
                f32x4_t p[2], ds[2];
                {
                    u32x4_t qr[2][KS];
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int y = 0; y < 2; ++y) qr[y][j] = BlocksReadRow(at + ad.rows[j] + y * TILE);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int y = 0; y < 2; ++y) p[y] = ds[y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int y = 0; y < 2; ++y) p[y] = BlocksMfma<BF16>(qr[y][j], kf[j], p[y]);
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int y = 0; y < 2; ++y) qr[y][j] = BlocksReadRow(at + ad.rows[j] + S::TENSOR + y * TILE);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int y = 0; y < 2; ++y) ds[y] = BlocksMfma<BF16>(qr[y][j], vf[j], ds[y]);
                }
                u32x4_t about[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) about[i] = BlocksReadRow(lds + buf * S::STAGE + 2 * S::TENSOR + (rg * 32 + (i >> 2) * 16 + g * 4 + (i & 3)) * 16);
                u32x2_t ot[OD][2], qt[OD][2];
#pragma unroll
                for (int d = 0; d < OD; ++d)
#pragma unroll
                    for (int y = 0; y < 2; ++y) ot[d][y] = BlocksReadTransposed(at + ad.turned[hd * OD + d] + S::TENSOR + y * TILE);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const u32x4_t& row = about[y * 4 + i];
                        const bool ok = key < (int)row[2] && s * S::ROWS + rg * 32 + y * 16 + g * 4 + i < rows;
                        const float e = BlocksExp2(__builtin_fmaf(p[y][i], scale2, -__uint_as_float(row[0])));
                        p[y][i] = ok ? e : 0.f;
                        ds[y][i] = ok ? e * (ds[y][i] - __uint_as_float(row[1])) : 0.f;
                    }
                const u32x4_t po = BlocksPackOperand<BF16>(p[0], p[1]), dso = BlocksPackOperand<BF16>(ds[0], ds[1]);
#pragma unroll
                for (int d = 0; d < OD; ++d)
#pragma unroll
                    for (int y = 0; y < 2; ++y) qt[d][y] = BlocksReadTransposed(at + ad.turned[hd * OD + d] + y * TILE);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < OD; ++d) av[d] = BlocksMfma<BF16>(po, u32x4_t{ot[d][0][0], ot[d][0][1], ot[d][1][0], ot[d][1][1]}, av[d]);
#pragma unroll
                for (int d = 0; d < OD; ++d) ak[d] = BlocksMfma<BF16>(dso, u32x4_t{qt[d][0][0], qt[d][0][1], qt[d][1][0], qt[d][1][1]}, ak[d]);
            }
            buf = buf + 1 == S::BUFFERS ? 0 : buf + 1;
        }
    }
    // row groups are added in their order, first the keys' sums, then the values'
    float* s_add = reinterpret_cast<float*>(s_keys);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        f32x4_t(&acc)[OD] = which ? av : ak;
        for (uint32_t from = 1; from < RGS; ++from) {
            __syncthreads();
            if (works && rg == from)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < OD; ++d) s_add[(kt * 16 + g * 4 + i) * D + (hd * OD + d) * 16 + r] = acc[d][i];
            __syncthreads();
            if (works && rg == 0)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < OD; ++d) acc[d][i] += s_add[(kt * 16 + g * 4 + i) * D + (hd * OD + d) * 16 + r];
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

// adds the parts of a block; four dimensions a thread
template <bool BF16>
__global__ void __launch_bounds__(256) BlocksKeyGradJoinKernel(BlocksArgs a, uint32_t d, uint32_t part_rows, uint32_t slots, const uint32_t* __restrict__ counts,
                                                               const int* __restrict__ first_slot, const float* __restrict__ partial, uint16_t* __restrict__ dk,
                                                               uint16_t* __restrict__ dv) {
    const uint32_t block = blockIdx.x, pair = blockIdx.y, b = pair / a.Hkv, h = pair % a.Hkv;
    const int slot = first_slot[(uint64_t)pair * a.nblk + block];
    if (slot < 0) return;
    const uint32_t n = (counts[(uint64_t)pair * a.nblk + block] + part_rows - 1) / part_rows;
    const uint64_t step = (uint64_t)a.bs * 2 * d;
    const float* from = partial + ((uint64_t)pair * slots + slot) * step;
    for (uint32_t i = threadIdx.x * 4; i < a.bs * 2 * d; i += 1024) {
        const uint32_t row = block * a.bs + i / (2 * d), value = i / d % 2, c = i % d;
        if (row >= a.Tk) break;
        float4 x = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t p = 0; p < n; ++p) {
            const float4 y = *reinterpret_cast<const float4*>(from + p * step + i);
            x.x += y.x;
            x.y += y.y;
            x.z += y.z;
            x.w += y.w;
        }
        const float f = value ? 1.f : a.scale;
        uint16_t* to = value ? dv + b * a.vs[0] + row * a.vs[1] + h * a.vs[2] + c : dk + b * a.ks[0] + row * a.ks[1] + h * a.ks[2] + c;
        *reinterpret_cast<u32x2_t*>(to) = u32x2_t{BlocksPack<BF16>(x.x * f, x.y * f), BlocksPack<BF16>(x.z * f, x.w * f)};
    }
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
    // 4096 (row, head) rows a part: a workgroup's work then is a few times the longest ordinary block's, and few blocks are divided
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
    s.info = take((size_t)a.B * a.Tq * a.Hq * sizeof(BlocksRowInfo));
    s.parts = take(pairs * s.capacity * sizeof(BlocksPart));
    s.used = take(pairs * 4);
    s.first_slot = take(blocks * 4);
    s.partial = take(pairs * s.slots * a.bs * 2 * d * 4);
    s.total = at;
    return s;
}

template <bool BF16, int DC, int RGS>
gpann_status KeyGrad(const BlocksArgs& a, const BackwardSpace& s, const uint16_t* dout, uint16_t* dk, uint16_t* dv, char* ws, hipStream_t st) {
    using S = BlocksKeyShape<DC, RGS>;
    const uint32_t groups = (a.bs / 16 + 3) / 4;
    const uint64_t per_pair = (uint64_t)s.capacity * groups;
    const size_t lds = std::max<size_t>(S::BUFFERS * S::STAGE, 64 * S::D * 4) + (size_t)std::min(s.part_rows, a.Tq) * 4;
    return BlocksLaunch(BlocksKeyGradKernel<BF16, DC, RGS>, BlocksPairGrid((uint64_t)a.B * a.Hkv, per_pair), lds, st, a, s.words, s.part_rows, s.capacity, s.slots, groups,
                        (uint32_t)per_pair, reinterpret_cast<const uint32_t*>(ws + s.bits), reinterpret_cast<const BlocksPart*>(ws + s.parts),
                        reinterpret_cast<const uint32_t*>(ws + s.used), dout, reinterpret_cast<const BlocksRowInfo*>(ws + s.info), dk, dv,
                        reinterpret_cast<float*>(ws + s.partial));
}

template <bool BF16, int DC>
gpann_status Backward(const BlocksArgs& a, const uint16_t* out, const float* lse, const uint16_t* dout, uint16_t* dq, uint16_t* dk, uint16_t* dv, char* ws,
                      hipStream_t st) {
    const BackwardSpace s = BackwardLayout(a, DC * 16);
    uint32_t* counts = reinterpret_cast<uint32_t*>(ws + s.counts);
    int* first_slot = reinterpret_cast<int*>(ws + s.first_slot);
    const uint64_t pairs = (uint64_t)a.B * a.Hkv;
    if (a.Tq > 0) {
        const uint32_t mtiles = (a.G + 15) / 16, tpw = std::max(1u, 16 / a.G);
        const uint64_t waves = mtiles > 1 ? (uint64_t)a.Tq * mtiles : (a.Tq + tpw - 1) / tpw, tiles = (waves + 7) / 8;
        GPANN_TRY(BlocksLaunch(BlocksQueryGradKernel<BF16, DC>, BlocksPairGrid(pairs, tiles), BlocksWalkShape<DC>::LDS, st, a, tpw, mtiles, (uint32_t)tiles, out, dout, lse,
                               dq, reinterpret_cast<BlocksRowInfo*>(ws + s.info)));
    }
    if (a.Tk == 0) return GPANN_OK;
    GPANN_TRY(BlocksMarkProbes(a, s.words, reinterpret_cast<uint32_t*>(ws + s.bits), counts, st));
    hipLaunchKernelGGL(BlocksPartsKernel, dim3((uint32_t)pairs), dim3(256), 0, st, a, s.part_rows, s.capacity, counts, reinterpret_cast<BlocksPart*>(ws + s.parts),
                       reinterpret_cast<uint32_t*>(ws + s.used), first_slot);
    GPANN_HIP_TRY(hipGetLastError());
    // wavefronts beside the block's (up to four) 16-key tiles take more rows at a time
    constexpr int most = DC > 8 ? 1 : 2;
    if (a.bs <= 32)
        GPANN_TRY((KeyGrad<BF16, DC, 2 * most>(a, s, dout, dk, dv, ws, st)));
    else
        GPANN_TRY((KeyGrad<BF16, DC, most>(a, s, dout, dk, dv, ws, st)));
    if (s.slots > 0) {
        hipLaunchKernelGGL(BlocksKeyGradJoinKernel<BF16>, dim3(a.nblk, (uint32_t)pairs), dim3(256), 0, st, a, DC * 16, s.part_rows, s.slots, counts, first_slot,
                           reinterpret_cast<const float*>(ws + s.partial), dk, dv);
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
    GPANN_REQUIRE((uint64_t)L->batch * L->kv_heads <= 65535, "more than 65535 (sequence, head) pairs");
    const BlocksArgs a = BlocksMakeArgs(L, q, k, v, probes, nprobe);
    GPANN_TRY(BlocksCheckWorkspace(workspace, workspace_bytes, BackwardLayout(a, L->head_dim).total));
    GPANN_BLOCKS_ENTER(L, stream);
    if (a.B == 0) return GPANN_OK;
    GPANN_BLOCKS_DISPATCH(L, Backward, a, static_cast<const uint16_t*>(out), lse, static_cast<const uint16_t*>(dout), static_cast<uint16_t*>(dq),
                          static_cast<uint16_t*>(dk), static_cast<uint16_t*>(dv), static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
}

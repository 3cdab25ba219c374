// blocks_attend.hip — attention over probed cache blocks, its gradients, and the attention weights of the cache rows (include/gpann_blocks.h).
#include "blocks_walk.h"

#include <algorithm>

namespace gpann {

// ---- forward --------------------------------------------------------------------------------------------------------------------------------
// One pass over the probed rows with a running maximum and sum per query row, in powers of two (softmax(x) = 2^(x log2 e - max) / sum).  A wavefront works
// on one query row's heads of a group (at most 16: the columns of the matrix tiles): X^T = K Q^T, then O^T += V^T P^T.
//
// First the form that reads both operands straight from memory, 32 keys a step (blocks_tile.h): for rows that are done again by themselves.
template <bool BF16, int DC>
struct BlocksStep {
    static constexpr int KS = DC / 2, N = DC / 2;
    u32x4_t k[2][KS];
    uint32_t v[8][N];
    int start[2];     // position of the tiles' first rows
    bool second;      // the second tile is a tile of the range
};

template <bool BF16, int DC>
__device__ __forceinline__ void BlocksLoadStep(const BlocksArgs& a, uint32_t h, int visible, int block, int64_t ko, int64_t vo, BlocksCursor& c, uint32_t left,
                                               uint32_t lane, BlocksStep<BF16, DC>& st) {
    const uint32_t r = lane & 15, g = lane >> 4;
    st.second = left > 1;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int blk = __builtin_amdgcn_readlane(block, (int)c.slot);
        const int64_t kb = BlocksReadLane64(ko, c.slot), vb = BlocksReadLane64(vo, c.slot);
        const int base = (int)c.sub * 16, most = visible - 1 - blk * (int)a.bs;   // rows past the last visible one are not read
        st.start[x] = blk * (int)a.bs + base;
        BlocksLoadRows<DC / 2>(a.k + kb + h * a.ks[2] + min(base + (int)r, most) * a.ks[1] + g * 8, st.k[x]);
        const uint16_t* v = a.v + vb + h * a.vs[2] + r * DC;
#pragma unroll
        for (int i = 0; i < 4; ++i) BlocksLoadColumns<DC / 2>(v + min(base + (int)g * 4 + i, most) * a.vs[1], st.v[x * 4 + i]);
        if (x == 0 && st.second) c.Next();
    }
    c.Next();
}

template <bool BF16, int DC>
__device__ __forceinline__ void BlocksAttendStep(const BlocksArgs& a, int visible, uint32_t lane, BlocksStep<BF16, DC>& st, const u32x4_t (&q)[DC / 2],
                                                 f32x4_t (&o)[DC], float& top, float& sum) {
    const int g4 = (int)(lane >> 4) * 4;
    f32x4_t x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < DC / 2; ++s) {
        x[0] = BlocksMfma<BF16>(st.k[0][s], q[s], x[0]);
        x[1] = BlocksMfma<BF16>(st.k[1][s], q[s], x[1]);
    }
    const float inf = __builtin_inff();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[0][i] *= a.scale2;
        x[1][i] *= a.scale2;
    }
    if (!st.second || st.start[0] + 16 > visible || st.start[1] + 16 > visible) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool ok0 = st.start[0] + g4 + i < visible, ok1 = st.second && st.start[1] + g4 + i < visible;
            x[0][i] = ok0 ? x[0][i] : -inf;
            x[1][i] = ok1 ? x[1][i] : -inf;
#pragma unroll
            for (int c = 0; c < DC / 2; ++c) {   // 0 * value, whatever a row outside holds
                st.v[i][c] = ok0 ? st.v[i][c] : 0u;
                st.v[4 + i][c] = ok1 ? st.v[4 + i][c] : 0u;
            }
        }
    }
    float best = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    best = BlocksMaxOver4(best);
    if (__ballot(best > top + kBlocksSlack<BF16>)) {
        best = fmaxf(top, best - kBlocksLift<BF16>);
        const float shrink = top == best ? 1.f : BlocksExp2(top - best);   // (top = best = -inf: nothing seen yet)
        top = best;
        sum *= shrink;
#pragma unroll
        for (int d = 0; d < DC; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] *= shrink;
    }
    const float from = top == -inf ? 0.f : top;   // 2^(-inf - 0) = 0
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[y][i] = BlocksExp2(x[y][i] - from);
            sum += x[y][i];
        }
    // the weights enter the second product in the type of the values: 2^-8 (bf16) or 2^-11 (fp16) of each at most, as the values themselves (fp16: of those
    // above 2^-21 of the largest)
    const u32x4_t p = BlocksPackOperand<BF16>(x[0], x[1]);
#pragma unroll
    for (int d = 0; d < DC; ++d) o[d] = BlocksMfma<BF16>(BlocksColumn<DC / 2>(st.v, d), p, o[d]);
}

// All of a query row's probed rows from tile `u` to `end`, 32 a step
template <bool BF16, int DC>
__device__ __forceinline__ void BlocksAttendRange(const BlocksArgs& a, uint32_t h, int visible, int block, int64_t ko, int64_t vo, uint32_t u, uint32_t end,
                                                  uint32_t lane, const u32x4_t (&q)[DC / 2], f32x4_t (&o)[DC], float& top, float& sum) {
    BlocksCursor c(u, a.bs / 16);
    for (; u < end; u += 2) {
        BlocksStep<BF16, DC> s;
        BlocksLoadStep(a, h, visible, block, ko, vo, c, end - u, lane, s);
        BlocksAttendStep(a, visible, lane, s, q, o, top, sum);
    }
}

// a wavefront's sums in the column layout (slot d of lane column: dimension (4 g + i) * DC + d) -> out and lse of its rows
template <bool BF16, int DC>
__device__ __forceinline__ void BlocksAttendStore(const BlocksArgs& a, uint32_t b, uint32_t t, uint32_t head, uint32_t g, const f32x4_t (&o)[DC], float top, float sum,
                                                  uint16_t* out, float* lse) {
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);   // (a NaN sum stays one)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[DC / 2];
#pragma unroll
        for (int c = 0; c < DC / 2; ++c) w[c] = BlocksPack<BF16>(o[2 * c][i] * inv, o[2 * c + 1][i] * inv);
        BlocksStoreColumns<DC / 2>(out + b * a.os[0] + (int64_t)t * a.os[1] + head * a.os[2] + (g * 4 + i) * DC, w);
    }
    if (lse && g == 0) lse[((int64_t)b * a.Tq + t) * a.Hq + head] = sum == 0.f ? -__builtin_inff() : (top + __log2f(sum)) * kLn2;
}

// The form for few query rows, each apart: `waves` wavefronts of `splits` workgroups share a query row's keys and join through LDS (and memory).  Rows come to
// LDS by DMA, whole rows an instruction, into a place of the wavefront's own; from there a step's K, then its V, go to registers, and the next step's follow at
// once.  (Read from memory as the matrix instruction wants them, 16 bytes of 16 rows side by side, K costs the address unit 64 cycles an instruction instead
// of 16: 8 x 64 rows for each of 8 heads 8.3 us, 10.1 that way.)  Bound by memory in a batch (64 sequences, 32 x 64 rows for each of 8 heads of 128
// dimensions, 538 MB: 100 us, 5.4 TB/s), by the trips one after the other alone (16 x 64 rows for each of 8 heads: 8.2 us and 3.8 for the join).
template <int DC>
struct BlocksTokenShape {
    using W = BlocksWalkShape<DC>;
    static constexpr uint32_t D = DC * 16, TILES = D <= 128 ? 2 : 1, TILE = D * 32, TENSOR = TILES * TILE, PER = W::CPR / 4, LOADS = TILES * PER, RING = 8 * 2 * TENSOR;
};
struct BlocksTokenStep {   // 16-row tiles of a step
    uint64_t k[2], v[2];   // addresses of their first rows
    int start[2], last[2]; // positions of those; the last row that may be read, in the tile
    uint64_t second;       // the second tile is a tile of the range (64 bits: padding behind it would be copied through memory)
};
template <int DC>
struct BlocksTokenLoader {
    using S = BlocksTokenShape<DC>;
    uint32_t kplace[S::PER], vplace[S::PER], lane, krow, vrow;
    __device__ __forceinline__ BlocksTokenLoader(const BlocksArgs& a, uint32_t lane_) : lane(lane_), krow((uint32_t)a.ks[1] * 2), vrow((uint32_t)a.vs[1] * 2) {
#pragma unroll
        for (uint32_t j = 0; j < S::PER; ++j) {
            kplace[j] = Place(j, krow, 15);
            vplace[j] = Place(j, vrow, 15);
        }
    }
    __device__ __forceinline__ uint32_t Place(uint32_t j, uint32_t stride, int last) const {
        const uint32_t at = j * 64 + lane, row = at / S::W::CPR;
        return (uint32_t)min((int)row, last) * stride + S::W::Slot(at % S::W::CPR, row) * 16;
    }
    __device__ __forceinline__ void Load(const BlocksTokenStep& st, bool value, uint32_t to) const {
#pragma unroll
        for (uint32_t x = 0; x < S::TILES; ++x)
#pragma unroll
            for (uint32_t j = 0; j < S::PER; ++j) {
                uint32_t offset = value ? vplace[j] : kplace[j];
                if (st.last[x] < 15) offset = Place(j, value ? vrow : krow, st.last[x]);   // rows past the last visible one are not read
                BlocksDma(value ? st.v[x] : st.k[x], offset, to + (x * S::PER + j) * 1024);
            }
    }
};

template <bool BF16, int DC>
__device__ __forceinline__ void BlocksAttendTokens(const BlocksArgs& a, uint32_t h, int visible, int block, int64_t ko, int64_t vo, uint32_t u, uint32_t end,
                                                   uint32_t lane, uint32_t ring, u32x4_t (&q)[DC / 2], f32x4_t (&o)[DC], float& top, float& sum) {
    using S = BlocksTokenShape<DC>;
    constexpr int KS = DC / 2, T = S::TILES;
    const float inf = __builtin_inff();
    const int g4 = (int)(lane >> 4) * 4;
    BlocksCursor c(u, a.bs / 16);
    const BlocksTokenLoader<DC> loader(a, lane);
    const BlocksWalkAddresses<DC> ad(lane);
    auto describe = [&](uint32_t left) {
        BlocksTokenStep st{};
        st.second = T == 2 && left > 1;
#pragma unroll
        for (int x = 0; x < T; ++x) {
            const int blk = __builtin_amdgcn_readlane(block, (int)c.slot), base = (int)c.sub * 16, most = visible - 1 - blk * (int)a.bs;
            const int first = min(base, most & ~15);   // a tile without visible rows: the rows of the last one with any
            st.start[x] = blk * (int)a.bs + base;
            st.last[x] = min(15, most - first);
            st.k[x] = (uint64_t)(a.k + BlocksReadLane64(ko, c.slot) + h * a.ks[2] + first * a.ks[1]);
            st.v[x] = (uint64_t)(a.v + BlocksReadLane64(vo, c.slot) + h * a.vs[2] + first * a.vs[1]);
            if (x == 0 && st.second) c.Next();
        }
        c.Next();
        return st;
    };
    BlocksTokenStep st = describe(end - u);
    loader.Load(st, false, ring);
    loader.Load(st, true, ring + S::TENSOR);
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[s]));   // here, not in the loop, is where these loads are waited for
    for (; u < end; u += T) {
        const bool more = u + T < end;
        const BlocksTokenStep next = more ? describe(end - u - T) : st;
        BlocksDmaWait<S::LOADS>();   // K has landed; V is on its way
        f32x4_t x[2];
        {
            uint32_t step[KS];
            u32x4_t k[T][KS];
            ad.RowSteps(ring, step);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int y = 0; y < T; ++y) k[y][s] = BlocksReadRow(step[s] + y * S::TILE);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // its place is free again
            if (more) loader.Load(next, false, ring);
            x[0] = x[1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int y = 0; y < T; ++y) x[y] = BlocksMfma<BF16>(k[y][s], q[s], x[y]);
        }
        const bool edge = (T == 2 && !st.second) || st.start[0] + 16 > visible || (T == 2 && st.start[1] + 16 > visible);
        float best = -inf;
#pragma unroll
        for (int y = 0; y < T; ++y) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[y][i] *= a.scale2;
            if (edge)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[y][i] = (y == 0 || st.second) && st.start[y] + g4 + i < visible ? x[y][i] : -inf;
            best = BlocksMaxOf4(x[y], best);
        }
        best = BlocksMaxOver4(best);
        if (__ballot(best > top + kBlocksSlack<BF16>)) {
            best = fmaxf(top, best - kBlocksLift<BF16>);
            const float shrink = top == best ? 1.f : BlocksExp2(top - best);   // (top = best = -inf: nothing seen yet)
            top = best;
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < DC; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] *= shrink;
        }
        const float from = top == -inf ? 0.f : top;   // 2^(-inf - 0) = 0
#pragma unroll
        for (int y = 0; y < T; ++y) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[y][i] = BlocksExp2(x[y][i] - from);
            sum += (x[y][0] + x[y][1]) + (x[y][2] + x[y][3]);
        }
        // the weights enter the second product in the type of the values: 2^-8 (bf16) or 2^-11 (fp16) of each at most, as the values themselves (fp16: of
        // those above 2^-21 of the largest)
        const u32x4_t p = BlocksPackOperand<BF16>(x[0], x[1]);
        if (more)
            BlocksDmaWait<S::LOADS>();   // V has landed; the next K is on its way
        else
            BlocksDmaWait<0>();
        u32x2_t v[DC][2];
        uint32_t turned[DC];
        ad.template Dimensions<DC>(ring + S::TENSOR, turned);
#pragma unroll
        for (int d = 0; d < DC; ++d)
#pragma unroll
            for (int y = 0; y < 2; ++y) v[d][y] = y < T ? BlocksReadTransposed(turned[d] + y * S::TILE) : u32x2_t{0u, 0u};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) loader.Load(next, true, ring + S::TENSOR);
        if (edge)   // 0 * value, whatever stands in for a row outside
#pragma unroll
            for (int y = 0; y < T; ++y)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const int at = st.start[y] + g4 + 2 * w;
                    const bool there = y == 0 || st.second;
                    const uint32_t keep = (there && at < visible ? 0xFFFFu : 0u) | (there && at + 1 < visible ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int d = 0; d < DC; ++d) v[d][y][w] &= keep;
                }
#pragma unroll
        for (int d = 0; d < DC; ++d) o[d] = BlocksMfma<BF16>(u32x4_t{v[d][0][0], v[d][0][1], v[d][1][0], v[d][1][1]}, p, o[d]);
        st = next;
    }
}

template <bool BF16, int DC>
__global__ void __launch_bounds__(512) BlocksAttendKernel(BlocksArgs a, uint32_t waves, uint32_t splits, uint32_t mtiles, uint32_t tiles, uint16_t* __restrict__ out,
                                                          float* __restrict__ lse, float* __restrict__ sums) {
    TakeWholeRegisterFile();
    constexpr int D = DC * 16;
    extern __shared__ __attribute__((aligned(1024))) float s_join[];   // the wavefronts' places; behind them, waves > 1: [wavefront][16 rows][D + 2]
    __shared__ uint32_t s_scratch[8][64];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t pair, tile;
    if (!BlocksPairOf(blockIdx.x, a.B * a.Hkv, tiles * splits, pair, tile)) return;
    const uint32_t split = tile % splits;
    tile /= splits;
    const uint32_t b = pair / a.Hkv, h = pair % a.Hkv, per = 8 / waves;
    const int n = BlocksKvLen(a, b), m = BlocksQLen(a, b);
    const uint32_t task = tile * per + wave / waves, part = split * waves + wave % waves, parts = splits * waves, t = task / mtiles, mt = task % mtiles;
    const uint32_t heads = min(16u, a.G - mt * 16), head = h * a.G + mt * 16 + min(r, heads - 1);
    const bool live = (int)t < m;
    const int visible = live ? BlocksVisible(a, n, m, (int)t) : 0;

    f32x4_t o[DC];
#pragma unroll
    for (int d = 0; d < DC; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float top = -__builtin_inff(), sum = 0.f;
    if (visible > 0) {
        int block;
        int64_t ko, vo;
        const uint32_t count = BlocksGatherProbes(a, a.probes + (((int64_t)b * a.Tq + t) * a.Hkv + h) * a.P, b, visible, s_scratch[wave], lane, block, ko, vo);
        const uint32_t tpb = a.bs / 16, units = count * tpb, chunk = ((units + parts - 1) / parts + 1) & ~1u;
        uint32_t u = part * chunk;
        const uint32_t end = min(units, u + chunk);
        if (u < end) {
            u32x4_t q[DC / 2];
            BlocksLoadRows<DC / 2>(a.q + b * a.qs[0] + t * a.qs[1] + head * a.qs[2] + g * 8, q);
            BlocksAttendTokens<BF16, DC>(a, h, visible, block, ko, vo, u, end, lane, BlocksLdsAddress(s_join) + wave * 2 * BlocksTokenShape<DC>::TENSOR, q, o, top, sum);
        }
    }
    sum = BlocksSumOver4(sum);
    if (waves == 1) {
        if (!live || r >= heads) return;
        const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);   // (a NaN sum stays one)
        uint16_t* dst = out + b * a.os[0] + (int64_t)t * a.os[1] + head * a.os[2] + g * 4;
#pragma unroll
        for (int d = 0; d < DC; ++d) *reinterpret_cast<u32x2_t*>(dst + d * 16) = u32x2_t{BlocksPack<BF16>(o[d][0] * inv, o[d][1] * inv), BlocksPack<BF16>(o[d][2] * inv, o[d][3] * inv)};
        if (lse && g == 0) lse[((int64_t)b * a.Tq + t) * a.Hq + head] = sum == 0.f ? -__builtin_inff() : (top + __log2f(sum)) * kLn2;
        return;
    }
    __syncthreads();   // (the sums take the place of the rows)
    float* s_ml = s_join + 8 * 16 * D;
    if (g == 0) {
        s_ml[(wave * 16 + r) * 2] = top;
        s_ml[(wave * 16 + r) * 2 + 1] = sum;
    }
    if (r < heads && sum != 0.f) {
#pragma unroll
        for (int d = 0; d < DC; ++d) *reinterpret_cast<f32x4_t*>(s_join + (wave * 16 + r) * D + d * 16 + g * 4) = o[d];
    }
    __syncthreads();
    // two neighbouring dimensions of one row a thread
    for (uint32_t i = threadIdx.x; i < per * 16 * (D / 2); i += 512) {
        const uint32_t c = i % (D / 2) * 2, row = i / (D / 2) % 16, which = i / (D / 2) / 16;
        const uint32_t task2 = tile * per + which, t2 = task2 / mtiles, mt2 = task2 % mtiles, heads2 = min(16u, a.G - mt2 * 16);
        if ((int)t2 >= m || row >= heads2) continue;
        float best = -__builtin_inff();
        for (uint32_t w = 0; w < waves; ++w) best = fmaxf(best, s_ml[((which * waves + w) * 16 + row) * 2]);
        const float from = best == -__builtin_inff() ? 0.f : best;
        float total = 0.f, x = 0.f, y = 0.f;
        for (uint32_t w = 0; w < waves; ++w) {
            const uint32_t at = (which * waves + w) * 16 + row;
            const float part_sum = s_ml[at * 2 + 1];
            if (part_sum == 0.f) continue;
            const float f = BlocksExp2(s_ml[at * 2] - from);
            total += f * part_sum;
            x += f * s_join[at * D + c];
            y += f * s_join[at * D + c + 1];
        }
        if (splits > 1) {
            float* to = sums + ((uint64_t)(pair * tiles + tile) * splits + split) * 16 * (D + 2) + row * (D + 2);
            *reinterpret_cast<float2*>(to + c) = float2{x, y};
            if (c == 0) *reinterpret_cast<float2*>(to + D) = float2{best, total};
            continue;
        }
        const float inv = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
        const uint32_t head2 = h * a.G + mt2 * 16 + row;
        *reinterpret_cast<uint32_t*>(out + b * a.os[0] + (int64_t)t2 * a.os[1] + head2 * a.os[2] + c) = BlocksPack<BF16>(x * inv, y * inv);
        if (lse && c == 0) lse[((int64_t)b * a.Tq + t2) * a.Hq + head2] = total == 0.f ? -__builtin_inff() : (best + __log2f(total)) * kLn2;
    }
}

// joins the parts of a query row's keys that workgroups had; two neighbouring dimensions of one head a thread.  A launch's time, 3.8 us.
template <bool BF16>
__global__ void __launch_bounds__(256) BlocksAttendJoinKernel(BlocksArgs a, uint32_t d, uint32_t splits, uint32_t mtiles, uint32_t tiles, const float* __restrict__ sums,
                                                              uint16_t* __restrict__ out, float* __restrict__ lse) {
    const uint32_t task = blockIdx.y, pair = task / tiles, tile = task % tiles, b = pair / a.Hkv, h = pair % a.Hkv, t = tile / mtiles, mt = tile % mtiles;
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, c = i % (d / 2) * 2, row = i / (d / 2);
    if (row >= min(16u, a.G - mt * 16) || (int)t >= BlocksQLen(a, b)) return;
    const float* from = sums + ((uint64_t)task * splits * 16 + row) * (d + 2);
    const uint64_t step = (uint64_t)16 * (d + 2);
    float best = -__builtin_inff();
    for (uint32_t s = 0; s < splits; ++s) best = fmaxf(best, from[s * step + d]);
    const float base = best == -__builtin_inff() ? 0.f : best;
    float total = 0.f, x = 0.f, y = 0.f;
#pragma unroll 4
    for (uint32_t s = 0; s < splits; ++s) {
        const float2 part = *reinterpret_cast<const float2*>(from + s * step + d), v = *reinterpret_cast<const float2*>(from + s * step + c);
        const float f = part.y == 0.f ? 0.f : BlocksExp2(part.x - base);   // (a part without rows holds zeros)
        total += f * part.y;
        x += f * v.x;
        y += f * v.y;
    }
    const float inv = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
    const uint32_t head = h * a.G + mt * 16 + row;
    *reinterpret_cast<uint32_t*>(out + b * a.os[0] + (int64_t)t * a.os[1] + head * a.os[2] + c) = BlocksPack<BF16>(x * inv, y * inv);
    if (lse && c == 0) lse[((int64_t)b * a.Tq + t) * a.Hq + head] = total == 0.f ? -__builtin_inff() : (best + __log2f(total)) * kLn2;
}

// ---- forward, neighbouring query rows together ----------------------------------------------------------------------------------------------------
// NT tiles of 16 keys, the first at LDS byte `at`, against a wavefront's CT x 16 columns.  `mask`: which of its query rows look at them, of every tile or once
// for all, which are of one block then; `start`: their positions, or the first one's.  Operands are read in batches ahead of the products that need them (the
// scheduling barriers keep the compiler from pairing every read with its use, a full LDS latency each).  scale2 >= 0 (the sign is the queries').
template <bool BF16, int DC, int CT, int NT, int NM, typename F>
__device__ __forceinline__ void BlocksWalkAttend(float scale2, const BlocksWalkAddresses<DC>& ad, uint32_t at, const int (&start)[NM],
                                                 const uint32_t (&mask)[NM], const BlocksWalkColumns<CT>& col, uint32_t g4, const u32x4_t (&q)[CT][DC / 2],
                                                 f32x4_t (&o)[CT][DC], float (&top)[CT], float (&sum)[CT], F&& meanwhile) {
    using S = BlocksWalkShape<DC>;
    constexpr uint32_t TILE = S::D * 32;   // bytes of 16 rows
    constexpr int KS = DC / 2, BATCH = DC * CT > 8 ? 2 : NT, PER = NT / NM;
    const float inf = __builtin_inff();
    f32x4_t x[CT][NT];
    {
        uint32_t step[KS];
        ad.RowSteps(at, step);
#pragma unroll
        for (int y0 = 0; y0 < NT; y0 += BATCH) {
            u32x4_t k[BATCH][KS];
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int y = 0; y < BATCH; ++y) k[y][s] = BlocksReadRow(step[s] + (y0 + y) * TILE);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int y = 0; y < BATCH; ++y) x[c][y0 + y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int y = 0; y < BATCH; ++y) x[c][y0 + y] = BlocksMfma<BF16>(k[y][s], q[c][s], x[c][y0 + y]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    meanwhile();   // the next stage is asked for under the products' cover: asked for by all wavefronts right behind a barrier, it would hold them all up
    uint32_t turned[DC];
    u32x2_t v[DC][2];
    ad.template Dimensions<DC>(at, turned);
#pragma unroll
    for (int d = 0; d < DC; ++d)
#pragma unroll
        for (int y = 0; y < 2; ++y) v[d][y] = BlocksReadTransposed(turned[d] + S::TENSOR + y * TILE);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < NM; ++e)
        if (start[e] + 16 * PER > col.seen_by_all) {   // not every column sees every key
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const int limit = col.visible[c] - start[e] - (int)g4;
#pragma unroll
                for (int y = 0; y < PER; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[c][e * PER + y][i] = y * 16 + i < limit ? x[c][e * PER + y][i] : -inf;
            }
        }
    bool member[CT][NM];
    float best[CT];
    bool raise = false;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        best[c] = -inf;
#pragma unroll
        for (int e = 0; e < NM; ++e) {
            member[c][e] = (mask[e] >> col.in[c]) & 1;
            float most = BlocksMaxOf4(x[c][e * PER]);
#pragma unroll
            for (int y = 1; y < PER; ++y) most = BlocksMaxOf4(x[c][e * PER + y], most);
            best[c] = fmaxf(best[c], member[c][e] ? most : -inf);
        }
        best[c] = BlocksMaxOver4(best[c]) * scale2;
        raise = raise || best[c] > top[c] + kBlocksSlack<BF16>;
    }
    if (__ballot(raise)) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            best[c] = fmaxf(top[c], best[c] - kBlocksLift<BF16>);
            const float shrink = top[c] == best[c] ? 1.f : BlocksExp2(top[c] - best[c]);
            top[c] = best[c];
            sum[c] *= shrink;
#pragma unroll
            for (int d = 0; d < DC; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][d][i] *= shrink;
        }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const float base = top[c] == -inf ? 0.f : -top[c];
#pragma unroll
        for (int y = 0; y < NT; ++y) {
            const float less = member[c][y / PER] ? base : -inf;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[c][y][i] = BlocksExp2(__builtin_fmaf(x[c][y][i], scale2, less));
            sum[c] += (x[c][y][0] + x[c][y][1]) + (x[c][y][2] + x[c][y][3]);
        }
    }
#pragma unroll
    for (int z = 0; z < NT / 2; ++z) {
        u32x2_t next[DC][2];
        if (z + 1 < NT / 2) {
#pragma unroll
            for (int d = 0; d < DC; ++d)
#pragma unroll
                for (int y = 0; y < 2; ++y) next[d][y] = BlocksReadTransposed(turned[d] + S::TENSOR + (2 * z + 2 + y) * TILE);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const u32x4_t p = BlocksPackOperand<BF16>(x[c][2 * z], x[c][2 * z + 1]);
#pragma unroll
            for (int d = 0; d < DC; ++d) o[c][d] = BlocksMfma<BF16>(u32x4_t{v[d][0][0], v[d][0][1], v[d][1][0], v[d][1][1]}, p, o[c][d]);
        }
        if (z + 1 < NT / 2)
#pragma unroll
            for (int d = 0; d < DC; ++d)
#pragma unroll
                for (int y = 0; y < 2; ++y) v[d][y] = next[d][y];
    }
}

// The walk of blocks_walk.h with the running maximum and sum of a softmax.  NT: tiles taken at a time; NM: of how many blocks they may be.
//
// 8192 query rows of 32 heads, 8 key/value heads of 128 dimensions, 16 probes of 64 rows (125 GFLOP of probed products): 355 us a call, 352 TFLOP/s.  The matrix
// cores are busy for 28 % of the cycles, the vector units for 40 %, LDS for 14 %.  228 GFLOP are issued: a wavefront's columns are multiplied together when one of
// their query rows looks at a block.  And a wavefront goes through reads, products and weights of a stage one after the other, a SIMD has only two of them (256
// registers each, 3 more in scratch, and LDS has room for one workgroup), and a barrier waits for the one with most to do.  What made it faster was fewer vector
// instructions (493 -> 383 us), not more overlap inside a wavefront (no difference) or wavefront priorities (none).  Rows of 256 dimensions keep 76 registers in
// scratch.
template <bool BF16, int DC, int CT, int NT, int NM>
__global__ void __launch_bounds__(512) BlocksAttendWalkKernel(BlocksArgs a, uint32_t tpw, uint32_t mtiles, uint32_t tiles, uint16_t* __restrict__ out,
                                                              float* __restrict__ lse) {
    TakeWholeRegisterFile();
    using S = BlocksWalkShape<DC>;
    constexpr int KS = DC / 2;
    extern __shared__ __attribute__((aligned(1024))) char s_walk[];   // stages, tables
    __shared__ uint32_t s_count, s_scratch[8][64];
    const BlocksWalkTables<DC> tab(s_walk);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t pair, tile;
    if (!BlocksPairOf(blockIdx.x, a.B * a.Hkv, tiles, pair, tile)) return;
    BlocksWalkRows w;
    w.b = pair / a.Hkv;
    w.h = pair % a.Hkv;
    w.wt0 = (tiles - 1 - tile) * 8;   // the rows with the longest walks first
    w.tpw = tpw;
    w.mtiles = mtiles;
    w.n = BlocksKvLen(a, w.b);
    w.m = BlocksQLen(a, w.b);
    if ((int)w.FirstRow(w.wt0) >= w.m) return;
    const BlocksWalkColumns<CT> col(a, w, wave, r);
    const uint32_t blocks = ((uint32_t)BlocksVisible(a, w.n, w.m, (int)w.EndRow() - 1) + a.bs - 1) / a.bs, tpb = a.bs / 16;

    // a negative scale is the queries' sign, a zero one makes them zero: the walk's own scale is positive
    const float scale2 = a.scale2 == 0.f ? 1.f : fabsf(a.scale2);
    u32x4_t q[CT][KS];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        BlocksLoadRows<KS>(a.q + w.b * a.qs[0] + (int64_t)col.Row(w, c) * a.qs[1] + col.head[c] * a.qs[2] + g * 8, q[c]);
        if (a.scale2 <= 0.f)
#pragma unroll
            for (int s = 0; s < KS; ++s) q[c][s] = a.scale2 == 0.f ? u32x4_t{0u, 0u, 0u, 0u} : q[c][s] ^ 0x80008000u;
    }
    const BlocksWalkAddresses<DC> ad(lane);
    f32x4_t o[CT][DC];
    float top[CT], sum[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
#pragma unroll
        for (int d = 0; d < DC; ++d) o[c][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        top[c] = -__builtin_inff();
        sum[c] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[c][s]));   // here, not in the loop, is where these loads are waited for
    }
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
                if (any)
                    BlocksWalkAttend<BF16, DC, CT, NT>(scale2, ad, at + z * S::D * 32, start, mask, col, g * 4, q, o, top, sum, load);
            }
            load();
        }
        __syncthreads();
    }
    // A value that is not finite may have met the weight 0 of a row that does not look at it.  Such columns are rare: their query rows are done again one by
    // one, where nothing but what a row sees takes part.
    float bad = 0.f;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        sum[c] = BlocksSumOver4(sum[c]);
        bad += sum[c] * 0.f;
#pragma unroll
        for (int d = 0; d < DC; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) bad += o[c][d][i] * 0.f;
    }
    if (__ballot(bad != 0.f)) {
        const uint32_t first_head = w.h * a.G + col.mt * 16 * CT, heads = mtiles > 1 ? col.cols : a.G;
        for (uint32_t x = 0; x < col.rows * ((heads + 15) / 16); ++x) {
            const uint32_t t = col.t0 + x % col.rows, h0 = x / col.rows * 16, some = min(16u, heads - h0), head = first_head + h0 + min(r, some - 1);
            const int vis = BlocksVisible(a, w.n, w.m, (int)t);
            top[0] = -__builtin_inff();
            sum[0] = 0.f;
#pragma unroll
            for (int d = 0; d < DC; ++d) o[0][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            int block;
            int64_t ko, vo;
            const uint32_t count = vis > 0 ? BlocksGatherProbes(a, a.probes + (((int64_t)w.b * a.Tq + t) * a.Hkv + w.h) * a.P, w.b, vis, s_scratch[wave], lane, block, ko, vo) : 0;
            if (count) {
                BlocksLoadRows<KS>(a.q + w.b * a.qs[0] + (int64_t)t * a.qs[1] + head * a.qs[2] + g * 8, q[0]);
                BlocksAttendRange<BF16, DC>(a, w.h, vis, block, ko, vo, 0, count * tpb, lane, q[0], o[0], top[0], sum[0]);
            }
            sum[0] = BlocksSumOver4(sum[0]);
            if (r < some) BlocksAttendStore<BF16, DC>(a, w.b, t, head, g, o[0], top[0], sum[0], out, lse);
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        if (!col.live[c]) continue;
        const float inv = sum[c] > 0.f ? 1.f / sum[c] : 0.f;
        const uint32_t t = col.t0 + col.in[c];
        uint16_t* dst = out + w.b * a.os[0] + (int64_t)t * a.os[1] + col.head[c] * a.os[2] + g * 4;
#pragma unroll
        for (int d = 0; d < DC; ++d)
            *reinterpret_cast<u32x2_t*>(dst + d * 16) =
                u32x2_t{BlocksPack<BF16>(o[c][d][0] * inv, o[c][d][1] * inv), BlocksPack<BF16>(o[c][d][2] * inv, o[c][d][3] * inv)};
        if (lse && g == 0) lse[((int64_t)w.b * a.Tq + t) * a.Hq + col.head[c]] = sum[c] == 0.f ? -__builtin_inff() : (top[c] + __log2f(sum[c])) * kLn2;
    }
}

// ---- attention weights of the cache rows ------------------------------------------------------------------------------------------------------
// One query row per sequence: a cache row gets the weights of one group's heads, from one wavefront.  `shares` workgroups divide a pair: its probed tiles, whose
// masses are written with their weights, and the copying of all other rows' masses.  Bound by memory in a batch (64 sequences of up to 32768 rows, 32 x 64 of
// them probed, 8 heads of 128 dimensions, 403 MB: 102 us, 3.9 TB/s); one sequence 7.3 us (28 by a workgroup for each head).
template <bool BF16, int DC>
__global__ void __launch_bounds__(512) BlocksWeighTokenKernel(BlocksArgs a, uint32_t mtiles, uint32_t vector, uint32_t shares, const float* __restrict__ lse,
                                                              const float* mass_in, float* mass_out) {
    TakeWholeRegisterFile();
    constexpr int KS = DC / 2;
    __shared__ uint32_t s_scratch[8][64], s_probed[GPANN_BLOCKS_MAX_BLOCKS / 32];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t pair = blockIdx.x / shares, share = blockIdx.x % shares, b = pair / a.Hkv, h = pair % a.Hkv;
    const int n = BlocksKvLen(a, b), visible = a.Tq ? BlocksVisible(a, n, BlocksQLen(a, b), 0) : 0;
    const float* from = mass_in + (uint64_t)pair * a.Tk;
    float* to = mass_out + (uint64_t)pair * a.Tk;
    const bool copies = mass_in != mass_out;
    if (copies) {
        s_probed[threadIdx.x] = 0;
        __syncthreads();
    }
    int block;
    int64_t ko, vo;
    const uint32_t count = visible > 0 ? BlocksGatherProbes(a, a.probes + (int64_t)pair * a.P, b, visible, s_scratch[wave], lane, block, ko, vo) : 0;
    const uint32_t tpb = a.bs / 16, units = count * tpb;
    auto load = [&](uint32_t u, u32x4_t(&rows)[KS], int& start, float& before) {   // (clamped behind the last unit: of no use there)
        const uint32_t unit = min(u, units - 1), slot = unit / tpb, base = unit % tpb * 16;
        const int blk = __builtin_amdgcn_readlane(block, (int)slot), last = visible - 1 - blk * (int)a.bs;
        start = blk * (int)a.bs + (int)base;
        BlocksLoadRows<KS>(a.k + BlocksReadLane64(ko, slot) + h * a.ks[2] + min((int)(base + r), last) * a.ks[1] + g * 8, rows);
        before = from[min(start + (int)(g * 4 + (r & 3)), (int)a.Tk - 1)];
    };
    u32x4_t kr[KS], q[KS];
    int start = 0;
    float before = 0.f, l0 = 0.f;
    const uint32_t heads0 = min(16u, a.G);
    const uint32_t u0 = share * 8 + wave;
    if (u0 < units) {
        load(u0, kr, start, before);
        BlocksLoadRows<KS>(a.q + b * a.qs[0] + (h * a.G + min(r, heads0 - 1)) * a.qs[2] + g * 8, q);
        l0 = lse[(int64_t)b * a.Hq + h * a.G + min(r, heads0 - 1)];
    }
    if (copies) {
        if (wave == 0 && lane < count) atomicOr(s_probed + block / 32, 1u << (block & 31));
        __syncthreads();
        auto probed = [&](uint32_t row) { return (s_probed[row / a.bs / 32] >> (row / a.bs & 31)) & 1; };
        // a batch of loads, then their stores (which the compiler has to take for writes to what is loaded next)
        const uint32_t part = ((a.Tk + shares - 1) / shares + 3) & ~3u, row0 = share * part, rows = min(a.Tk, row0 + part);
        constexpr uint32_t SOME = 8;
        if (vector)
            for (uint32_t i0 = row0 + threadIdx.x * 4; i0 < rows; i0 += 2048 * SOME) {
                f32x4_t x[SOME];
#pragma unroll
                for (uint32_t y = 0; y < SOME; ++y) x[y] = *reinterpret_cast<const f32x4_t*>(from + min(i0 + y * 2048, rows - 4));
#pragma unroll
                for (uint32_t y = 0; y < SOME; ++y)
                    if (i0 + y * 2048 < rows && !probed(i0 + y * 2048)) *reinterpret_cast<f32x4_t*>(to + i0 + y * 2048) = x[y];
            }
        else
            for (uint32_t i0 = row0 + threadIdx.x; i0 < rows; i0 += 512 * SOME) {
                float x[SOME];
#pragma unroll
                for (uint32_t y = 0; y < SOME; ++y) x[y] = from[min(i0 + y * 512, rows - 1)];
#pragma unroll
                for (uint32_t y = 0; y < SOME; ++y)
                    if (i0 + y * 512 < rows && !probed(i0 + y * 512)) to[i0 + y * 512] = x[y];
            }
    }
    for (uint32_t u = u0; u < units; u += 8 * shares) {
        u32x4_t next[KS];
        int next_start;
        float next_before;
        load(u + 8 * shares, next, next_start, next_before);
        f32x4_t w = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t mt = 0; mt < mtiles; ++mt) {
            const uint32_t heads = min(16u, a.G - mt * 16), head = h * a.G + mt * 16 + min(r, heads - 1);
            if (mtiles > 1) BlocksLoadRows<KS>(a.q + b * a.qs[0] + head * a.qs[2] + g * 8, q);
            const float l = mtiles > 1 ? lse[(int64_t)b * a.Hq + head] : l0, lse2 = l == -__builtin_inff() ? __builtin_inff() : l * kLog2e;
            f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS; ++j) s = BlocksMfma<BF16>(kr[j], q[j], s);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] += r < heads ? BlocksExp2(s[i] * a.scale2 - lse2) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = BlocksSumRow16(w[i]);
            const int key = start + (int)g * 4 + i;
            if ((int)r == i && key < (copies ? (int)a.Tk : visible)) to[key] = key < visible ? before + w[i] : before;
        }
        start = next_start;
        before = next_before;
#pragma unroll
        for (int j = 0; j < KS; ++j) kr[j] = next[j];
    }
}

// Many query rows: a wavefront takes a 64-key piece of a block, lists the query rows that probe it and lets their heads stream past the keys, 16 rows a
// product with a key per lane column; what a key gets is added in one lane group's registers.  Wavefronts share nothing and go from piece to piece (those of a
// pair on one die): a piece is two or three dependent trips to memory, so what counts is that eight are always under way on a CU.  8 sequences x 128 query rows,
// 32 probes of 64 rows in 32768, 8 key/value heads of 128 dimensions: 118 us.
template <bool BF16, int DC>
__global__ void __launch_bounds__(512) BlocksWeighKernel(BlocksArgs a, uint32_t words, uint32_t pieces, const uint32_t* __restrict__ bits, const float* __restrict__ lse,
                                                         const float* mass_in, float* mass_out) {
    TakeWholeRegisterFile();
    constexpr int KS = DC / 2;
    struct About {
        float lse2;
        int visible;
    };
    __shared__ uint16_t s_list[8][kRange];
    __shared__ About s_about[8][16];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t die = blockIdx.x & 7, pairs = a.B * a.Hkv, per_pair = a.nblk * pieces, waves = (gridDim.x >> 3) * 8;
    const uint64_t tasks = (uint64_t)((pairs + 7 - die) / 8) * per_pair;   // of the pairs that are `die` modulo 8
    const uint32_t inverse = a.G > 1 ? 0xFFFFFFFFu / a.G + 1 : 0;
    // a pair's pieces are dealt to the wavefronts in an order of its own: the first block, which most query rows probe, would else always fall to the same one
    auto piece_of = [&](uint64_t task, uint32_t& pair) -> uint32_t {
        const uint32_t which = (uint32_t)(task / per_pair);
        pair = which * 8 + die;
        return (uint32_t)((task % per_pair + (uint64_t)which * 61) % per_pair);
    };
    auto first_words = [&](uint64_t task) -> uint32_t {
        if (task >= tasks) return 0u;
        uint32_t pair;
        const uint32_t x = piece_of(task, pair);
        const uint64_t block = (uint64_t)pair * a.nblk + x / pieces;
        return lane < words ? bits[block * words + lane] : 0u;
    };
    uint64_t task = (blockIdx.x >> 3) * 8 + wave;
    uint32_t ahead = first_words(task);
    for (; task < tasks; task += waves) {
        uint32_t pair;
        const uint32_t x = piece_of(task, pair), block = x / pieces, in_block = x % pieces * 64;
        const uint32_t b = pair / a.Hkv, h = pair % a.Hkv, tiles = min(4u, (a.bs - in_block) / 16);
        const int key0 = (int)(block * a.bs + in_block), mine = key0 + (int)lane;
        const bool writes = lane < tiles * 16 && mine < (int)a.Tk;
        const float before = writes ? mass_in[(uint64_t)pair * a.Tk + mine] : 0.f;
        uint32_t word = ahead;
        ahead = first_words(task + waves);
        const int n = BlocksKvLen(a, b), m = BlocksQLen(a, b);
        float w[4] = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t first = 0;;) {
            const uint32_t c = (uint32_t)__popc(word);
            uint32_t at = c;
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t y = __shfl_up(at, s);
                if ((int)lane >= s) at += y;
            }
            const uint32_t rows = (uint32_t)__builtin_amdgcn_readlane((int)at, 63) * a.G;
            at -= c;
            while (word) {
                s_list[wave][at++] = (uint16_t)(lane * 32 + (uint32_t)__ffs(word) - 1);
                word &= word - 1;
            }
            BlocksWaveSync();
            if (rows > 0) {
                u32x4_t kf[4][KS], q[KS];
                int64_t ko, vo;
                (void)BlocksBase(a, b, (int)block, ko, vo);
                const int last = n - 1 - (int)(block * a.bs);   // >= 0: a listed block holds a visible row
                const uint16_t* k = a.k + ko + h * a.ks[2] + g * 8;
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y) BlocksLoadRows<KS>(k + min((int)(in_block + min(y, tiles - 1) * 16 + r), last) * a.ks[1], kf[y]);
                float l;
                int t;
                auto load = [&](uint32_t row0, u32x4_t(&to)[KS]) {   // (clamped behind the last row: of no use there)
                    const uint32_t i = min(row0 + r, rows - 1), in = inverse ? __umulhi(i, inverse) : i, head = h * a.G + i - in * a.G;
                    t = (int)(first * 32 + s_list[wave][in]);
                    BlocksLoadRows<KS>(a.q + b * a.qs[0] + t * a.qs[1] + head * a.qs[2] + g * 8, to);
                    l = lse[((int64_t)b * a.Tq + t) * a.Hq + head];
                };
                load(0, q);
                for (uint32_t row0 = 0; row0 < rows; row0 += 16) {
                    if (g == 0) s_about[wave][r] = About{l == -__builtin_inff() ? __builtin_inff() : l * kLog2e, row0 + r < rows ? BlocksVisible(a, n, m, t) : 0};
                    u32x4_t next[KS];
                    load(row0 + 16, next);
                    BlocksWaveSync();
                    About about[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) about[j] = s_about[wave][g * 4 + j];
                    BlocksWaveSync();
                    f32x4_t s[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) s[y] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int y = 0; y < 4; ++y) s[y] = BlocksMfma<BF16>(q[j], kf[y][j], s[y]);
#pragma unroll
                    for (int y = 0; y < 4; ++y)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            w[y] += key0 + y * 16 + (int)r < about[j].visible ? BlocksExp2(s[y][j] * a.scale2 - about[j].lse2) : 0.f;
#pragma unroll
                    for (int j = 0; j < KS; ++j) q[j] = next[j];
                }
            }
            first += kRange / 32;
            if (first >= words) break;
            word = first + lane < words ? bits[((uint64_t)pair * a.nblk + block) * words + first + lane] : 0u;
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) w[y] = BlocksSumOver4(w[y]);
        const float more = g == 0 ? w[0] : g == 1 ? w[1] : g == 2 ? w[2] : w[3];   // lane = key of the piece
        if (writes) mass_out[(uint64_t)pair * a.Tk + mine] = before + more;
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------
static size_t WeighSpace(const BlocksArgs& a) { return a.Tq <= 1 ? 0 : BlocksAlign((size_t)a.B * a.Hkv * a.nblk * ((a.Tq + 31) / 32) * 4); }

template <bool BF16, int DC, int CT, int NT, int NM>
static gpann_status AttendWalk(const BlocksArgs& a, uint16_t* out, float* lse, hipStream_t st) {
    const uint32_t cols = 16 * CT, mtiles = (a.G + cols - 1) / cols, tpw = std::max(1u, cols / a.G);
    const uint64_t waves = mtiles > 1 ? (uint64_t)a.Tq * mtiles : (a.Tq + tpw - 1) / tpw, tiles = (waves + 7) / 8;
    return BlocksLaunch(BlocksAttendWalkKernel<BF16, DC, CT, NT, NM>, BlocksPairGrid((uint64_t)a.B * a.Hkv, tiles), BlocksWalkShape<DC>::LDS, st, a, tpw, mtiles, (uint32_t)tiles, out, lse);
}

// How a query row's keys are divided where there are few of them: over the wavefronts of a workgroup until the chip's 2048 have something to do, then, where
// that leaves more than two steps each and there are few of them, over workgroups until there is one per CU (8 heads of 128 dimensions, undivided and divided:
// 8 x 64 rows 10.0 and 10.1 us, 16 x 64 14.9 and 11.0, 32 x 64 24.1 and 12.8; 64 heads, 32 x 64: 27.3 and 21.8; 128 heads 28.8 and 29.6)
struct BlocksDivision {
    uint32_t waves = 1, splits = 1, mtiles;
    uint64_t pairs, tiles;
    explicit BlocksDivision(const BlocksArgs& a) : mtiles((a.G + 15) / 16), pairs((uint64_t)a.B * a.Hkv) {
        const uint64_t tasks = (uint64_t)a.Tq * mtiles, units = (uint64_t)std::min(a.P, a.nblk) * (a.bs / 16);
        while (waves < 8 && pairs * tasks * waves < 2048) waves *= 2;
        if (waves == 8 && units > 32 && pairs * tasks <= 64)
            while (pairs * tasks * splits * 2 <= 256 && splits * 16 < units) splits *= 2;
        tiles = (tasks * waves + 7) / 8;
    }
    size_t Space(uint32_t d) const { return splits > 1 ? BlocksAlign(pairs * tiles * splits * 16 * (d + 2) * 4) : 0; }
};
// ... where it has its wavefronts for itself: with more, neighbours share what they read (8 heads of 128 dimensions, 16 probes of 64 rows: 256 query rows 52 us
// apart, 68 together, 512 rows 100 and 100; 64 heads: 32 rows 56 and 107, 64 rows 104 and 104, 128 rows 194 and 109)
static bool BlocksApart(const BlocksArgs& a) { return a.Tq == 1 || (uint64_t)a.B * a.Hkv * a.Tq * ((a.G + 15) / 16) <= 2048; }
static size_t AttendSpace(const BlocksArgs& a, uint32_t d) { return BlocksApart(a) ? BlocksDivision(a).Space(d) : 0; }

template <bool BF16, int DC>
static gpann_status Attend(const BlocksArgs& a, uint16_t* out, float* lse, float* ws, hipStream_t st) {
    const uint64_t pairs = (uint64_t)a.B * a.Hkv;
    if (!BlocksApart(a)) {
        // 32 columns a wavefront read LDS half as often for each, but make half the workgroups (one per CU at a time) of a larger union: 32 heads of 128
        // dimensions, 8192 rows (1024 workgroups of 32 columns) 367 us against 419, 4096 rows (512) 273 and 278, 2048 rows (256) 170 and 162; 777 rows x 12 heads
        // of 96 (120) 122 and 79.  (Wide heads have no registers for it.)  Pairs of blocks of 32 rows in one chain of products, 777 rows: 79 us against 89.
        if constexpr (DC <= 8)
            if (pairs * (((uint64_t)a.Tq * a.G + 255) / 256) >= 512)
                return a.bs % 64 == 0   ? AttendWalk<BF16, DC, 2, 4, 1>(a, out, lse, st)
                       : a.bs % 32 == 0 ? AttendWalk<BF16, DC, 2, 2, 1>(a, out, lse, st)
                                        : AttendWalk<BF16, DC, 2, 2, 2>(a, out, lse, st);
        if constexpr (DC <= 8)
            if (a.bs % 32 == 0) return a.bs % 64 == 0 ? AttendWalk<BF16, DC, 1, 4, 1>(a, out, lse, st) : AttendWalk<BF16, DC, 1, 4, 2>(a, out, lse, st);
        return a.bs % 32 == 0 ? AttendWalk<BF16, DC, 1, 2, 1>(a, out, lse, st) : AttendWalk<BF16, DC, 1, 2, 2>(a, out, lse, st);
    }
    const BlocksDivision v(a);
    const size_t lds = std::max<size_t>(BlocksTokenShape<DC>::RING, v.waves > 1 ? (size_t)8 * 16 * (DC * 16 + 2) * 4 : 0);
    GPANN_TRY(BlocksLaunch(BlocksAttendKernel<BF16, DC>, BlocksPairGrid(pairs, v.tiles * v.splits), lds, st, a, v.waves, v.splits, v.mtiles, (uint32_t)v.tiles, out, lse, ws));
    if (v.splits == 1) return GPANN_OK;
    hipLaunchKernelGGL(BlocksAttendJoinKernel<BF16>, dim3((std::min(16u, a.G) * DC * 8 + 255) / 256, (uint32_t)(pairs * v.tiles)), dim3(256), 0, st, a, DC * 16, v.splits,
                       v.mtiles, (uint32_t)v.tiles, ws, out, lse);
    GPANN_HIP_TRY(hipGetLastError());
    return GPANN_OK;
}

template <bool BF16, int DC>
static gpann_status Weigh(const BlocksArgs& a, const float* lse, const float* mass_in, float* mass_out, char* ws, hipStream_t st) {
    const uint64_t pairs = (uint64_t)a.B * a.Hkv;
    if (a.Tq <= 1) {
        const uint32_t vector = a.Tk % 4 == 0 && BlocksAligned(16, mass_in) && BlocksAligned(16, mass_out) ? 1 : 0;
        uint32_t shares = 1;   // a pair is divided until there is a workgroup per CU, or a tile a wavefront
        while (pairs * shares * 2 <= 256 && shares * 16 <= std::min(a.P, a.nblk) * (a.bs / 16)) shares *= 2;
        return BlocksLaunch(BlocksWeighTokenKernel<BF16, DC>, pairs * shares, 0, st, a, (a.G + 15) / 16, vector, shares, lse, mass_in, mass_out);
    }
    const uint32_t words = (a.Tq + 31) / 32, pieces = (a.bs + 63) / 64;
    uint32_t* bits = reinterpret_cast<uint32_t*>(ws);
    GPANN_TRY(BlocksMarkProbes(a, words, bits, st));
    const uint64_t tasks = pairs * a.nblk * pieces;   // one workgroup per CU, fewer where there is less to do; a multiple of the eight dies
    const uint64_t grid = std::min<uint64_t>(256, (tasks + 63) / 64 * 8);
    return BlocksLaunch(BlocksWeighKernel<BF16, DC>, grid, 0, st, a, words, pieces, bits, lse, mass_in, mass_out);
}

}  // namespace gpann

using namespace gpann;

extern "C" {

gpann_status gpann_blocks_workspace_bytes(const gpann_blocks_layout* L, uint32_t nprobe, uint32_t calls, size_t* out_bytes) {
    GPANN_REQUIRE(out_bytes != nullptr, "out_bytes is null");
    GPANN_TRY(BlocksCheckLayout(L));
    GPANN_REQUIRE(nprobe <= GPANN_BLOCKS_MAX_PROBE, "nprobe above GPANN_BLOCKS_MAX_PROBE");
    GPANN_REQUIRE((calls & ~31u) == 0, "unknown bits in calls");
    const BlocksArgs a = BlocksMakeArgs(L, nullptr, nullptr, nullptr, nullptr, nprobe);
    size_t need = 0;
    if (calls & GPANN_BLOCKS_ATTEND) need = std::max(need, AttendSpace(a, L->head_dim));
    if (calls & GPANN_BLOCKS_BACKWARD) need = std::max(need, BlocksBackwardSpace(a, L->head_dim));
    if (calls & GPANN_BLOCKS_WEIGH) need = std::max(need, WeighSpace(a));
    *out_bytes = need;
    return GPANN_OK;
}

gpann_status gpann_blocks_attend(const gpann_blocks_layout* L, const void* q, const void* k, const void* v, const int32_t* probes, uint32_t nprobe, void* out,
                                 float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    GPANN_TRY(BlocksCheckLayout(L));
    GPANN_REQUIRE(q && k && v && probes && out, "a tensor is null");
    GPANN_REQUIRE(BlocksAligned(16, q) && BlocksAligned(16, k) && BlocksAligned(16, v) && BlocksAligned(16, out), "q, k, v and out must be 16-byte aligned");
    GPANN_REQUIRE(BlocksAligned(4, probes) && BlocksAligned(4, lse), "probes and lse must be 4-byte aligned");
    GPANN_REQUIRE(nprobe >= 1 && nprobe <= GPANN_BLOCKS_MAX_PROBE, "nprobe must be 1 .. GPANN_BLOCKS_MAX_PROBE");
    GPANN_REQUIRE(BlocksDisjoint(L->out_stride, L->batch, L->q_rows, L->q_heads, L->head_dim), "out overlaps itself");
    const BlocksArgs a = BlocksMakeArgs(L, q, k, v, probes, nprobe);
    GPANN_TRY(BlocksCheckWorkspace(workspace, workspace_bytes, AttendSpace(a, L->head_dim)));
    GPANN_BLOCKS_ENTER(L, stream);
    if (a.B == 0 || a.Tq == 0) return GPANN_OK;
    GPANN_BLOCKS_DISPATCH(L, Attend, a, static_cast<uint16_t*>(out), lse, static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
}

gpann_status gpann_blocks_weigh(const gpann_blocks_layout* L, const void* q, const void* k, const int32_t* probes, uint32_t nprobe, const float* lse,
                                const float* mass_in, float* mass_out, void* workspace, size_t workspace_bytes, void* stream) {
    GPANN_TRY(BlocksCheckLayout(L));
    GPANN_REQUIRE(q && k && probes && lse && mass_in && mass_out, "a tensor is null");
    GPANN_REQUIRE(BlocksAligned(16, q) && BlocksAligned(16, k), "q and k must be 16-byte aligned");
    GPANN_REQUIRE(BlocksAligned(4, probes) && BlocksAligned(4, lse) && BlocksAligned(4, mass_in) && BlocksAligned(4, mass_out), "probes, lse and mass must be 4-byte aligned");
    GPANN_REQUIRE(nprobe >= 1 && nprobe <= GPANN_BLOCKS_MAX_PROBE, "nprobe must be 1 .. GPANN_BLOCKS_MAX_PROBE");
    if (L->q_rows > 1) GPANN_TRY(BlocksCheckMarks(L));
    const BlocksArgs a = BlocksMakeArgs(L, q, k, nullptr, probes, nprobe);
    GPANN_TRY(BlocksCheckWorkspace(workspace, workspace_bytes, WeighSpace(a)));
    GPANN_BLOCKS_ENTER(L, stream);
    if (a.B == 0 || a.Tk == 0) return GPANN_OK;
    GPANN_BLOCKS_DISPATCH(L, Weigh, a, lse, mass_in, mass_out, static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
}

}  // extern "C"

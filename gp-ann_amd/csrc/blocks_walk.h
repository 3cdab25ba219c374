// blocks_walk.h — how a workgroup walks the blocks that neighbouring query rows probe (blocks_attend.hip, blocks_grad.hip).
//
// A wavefront's 16 CT matrix columns are the heads of a group of max(1, 16 CT / G) neighbouring query rows; a workgroup holds eight wavefronts.  The walk
// goes over the UNION of the blocks its query rows probe, in block order: every row of K and V enters LDS once for the workgroup, and a wavefront multiplies
// the blocks that one of its own query rows probes.  Neighbouring rows share most of their probes (their own block, the first one, what their text is about),
// so the union is far smaller than the sum; a 16-column tile costs the same whether one or all of its rows want the block.
//
// Rows go to LDS by DMA (no registers, issued stages ahead), 64 rows of K and of V a stage.  The 16-byte chunks of a row are permuted by a function of the
// row such that both ways of reading are free of bank conflicts: by rows (ds_read_b128) and transposed (ds_read_b64_tr_b16).
#pragma once

#include "blocks_tile.h"

namespace gpann {

template <int DC>
struct BlocksWalkShape {
    static constexpr uint32_t D = DC * 16, CPR = D / 8, ROWS = 64, TENSOR = ROWS * D * 2, STAGE = 2 * TENSOR;
    static constexpr uint32_t LOADS = CPR / 4;   // DMA instructions of a wavefront per stage
    // Stages go in groups, one being multiplied and one on its way: a barrier a group.  (Two stages a group, because a wavefront multiplies few or many of a
    // stage's tiles, and has to wait for the slowest one at every barrier.)
    static constexpr uint32_t GROUP = D <= 128 ? 2 : 1, BUFFERS = 2 * GROUP;
    static constexpr uint32_t WINDOW = D <= 96 ? 1024 : 512;   // blocks that LDS has room for at a time
    static constexpr size_t LDS = (size_t)BUFFERS * STAGE + WINDOW * (sizeof(uint4) + 32 + 4);

    // Slot of a row's chunk: an exclusive or with a function of the row.  LDS serves 256 bytes a cycle, so the lanes that it serves together have to lie in
    // sixteen different slots modulo 16, and a row begins CPR slots after the one before.  Read by rows, lanes {0-3, 12-15, 20-27}, {4-11, 16-19, 28-31} and the
    // same of the upper half go together: eight rows' chunk c and the eight others' chunk c + 1.  Transposed, half a wavefront goes together: eight rows'
    // chunks c and c + 1.  So the rows of each eight get different pairs of slots, and two rows that share a pair are both of the eight rows of one kind, with
    // different slots, or of different kinds, with the same one.
    static constexpr uint32_t TURNS = CPR % 16 == 0 ? 16 : CPR % 8 == 0 ? 8 : 4;
    static __device__ __forceinline__ uint32_t Turn(uint32_t row) {
        const uint32_t eighth = (row >> 3) & 1;
        return (((row / (16 / TURNS)) & (TURNS / 2 - 1)) ^ (eighth * (TURNS / 4))) << 1 | eighth;
    }
    static __device__ __forceinline__ uint32_t Slot(uint32_t chunk, uint32_t row) { return chunk ^ Turn(row); }   // and the chunk of a slot
};

// One LDS-DMA wave-instruction: 64 lanes x 16 bytes from base + offset to LDS bytes [lds, lds + 1024).  The compiler neither sees the bytes nor counts
// it in vmcnt: BlocksDmaWait comes before the barrier that publishes them (waits of its own only get longer by it).
__device__ __forceinline__ void BlocksDma(uint64_t base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "m0", "memory");
}
// ... from an address per lane
__device__ __forceinline__ void BlocksDmaFrom(const void* src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "m0", "memory");
}
// ... 4 bytes a lane, to LDS bytes [lds, lds + 256)
__device__ __forceinline__ void BlocksDmaWordFrom(const void* src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(src), "s"(lds) : "m0", "memory");
}
template <int LEFT>
__device__ __forceinline__ void BlocksDmaWait() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LEFT) : "memory");
}
// the same for a number known at run time (at most 16: with more in flight than that, until 16 are)
__device__ __forceinline__ void BlocksDmaWaitFor(uint32_t left) {
    switch (left) {
#define GPANN_WAIT(n) \
    case n: BlocksDmaWait<n>(); break;
        GPANN_WAIT(0) GPANN_WAIT(1) GPANN_WAIT(2) GPANN_WAIT(3) GPANN_WAIT(4) GPANN_WAIT(5) GPANN_WAIT(6) GPANN_WAIT(7) GPANN_WAIT(8) GPANN_WAIT(9)
        GPANN_WAIT(10) GPANN_WAIT(11) GPANN_WAIT(12) GPANN_WAIT(13) GPANN_WAIT(14) GPANN_WAIT(15)
        default: BlocksDmaWait<16>();
#undef GPANN_WAIT
    }
}
// every wavefront has its share of a stage in LDS and has read what it needs of the stage before
__device__ __forceinline__ void BlocksStageBarrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ uint32_t BlocksLdsAddress(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }
typedef short s16x4_t __attribute__((ext_vector_type(4)));
// lane l of 16: address of (row l / 4, four elements l % 4) of a 4 x 16 tile -> column l of its four rows
__device__ __forceinline__ u32x2_t BlocksReadTransposed(uint32_t lds) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)lds));
}
__device__ __forceinline__ u32x4_t BlocksReadRow(uint32_t lds) { return *(__attribute__((address_space(3))) const u32x4_t*)lds; }

// What a workgroup's query rows are
struct BlocksWalkRows {
    uint32_t b, h, wt0, tpw, mtiles;   // wavefront w: column tile wt0 + w; tpw query rows each, or one of mtiles tiles of a row's heads
    int n, m;
    __device__ __forceinline__ uint32_t FirstRow(uint32_t wt) const { return mtiles > 1 ? wt / mtiles : wt * tpw; }
    __device__ __forceinline__ uint32_t EndRow() const { return min((uint32_t)m, mtiles > 1 ? FirstRow(wt0 + 7) + 1 : FirstRow(wt0 + 8)); }
};
// ... a wavefront's
template <int CT>
struct BlocksWalkColumns {
    uint32_t t0, rows;                // first query row, how many are live
    int seen_by_all, seen_by_any;     // cache rows (a prefix) that its first and its last query row see
    uint32_t cols, mt;                // columns in use
    uint32_t in[CT], head[CT];        // this lane's columns: query row - t0, query head
    int visible[CT];
    bool live[CT];
    __device__ __forceinline__ BlocksWalkColumns(const BlocksArgs& a, const BlocksWalkRows& w, uint32_t wave, uint32_t r) {
        t0 = w.FirstRow(w.wt0 + wave);
        mt = w.mtiles > 1 ? (w.wt0 + wave) % w.mtiles : 0;
        cols = w.mtiles > 1 ? min(16u * CT, a.G - mt * 16 * CT) : w.tpw * a.G;
        rows = (int)t0 < w.m ? min(w.tpw, (uint32_t)w.m - t0) : 0;
        seen_by_all = rows ? BlocksVisible(a, w.n, w.m, (int)t0) : 0;
        seen_by_any = rows ? BlocksVisible(a, w.n, w.m, (int)(t0 + rows - 1)) : 0;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const uint32_t col = min(c * 16 + r, cols - 1);
            in[c] = w.mtiles > 1 ? 0 : col / a.G;
            head[c] = w.h * a.G + (w.mtiles > 1 ? mt * 16 * CT + col : col % a.G);
            live[c] = in[c] < rows && c * 16 + r < cols;
            visible[c] = in[c] < rows ? BlocksVisible(a, w.n, w.m, (int)(t0 + in[c])) : 0;
        }
    }
    __device__ __forceinline__ uint32_t Row(const BlocksWalkRows& w, int c) const { return min(t0 + in[c], (uint32_t)w.m - 1); }
};

// LDS of a walk behind the stages
template <int DC>
struct BlocksWalkTables {
    uint4* address;    // [WINDOW] of the list's blocks: byte addresses of the first row of the head in K and V
    uint32_t* masks;   // [WINDOW][8] which query rows of a wavefront probe a block
    int* list;         // [WINDOW] the blocks with any, ascending
    __device__ __forceinline__ explicit BlocksWalkTables(char* lds) {
        using S = BlocksWalkShape<DC>;
        address = reinterpret_cast<uint4*>(lds + S::BUFFERS * S::STAGE);
        masks = reinterpret_cast<uint32_t*>(address + S::WINDOW);
        list = reinterpret_cast<int*>(masks + S::WINDOW * 8);
    }
};

// Fills the tables for the blocks [window, window + in_window) and returns the length of the list.  Ends with a barrier.
template <int DC>
__device__ __forceinline__ uint32_t BlocksWalkList(const BlocksArgs& a, const BlocksWalkRows& w, uint32_t window, uint32_t in_window, const BlocksWalkTables<DC>& tab,
                                                   uint32_t* s_count) {
    const uint32_t tid = threadIdx.x;
    for (uint32_t i = tid; i < in_window * 8; i += 512) tab.masks[i] = 0;
    __syncthreads();
    const uint32_t t0 = w.FirstRow(w.wt0), t1 = w.EndRow();
    const uint32_t entries = t1 > t0 ? (t1 - t0) * a.P : 0;
    for (uint32_t i = tid; i < entries; i += 512) {
        const uint32_t t = t0 + i / a.P;
        const int p = a.probes[(((int64_t)w.b * a.Tq + t) * a.Hkv + w.h) * a.P + i % a.P];
        if (p < (int)window || (uint32_t)p >= window + in_window || (int64_t)p * a.bs >= BlocksVisible(a, w.n, w.m, (int)t)) continue;
        uint32_t* row = tab.masks + ((uint32_t)p - window) * 8;
        if (w.mtiles > 1) {
            for (uint32_t x = t * w.mtiles; x < (t + 1) * w.mtiles; ++x)
                if (x >= w.wt0 && x < w.wt0 + 8) row[x - w.wt0] = 1;
        } else {
            atomicOr(row + (t - t0) / w.tpw, 1u << (t - t0) % w.tpw);
        }
    }
    __syncthreads();
    if (tid < 64) {
        uint32_t at = 0;
        for (uint32_t j0 = 0; j0 < in_window; j0 += 64) {
            const uint32_t j = j0 + tid;
            bool any = false;
            int64_t ko = 0, vo = 0;
            if (j < in_window) {
                const uint4 x = *reinterpret_cast<const uint4*>(tab.masks + j * 8), y = *reinterpret_cast<const uint4*>(tab.masks + j * 8 + 4);
                any = (x.x | x.y | x.z | x.w | y.x | y.y | y.z | y.w) != 0 && BlocksBase(a, w.b, (int)(window + j), ko, vo);
            }
            const uint64_t votes = __ballot(any);
            if (any) {
                const uint32_t e = at + (uint32_t)__popcll(votes & ((1ull << tid) - 1));
                const uint64_t k = (uint64_t)(a.k + ko + w.h * a.ks[2]), v = (uint64_t)(a.v + vo + w.h * a.vs[2]);
                tab.address[e] = uint4{(uint32_t)k, (uint32_t)(k >> 32), (uint32_t)v, (uint32_t)(v >> 32)};
                tab.list[e] = (int)(window + j);
            }
            at += (uint32_t)__popcll(votes);
        }
        if (tid == 0) *s_count = at;
    }
    __syncthreads();
    return *s_count;
}

// What a stage's loads and products have to know of its four 16-row tiles, for sixteen stages at a time: tile y of stage s in lane 4 (s % 16) + y
constexpr uint32_t kDescribed = 16;
struct BlocksWalkSource {
    uint2 k, v;        // addresses of its first row
    int last;          // its last row that the sequence has, in the tile
};
struct BlocksWalkStage {
    int start;         // its position
    uint32_t mask;     // which query rows of this wavefront look at it
};

// The walk's bookkeeping and its DMA side: which rows and chunks of a tile a lane loads is the same in every stage
template <int DC>
struct BlocksWalker {
    using S = BlocksWalkShape<DC>;
    // byte offsets in a tile: all of a wavefront's instructions of a stage have the same two where a row is a power of two of chunks, of keys and of values
    static constexpr bool POWER = (S::CPR & (S::CPR - 1)) == 0;
    static constexpr uint32_t PLACES = POWER ? 2 : S::LOADS;
    uint32_t place[PLACES];
    uint32_t wave, lane, tpb, inverse, krow, vrow;
    __device__ __forceinline__ BlocksWalker(const BlocksArgs& a, uint32_t wave_, uint32_t lane_) : wave(wave_), lane(lane_), tpb(a.bs / 16) {
        inverse = tpb > 1 ? 0xFFFFFFFFu / tpb + 1 : 0;
        krow = (uint32_t)a.ks[1] * 2;
        vrow = (uint32_t)a.vs[1] * 2;
#pragma unroll
        for (uint32_t x = 0; x < PLACES; ++x) place[x] = Place(POWER ? 0 : x, POWER ? x == 1 : wave + 8 * x >= S::CPR, 15);
    }
    __device__ __forceinline__ uint32_t Place(uint32_t x, bool value, int last) const {
        const uint32_t at = (wave + 8 * x) % S::CPR * 64 + lane, r = at / S::CPR % 16;
        return (uint32_t)min((int)r, last) * (value ? vrow : krow) + S::Slot(at % S::CPR, r) * 16;
    }
    // of the stages from s on; `seen`: rows that the last query row of this wavefront sees (a prefix)
    __device__ __forceinline__ BlocksWalkSource Describe(const BlocksArgs& a, const BlocksWalkRows& w, const BlocksWalkTables<DC>& tab, uint32_t window, uint32_t s,
                                                         uint32_t units, int seen, BlocksWalkStage& st) const {
        BlocksWalkSource d;
        const uint32_t unit = 4 * s + lane, in = min(unit, units - 1), e = inverse ? __umulhi(in, inverse) : in;   // in / tpb, exact below 2^16
        const int block = tab.list[e], row = (int)(in - e * tpb) * 16, last = w.n - 1 - block * (int)a.bs;
        const uint32_t first = (uint32_t)min(row, last & ~15);   // a tile behind the sequence's end: its last one's rows (nobody looks at them)
        const uint4 base = tab.address[e];
        const uint64_t k = (((uint64_t)base.y << 32) | base.x) + (uint64_t)first * krow, v = (((uint64_t)base.w << 32) | base.z) + (uint64_t)first * vrow;
        d.k = uint2{(uint32_t)k, (uint32_t)(k >> 32)};
        d.v = uint2{(uint32_t)v, (uint32_t)(v >> 32)};
        d.last = min(15, last - (int)first);
        st.start = block * (int)a.bs + row;
        st.mask = tab.masks[(block - (int)window) * 8 + (int)wave];
        if (unit >= units || st.start >= seen) st.mask = 0;
        return d;
    }
    __device__ __forceinline__ void Load(const BlocksWalkSource& d, uint32_t s, uint32_t to) const {
#pragma unroll
        for (uint32_t x = 0; x < S::LOADS; ++x) {
            const uint32_t j = wave + 8 * x;
            const bool value = POWER ? x >= S::CPR / 8 : j >= S::CPR;
            const int tile = (int)(s % kDescribed * 4 + j % S::CPR / (S::CPR / 4));   // 16 rows are CPR / 4 instructions
            const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(value ? d.v.x : d.k.x), tile);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(value ? d.v.y : d.k.y), tile);
            const int last = __builtin_amdgcn_readlane(d.last, tile);
            uint32_t offset = place[POWER ? (value ? 1 : 0) : x];
            if (last < 15) offset = Place(x, value, last);   // rows past the sequence's end are not read
            BlocksDma(((uint64_t)hi << 32) | lo, offset, to + (value ? S::TENSOR : 0) + j % S::CPR * 1024);
        }
    }
};

// LDS addresses of a lane's part of a stage's operands.  A permuted chunk is an exclusive or in the low bits, so step s and dimension tile d are one exclusive
// or and one constant away from a base (stages begin at multiples of 1024 bytes): two registers instead of one for every step and tile.
template <int DC>
struct BlocksWalkAddresses {
    using S = BlocksWalkShape<DC>;
    uint32_t rows, turned, first;
    // `first_`: the first of the dimension tiles that this lane's wavefront reads transposed
    __device__ __forceinline__ explicit BlocksWalkAddresses(uint32_t lane, uint32_t first_ = 0) : first(first_) {
        const uint32_t r = lane & 15, g = lane >> 4, row = g * 4 + r / 4;
        rows = (r * S::CPR + S::Slot(g, r)) * 16;
        turned = (row * S::CPR + S::Slot((r & 3) / 2, row)) * 16 + (r & 1) * 8;
    }
    // by rows: step s of row lane % 16 of the tile at LDS byte `at`
    __device__ __forceinline__ void RowSteps(uint32_t at, uint32_t (&x)[DC / 2]) const {
        constexpr int N = S::TURNS / 4;
        uint32_t turn[N];
#pragma unroll
        for (int s = 0; s < N; ++s) {
            turn[s] = s == 0 ? at + rows : turn[0] ^ (64 * s);
            asm volatile("" : "+v"(turn[s]));   // (else the constant offsets that follow would be added on the vector unit, one by one)
        }
#pragma unroll
        for (int s = 0; s < DC / 2; ++s) x[s] = turn[s % N] + s / N * N * 64;
    }
    // transposed: 16 dimensions of rows 4 g .. of the tile at LDS byte `at`
    template <int COUNT>
    __device__ __forceinline__ void Dimensions(uint32_t at, uint32_t (&x)[COUNT]) const {
        constexpr int N = S::TURNS / 2;
        if constexpr (COUNT == DC || COUNT % N == 0 || N % COUNT == 0) {   // `first` is a multiple of COUNT: its bits are not d's
            uint32_t turn[COUNT < N ? COUNT : N];
#pragma unroll
            for (int d = 0; d < (COUNT < N ? COUNT : N); ++d) {
                turn[d] = d == 0 ? (at + turned + first / N * N * 32) ^ (first % N * 32) : turn[0] ^ (32 * d);
                asm volatile("" : "+v"(turn[d]));
            }
#pragma unroll
            for (int d = 0; d < COUNT; ++d) x[d] = turn[d % N] + d / N * N * 32;
        } else {
#pragma unroll
            for (int d = 0; d < COUNT; ++d) {
                x[d] = ((at + turned) ^ ((first + d) % N * 32)) + (first + d) / N * N * 32;
                asm volatile("" : "+v"(x[d]));
            }
        }
    }
};

// ---- which query rows probe a block: bits [sequence, head][block][query row] -----------------------------------------------------------------------
constexpr uint32_t kRange = 2048;   // query rows a wavefront lists at a time: 64 words

}  // namespace gpann

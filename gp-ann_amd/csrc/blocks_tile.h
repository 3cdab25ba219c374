// blocks_tile.h — matrix-core building blocks of the attention kernels over cache blocks (blocks_attend.hip).
//
// All products use the 16 x 16 x 32 matrix instruction: A and B hold, per lane l, eight consecutive k of row / column l % 16 (k = 8 * (l / 16) ..); C holds
// column l % 16, rows 4 * (l / 16) ...  Two facts of that layout carry every kernel here:
//   * a tile read "by rows" (lane l: row l % 16, 16 bytes at 32 * step + 8 * (l / 16)) is an operand of a product over the head dimension as it lies in
//     memory: queries, keys, values and output gradients go from HBM / L2 straight into the registers the matrix instruction reads;
//   * k may be permuted freely as long as A and B agree, so the C layout of one product (lane: four rows 4 g .. 4 g + 3 of two 16-row tiles, g = l / 16) IS
//     the operand layout of the next product over those 32 rows: probabilities never cross lanes.  The other operand then needs eight ROWS per lane at one
//     dimension: a tile read "by columns" — lane l: rows 4 g + i of both tiles, dimensions (l % 16) * DC .. + DC (DC = head_dim / 16) — whose 16-bit pairs
//     are turned with one v_perm_b32 per output register.  Output slot dt of lane column c is dimension c * DC + dt.
#pragma once

#include "blocks.h"

namespace gpann {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

template <bool BF16>
__device__ __forceinline__ f32x4_t BlocksMfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// two floats -> two 16-bit values, round to nearest even
template <bool BF16>
__device__ __forceinline__ uint32_t BlocksPack(float lo, float hi) {
    if constexpr (BF16) {
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        const bf16x2_t v = {(__bf16)lo, (__bf16)hi};
        return __builtin_bit_cast(uint32_t, v);
    } else {
        typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
        const f16x2_t v = {(_Float16)lo, (_Float16)hi};
        return __builtin_bit_cast(uint32_t, v);
    }
}
// eight values of two C tiles -> one operand over their 32 rows
template <bool BF16>
__device__ __forceinline__ u32x4_t BlocksPackOperand(const f32x4_t& a, const f32x4_t& b) {
    return u32x4_t{BlocksPack<BF16>(a[0], a[1]), BlocksPack<BF16>(a[2], a[3]), BlocksPack<BF16>(b[0], b[1]), BlocksPack<BF16>(b[2], b[3])};
}
// eight ones: the other operand's sum over its 32 rows, in every row of C
template <bool BF16>
__device__ __forceinline__ u32x4_t BlocksOnes() {
    constexpr uint32_t two = BF16 ? 0x3F803F80u : 0x3C003C00u;
    return u32x4_t{two, two, two, two};
}

// by rows: `p` = the lane's row + 8 * (lane / 16)
template <int KS>
__device__ __forceinline__ void BlocksLoadRows(const uint16_t* p, u32x4_t (&f)[KS]) {
#pragma unroll
    for (int s = 0; s < KS; ++s) f[s] = *reinterpret_cast<const u32x4_t*>(p + s * 32);
}
// by columns, one row: N dwords at `p` (4-byte aligned)
template <int N>
__device__ __forceinline__ void BlocksLoadColumns(const uint16_t* p, uint32_t (&w)[N]) {
    struct __attribute__((packed, aligned(4))) Dwords {
        uint32_t x[N];
    };
    const Dwords t = *reinterpret_cast<const Dwords*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = t.x[i];
}
template <int N>
__device__ __forceinline__ void BlocksStoreColumns(uint16_t* p, const uint32_t (&w)[N]) {
    struct __attribute__((packed, aligned(4))) Dwords {
        uint32_t x[N];
    } t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.x[i] = w[i];
    *reinterpret_cast<Dwords*>(p) = t;
}

// operand for output slot dt from eight rows read by columns
template <int N>
__device__ __forceinline__ u32x4_t BlocksColumn(const uint32_t (&w)[8][N], int dt) {
    const int c = dt >> 1;
    const uint32_t sel = (dt & 1) ? 0x07060302u : 0x05040100u;
    return u32x4_t{__builtin_amdgcn_perm(w[1][c], w[0][c], sel), __builtin_amdgcn_perm(w[3][c], w[2][c], sel),
                   __builtin_amdgcn_perm(w[5][c], w[4][c], sel), __builtin_amdgcn_perm(w[7][c], w[6][c], sel)};
}

__device__ __forceinline__ float BlocksExp2(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, -inf -> 0
__device__ __forceinline__ float BlocksMaxOf4(const f32x4_t& x) { return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])); }
__device__ __forceinline__ float BlocksMaxOf4(const f32x4_t& x, float y) { return fmaxf(fmaxf(fmaxf(fmaxf(y, x[0]), x[1]), x[2]), x[3]); }
// over the four lanes that hold a C column: v_permlane32_swap / v_permlane16_swap of a register with itself put a lane's value and that of lane ^ 32 (^ 16)
// side by side, without the trip through LDS of a shuffle
__device__ __forceinline__ float BlocksMaxOver4(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto y = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1])));
    const auto z = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1]));
}
__device__ __forceinline__ float BlocksSumOver4(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto y = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(__uint_as_float(y[0]) + __uint_as_float(y[1]));
    const auto z = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __uint_as_float(z[0]) + __uint_as_float(z[1]);
}
// over 16 neighbouring lanes: ^ 1, ^ 2, mirror of 8, mirror of 16 lanes
template <int CTRL>
__device__ __forceinline__ float BlocksAddLane(float x) {
    return x + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float BlocksSumRow16(float x) { return BlocksAddLane<0x140>(BlocksAddLane<0x141>(BlocksAddLane<0x4E>(BlocksAddLane<0xB1>(x)))); }
// What logits are measured against follows their running maximum only when that is more than `kBlocksSlack` powers of two ahead, and then to `kBlocksLift` below
// it: weights reach 2^8 instead of 1 in bf16, which holds them as exactly, and the accumulators are hardly ever rescaled.  Binary16 holds up to 2^16, and in full
// only what is above 2^-14: weights between 2^7 and 2^15 for the largest keep those of 2^-21 of it whole.
template <bool BF16>
constexpr float kBlocksLift = BF16 ? 0.f : 7.f;
template <bool BF16>
constexpr float kBlocksSlack = 8.f + kBlocksLift<BF16>;
__device__ __forceinline__ int64_t BlocksReadLane64(int64_t x, uint32_t lane) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, (int)lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), (int)lane);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}
// LDS written by some lanes of a wavefront is read by others: no barrier needed, but the compiler must keep the order
__device__ __forceinline__ void BlocksWaveSync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// unit `u` of a query row's tiles: probed block u / tpb, tile u % tpb of it
struct BlocksCursor {
    uint32_t slot, sub, tpb;
    __device__ __forceinline__ BlocksCursor(uint32_t u, uint32_t tiles_per_block) : slot(u / tiles_per_block), sub(u % tiles_per_block), tpb(tiles_per_block) {}
    __device__ __forceinline__ void Next() {
        if (++sub == tpb) {
            sub = 0;
            ++slot;
        }
    }
};

// The probed blocks of one query row, one per lane: those that exist and hold a visible row, each once, moved to the front.  Returns their number.
// `scratch`: 64 words of LDS of this wavefront.
__device__ __forceinline__ uint32_t BlocksGatherProbes(const BlocksArgs& a, const int32_t* probes, uint32_t b, int visible, uint32_t* scratch, uint32_t lane,
                                                       int& block, int64_t& ko, int64_t& vo) {
    int p = lane < a.P ? probes[lane] : -1;
    bool ok = p >= 0 && (uint32_t)p < a.nblk && (int64_t)p * a.bs < visible;
    if (ok) ok = BlocksBase(a, b, p, ko, vo);
    for (uint32_t j = 0; j + 1 < a.P; ++j) {
        const int other = __builtin_amdgcn_readlane(p, (int)j);
        if (lane > j && other == p) ok = false;
    }
    const uint64_t mask = __ballot(ok);
    if (ok) scratch[__popcll(mask & ((1ull << lane) - 1))] = (uint32_t)p;
    BlocksWaveSync();
    const uint32_t count = (uint32_t)__popcll(mask);
    block = lane < count ? (int)scratch[lane] : 0;
    ko = vo = 0;
    if (lane < count) (void)BlocksBase(a, b, block, ko, vo);
    BlocksWaveSync();
    return count;
}

}  // namespace gpann

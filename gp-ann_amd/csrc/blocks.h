// blocks.h — shared parts of the block operators (include/gpann_blocks.h): argument block, layout checks, device helpers.
#pragma once

#include "common.h"

#include "../../include/gpann_blocks.h"

namespace gpann {

// Device view of a gpann_blocks_layout.
struct BlocksArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    int64_t qs[3], ks[3], vs[3], os[3];   // strides in elements: batch (k, v: batch or page), row, head
    const int32_t* q_len;
    const int32_t* kv_len;
    const int32_t* table;
    const int32_t* probes;
    uint32_t B, Tq, Tk, Hq, Hkv, G;       // G: query heads per key/value head
    uint32_t bs, nblk, P;                 // rows per block, blocks per sequence, probes per query row
    uint32_t table_stride, n_pages;
    uint32_t causal;
    float scale, scale2;                  // scale2 = scale * log2(e): the kernels' exponentials are powers of two
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

gpann_status BlocksCheckLayout(const gpann_blocks_layout* L);
gpann_status BlocksCheckStream(const gpann_blocks_layout* L, void* stream);
bool BlocksDisjoint(const int64_t stride[3], uint64_t n0, uint64_t n1, uint64_t n2, uint32_t d);
BlocksArgs BlocksMakeArgs(const gpann_blocks_layout* L, const void* q, const void* k, const void* v, const int32_t* probes, uint32_t nprobe);

inline uint32_t BlocksPerSequence(const gpann_blocks_layout* L) { return (uint32_t)(((uint64_t)L->kv_rows + L->block_rows - 1) / L->block_rows); }
inline size_t BlocksAlign(size_t n) { return (n + 255) & ~(size_t)255; }

// Makes `device` current for a call and gives the caller's back.
struct BlocksDevice {
    int before = -1;
    gpann_status Enter(int device) {
        if (hipGetDevice(&before) != hipSuccess) {
            (void)hipGetLastError();
            before = -1;
        }
        return EnsureDevice(device);
    }
    ~BlocksDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// (the layout has been checked)
#define GPANN_BLOCKS_ENTER(L, stream)                \
    ::gpann::BlocksDevice blocks_device;             \
    GPANN_TRY(blocks_device.Enter((L)->device));     \
    GPANN_TRY(::gpann::BlocksCheckStream(L, stream))

// ---- device helpers -----------------------------------------------------------------------------------------------------------------------
// (constant address space: nothing writes the lengths while a kernel runs, and a scalar load does not queue behind the vector loads in flight)
__device__ __forceinline__ int BlocksLength(const int32_t* p, uint32_t b) { return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p)[b]; }
__device__ __forceinline__ int BlocksKvLen(const BlocksArgs& a, uint32_t b) {
    return a.kv_len ? min(max(BlocksLength(a.kv_len, b), 0), (int)a.Tk) : (int)a.Tk;
}
__device__ __forceinline__ int BlocksQLen(const BlocksArgs& a, uint32_t b) {
    return a.q_len ? min(max(BlocksLength(a.q_len, b), 0), (int)a.Tq) : (int)a.Tq;
}
// how many cache rows (a prefix) query row t sees; n, m: lengths of the sequence
__device__ __forceinline__ int BlocksVisible(const BlocksArgs& a, int n, int m, int t) {
    if (t >= m) return 0;
    return a.causal ? min(max(n - m + t + 1, 0), n) : n;
}
// element offset of a block's first row and head 0; false: the page does not exist
__device__ __forceinline__ bool BlocksBase(const BlocksArgs& a, uint32_t b, int block, int64_t& ko, int64_t& vo) {
    if (a.table) {
        const int page = a.table[(int64_t)b * a.table_stride + block];
        if (page < 0 || (uint32_t)page >= a.n_pages) return false;
        ko = page * a.ks[0];
        vo = page * a.vs[0];
    } else {
        const int64_t row = (int64_t)block * a.bs;
        ko = b * a.ks[0] + row * a.ks[1];
        vo = b * a.vs[0] + row * a.vs[1];
    }
    return true;
}
__device__ __forceinline__ double BlocksToDouble(uint16_t x, bool bf16) {
    return bf16 ? (double)__uint_as_float((uint32_t)x << 16) : (double)__builtin_bit_cast(_Float16, x);
}
__device__ __forceinline__ float BlocksToFloat(uint16_t x, bool bf16) {
    return bf16 ? __uint_as_float((uint32_t)x << 16) : (float)__builtin_bit_cast(_Float16, x);
}

// Workgroup id -> (pair, tile) such that the workgroups of one (sequence, key/value head) pair get ids that are equal modulo 8: workgroups are dealt to
// the chip's eight dies round robin, so a pair's keys and values stay in one die's L2.  Pairs that are left over when every die has as many as the others go
// over all dies (12 pairs of 20 tiles: 40 workgroups on four dies of 32 CUs and 20 on the others, or 30 on each).  false: nothing to do.
__device__ __forceinline__ bool BlocksPairOf(uint32_t id, uint32_t pairs, uint32_t tiles, uint32_t& pair, uint32_t& tile) {
    const uint32_t lane = id & 7, rest = id >> 3, own = pairs / 8 * tiles;   // workgroups of pairs of its own that a die has
    const uint32_t x = rest < own ? rest : (rest - own) * 8 + lane;
    pair = rest < own ? x / tiles * 8 + lane : pairs / 8 * 8 + x / tiles;
    tile = x % tiles;
    return pair < pairs;
}
inline uint64_t BlocksPairGrid(uint64_t pairs, uint64_t tiles) { return 8 * (pairs / 8 * tiles + (pairs % 8 * tiles + 7) / 8); }
// bits[sequence, head][block][query row / 32] of the rows that probe a block; every word is written.  A workgroup has kMarkRows query rows and kMarkBlocks blocks
constexpr uint32_t kMarkRows = 128, kMarkBlocks = 512;
gpann_status BlocksCheckMarks(const gpann_blocks_layout* L);   // what its grid, and the others of (sequence, head) pairs, have room for
gpann_status BlocksMarkProbes(const BlocksArgs& a, uint32_t words, uint32_t* bits, hipStream_t st);
size_t BlocksBackwardSpace(const BlocksArgs& a, uint32_t d);

inline bool BlocksAligned(uintptr_t n, const void* p) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline gpann_status BlocksCheckWorkspace(const void* p, size_t have, size_t need) {
    if (need == 0) return GPANN_OK;
    if (have < need) {
        SetLastError("invalid argument: the workspace has %zu bytes, the call needs %zu", have, need);
        return GPANN_ERR_INVALID;
    }
    GPANN_REQUIRE(p && BlocksAligned(16, p), "the workspace is null or not 16-byte aligned");
    return GPANN_OK;
}

// workgroups of 512 threads
inline gpann_status BlocksCheckGrid(uint64_t grid) {
    if (grid > 0x7fffffffull / 512 * 2) {   // (a launch has fewer than 2^32 threads)
        SetLastError("the call needs %llu workgroups of 512 threads", (unsigned long long)grid);
        return GPANN_ERR_UNSUPPORTED;
    }
    return GPANN_OK;
}
template <typename K, typename... A>
inline gpann_status BlocksLaunch(K kernel, uint64_t grid, size_t lds, hipStream_t st, A... args) {
    GPANN_TRY(BlocksCheckGrid(grid));
    if (lds > 32 * 1024) GPANN_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(512), lds, st, args...);
    GPANN_HIP_TRY(hipGetLastError());
    return GPANN_OK;
}

// head_dim and element type -> template arguments
#define GPANN_BLOCKS_DISPATCH(L, fn, ...)                                                                                                   \
    do {                                                                                                                                    \
        const bool bf16 = (L)->dtype == GPANN_BLOCKS_BF16;                                                                                  \
        switch ((L)->head_dim) {                                                                                                            \
            case 64: return bf16 ? fn<true, 4>(__VA_ARGS__) : fn<false, 4>(__VA_ARGS__);                                                    \
            case 96: return bf16 ? fn<true, 6>(__VA_ARGS__) : fn<false, 6>(__VA_ARGS__);                                                    \
            case 128: return bf16 ? fn<true, 8>(__VA_ARGS__) : fn<false, 8>(__VA_ARGS__);                                                   \
            case 192: return bf16 ? fn<true, 12>(__VA_ARGS__) : fn<false, 12>(__VA_ARGS__);                                                 \
            default: return bf16 ? fn<true, 16>(__VA_ARGS__) : fn<false, 16>(__VA_ARGS__);                                                  \
        }                                                                                                                                   \
    } while (0)

}  // namespace gpann

// blocks.hip — block operators: layout checks, centroids of the blocks, routing of query rows to blocks, eviction (include/gpann_blocks.h).
#include "blocks_tile.h"

#include <algorithm>
#include <cmath>

namespace gpann {

// ---- checks ---------------------------------------------------------------------------------------------------------------------------------
// no two elements of an [n0][n1][n2][d] tensor share an address: ordered by stride, every dimension steps over the extent of those below it
bool BlocksDisjoint(const int64_t stride[3], uint64_t n0, uint64_t n1, uint64_t n2, uint32_t d) {
    std::pair<int64_t, uint64_t> dim[3] = {{stride[0], n0}, {stride[1], n1}, {stride[2], n2}};
    std::sort(dim, dim + 3);
    int64_t extent = d;
    for (const auto& [s, n] : dim) {
        if (n <= 1) continue;
        if (s < extent) return false;
        extent += s * (int64_t)(n - 1);
    }
    return true;
}

gpann_status BlocksCheckLayout(const gpann_blocks_layout* L) {
    GPANN_REQUIRE(L != nullptr, "layout is null");
    GPANN_REQUIRE(L->struct_bytes == sizeof(gpann_blocks_layout), "layout.struct_bytes is not sizeof(gpann_blocks_layout) of this library");
    GPANN_REQUIRE(L->dtype == GPANN_BLOCKS_BF16 || L->dtype == GPANN_BLOCKS_FP16, "layout.dtype must be GPANN_BLOCKS_BF16 or GPANN_BLOCKS_FP16");
    GPANN_REQUIRE((L->flags & ~(uint32_t)GPANN_BLOCKS_CAUSAL) == 0, "unknown bits in layout.flags");
    GPANN_REQUIRE(L->batch <= 65535 && L->q_rows <= (1u << 24) && L->kv_rows <= (1u << 24), "batch above 65535 or more than 2^24 rows");
    GPANN_REQUIRE(L->kv_heads > 0 && L->q_heads > 0 && L->q_heads % L->kv_heads == 0, "q_heads must be a positive multiple of kv_heads");
    GPANN_REQUIRE(L->q_heads <= 1024, "more than 1024 query heads");
    const uint32_t d = L->head_dim;
    GPANN_REQUIRE(d == 64 || d == 96 || d == 128 || d == 192 || d == 256, "head_dim must be 64, 96, 128, 192 or 256");
    GPANN_REQUIRE(L->block_rows >= 16 && L->block_rows <= 256 && L->block_rows % 16 == 0, "block_rows must be a multiple of 16 from 16 to 256");
    GPANN_REQUIRE(BlocksPerSequence(L) <= GPANN_BLOCKS_MAX_BLOCKS, "more than GPANN_BLOCKS_MAX_BLOCKS blocks per sequence");
    GPANN_REQUIRE(std::isfinite(L->scale * kLog2e), "layout.scale (times log2 e) is not finite");
    const int64_t* strides[4] = {L->q_stride, L->k_stride, L->v_stride, L->out_stride};
    for (const int64_t* s : strides)
        for (int i = 0; i < 3; ++i) {
            GPANN_REQUIRE(s[i] >= 0 && s[i] % 8 == 0, "strides must be non-negative multiples of 8 elements");
            GPANN_REQUIRE(s[i] <= (i == 0 ? (int64_t)1 << 40 : i == 1 ? (int64_t)1 << 22 : (int64_t)1 << 31),
                          "a stride above 2^40 (batch or page), 2^22 (row) or 2^31 (head) elements");
        }
    GPANN_REQUIRE(BlocksAligned(4, L->q_len) && BlocksAligned(4, L->kv_len) && BlocksAligned(4, L->page_table), "lengths and page table must be 4-byte aligned");
    if (L->page_table) {
        GPANN_REQUIRE(L->page_stride >= BlocksPerSequence(L), "layout.page_stride is smaller than a sequence's blocks");
        GPANN_REQUIRE(L->n_pages <= 0x7fffffffu, "more than 2^31 - 1 pages");
    }
    return GPANN_OK;
}

gpann_status BlocksCheckMarks(const gpann_blocks_layout* L) {
    GPANN_REQUIRE((uint64_t)L->batch * L->kv_heads <= 65535, "more than 65535 (sequence, head) pairs");
    GPANN_REQUIRE(L->q_rows <= 65535 * kMarkRows, "more than 65535 * 128 query rows");
    return GPANN_OK;
}

// a stream of another device would run the kernels where the tensors are not
gpann_status BlocksCheckStream(const gpann_blocks_layout* L, void* stream) {
    if (!stream) return GPANN_OK;
    hipDevice_t dev = -1;
    GPANN_HIP_TRY(hipStreamGetDevice(static_cast<hipStream_t>(stream), &dev));
    GPANN_REQUIRE((int)dev == L->device, "the stream belongs to another device than the layout");
    return GPANN_OK;
}

BlocksArgs BlocksMakeArgs(const gpann_blocks_layout* L, const void* q, const void* k, const void* v, const int32_t* probes, uint32_t nprobe) {
    BlocksArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = L->q_stride[i];
        a.ks[i] = L->k_stride[i];
        a.vs[i] = L->v_stride[i];
        a.os[i] = L->out_stride[i];
    }
    a.q_len = L->q_len;
    a.kv_len = L->kv_len;
    a.table = L->page_table;
    a.probes = probes;
    a.B = L->batch;
    a.Tq = L->q_rows;
    a.Tk = L->kv_rows;
    a.Hq = L->q_heads;
    a.Hkv = L->kv_heads;
    a.G = L->q_heads / L->kv_heads;
    a.bs = L->block_rows;
    a.nblk = BlocksPerSequence(L);
    a.P = nprobe;
    a.table_stride = L->page_stride;
    a.n_pages = L->n_pages;
    a.causal = (L->flags & GPANN_BLOCKS_CAUSAL) ? 1 : 0;
    a.scale = L->scale;
    a.scale2 = L->scale * kLog2e;
    return a;
}

// ---- centroids ------------------------------------------------------------------------------------------------------------------------------
// One workgroup per (block, head, sequence).  A thread adds eight dimensions of every (256 * 8 / d)-th row in binary64 — sums of 16-bit floats, exact but
// for exponents that lie more than 2^40 apart — and the row groups are added in LDS, always in the same order.  Bound by reading K once: 8192 rows x 8
// heads of 128 dimensions (17 MB) 6.9 us; the last blocks of 64 sequences 5.6 us, a launch's time.
template <bool BF16>
__global__ void __launch_bounds__(256) BlocksSummarizeKernel(BlocksArgs a, uint32_t d, uint32_t new_rows, float* __restrict__ summary) {
    extern __shared__ double s_sum[];   // [row group][d]
    const uint32_t b = blockIdx.z, h = blockIdx.y;
    const int n = BlocksKvLen(a, b);
    if (n == 0) return;
    const int first = new_rows == 0 ? 0 : max(0, n - (int)min(new_rows, (uint32_t)n)) / (int)a.bs;
    const int block = first + (int)blockIdx.x, row0 = block * (int)a.bs;
    if (row0 >= n) return;
    int64_t ko, vo;
    const bool there = BlocksBase(a, b, block, ko, vo);
    const int rows = there ? min((int)a.bs, n - row0) : 0;
    const uint32_t chunks = d / 8, groups = 256 / chunks, chunk = threadIdx.x % chunks, group = threadIdx.x / chunks;
    if (group < groups) {
        double acc[8] = {};
        const uint16_t* p = a.k + ko + h * a.ks[2] + chunk * 8;
        for (int r = (int)group; r < rows; r += (int)groups) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + r * a.ks[1]);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[2 * i] += BlocksToDouble((uint16_t)w[i], BF16);
                acc[2 * i + 1] += BlocksToDouble((uint16_t)(w[i] >> 16), BF16);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s_sum[group * d + chunk * 8 + i] = acc[i];
    }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < d; c += 256) {
        double t = 0;
        for (uint32_t g = 0; g < groups; ++g) t += s_sum[g * d + c];
        summary[(((int64_t)b * a.Hkv + h) * a.nblk + block) * d + c] = rows > 0 ? (float)(t / rows) : 0.f;
    }
}

// ---- routing --------------------------------------------------------------------------------------------------------------------------------
// binary64 -> unsigned whose order is the numbers' order; NaN is the smallest, both zeros are equal
__device__ __forceinline__ uint64_t BlocksScoreKey(double x) {
    if (x != x) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// The nprobe best of a query row's `nb` blocks, by one wavefront (REGS keys a lane, or from LDS): bisection over the upper 32 key bits — 32-bit comparisons,
// counts on the scalar unit — until a threshold parts exactly P blocks from the rest; blocks that agree in those bits are told apart by the lower 32; of equal
// keys the lowest blocks stay.  Probes come out in block order.
template <int REGS>
__device__ __forceinline__ void BlocksSelect(const uint64_t* s_key, uint32_t nb, uint32_t P, uint32_t first, uint32_t last, uint32_t lane, int32_t* out) {
    constexpr int N = REGS > 0 ? REGS : 1;
    uint32_t hi[N], lo[N];
    auto key = [&](uint32_t j) -> uint64_t { return j >= nb ? 0 : (j < first || j + last >= nb) ? ~0ull : s_key[j]; };
    if (REGS > 0)
#pragma unroll
        for (int i = 0; i < REGS; ++i) {
            const uint64_t k = key(i * 64 + lane);
            hi[i] = (uint32_t)(k >> 32);
            lo[i] = (uint32_t)k;
        }
    const uint32_t rounds = REGS > 0 ? REGS : (nb + 63) / 64;
    auto each = [&](auto&& f) {   // f(round, block, hi, lo) for all of a lane's keys
        if (REGS > 0) {
#pragma unroll
            for (int i = 0; i < REGS; ++i) f(i, i * 64 + lane, hi[i], lo[i]);
        } else {
            for (uint32_t i = 0; i < rounds; ++i) {
                const uint64_t k = key(i * 64 + lane);
                f(i, i * 64 + lane, (uint32_t)(k >> 32), (uint32_t)k);
            }
        }
    };
    uint32_t v = 0, w = 0;
    bool exact = false;
    for (uint32_t bit = 1u << 31; bit && !exact; bit >>= 1) {
        const uint32_t trial = v | bit;
        uint32_t c = 0;
        each([&](int, uint32_t, uint32_t x, uint32_t) { c += (uint32_t)__popcll(__ballot(x >= trial)); });
        if (c >= P) v = trial;
        exact = c == P;
    }
    if (!exact) {   // (v = 0: all keys reach it)
        for (uint32_t bit = 1u << 31; bit && !exact; bit >>= 1) {
            const uint32_t trial = w | bit;
            uint32_t c = 0;
            each([&](int, uint32_t j, uint32_t x, uint32_t y) { c += (uint32_t)__popcll(__ballot(j < nb && (x > v || (x == v && y >= trial)))); });
            if (c >= P) w = trial;
            exact = c == P;
        }
    }
    const uint64_t below = (1ull << lane) - 1;
    uint32_t at = 0, equal = 0;
    if (!exact) {   // more than P reach the threshold: the lowest of those that equal it fill up
        uint32_t above = 0;
        each([&](int, uint32_t, uint32_t x, uint32_t y) { above += (uint32_t)__popcll(__ballot(x > v || (x == v && y > w))); });
        equal = P - above;
    }
    each([&](int, uint32_t j, uint32_t x, uint32_t y) {
        bool take = j < nb && (x > v || (x == v && y >= w));
        if (!exact) {
            const bool eq = j < nb && x == v && y == w;
            const uint64_t eqs = __ballot(eq);
            if (eq) take = (uint32_t)__popcll(eqs & below) < equal;
            equal -= min(equal, (uint32_t)__popcll(eqs));
        }
        const uint64_t taken = __ballot(take);
        if (take) out[at + (uint32_t)__popcll(taken & below)] = (int32_t)j;
        at += (uint32_t)__popcll(taken);
    });
}

// Scores in binary64, because a selection has to come out the same whatever the order of a sum: neighbouring scores differ by far more than 2^-50.  The
// products run on the binary64 matrix instruction (16 x 16 x 4, the vector unit's rate without its operand traffic; C: column l % 16, rows 4 i + l / 16): a
// wavefront holds the sums of `tokens` <= 16 query rows (lane: row l % 16, every fourth four dimensions) and takes 16 blocks' centroids at a time straight from
// memory; keys wait in LDS until the wavefronts turn to selecting, a query row each.  A workgroup has `groups` sets of query rows, whose blocks 8 / groups
// wavefronts divide.  8192 query rows x 8 heads of 128 dimensions over up to 128 blocks: 99 us, of which the selection is 49 (rounds of dependent comparisons and
// scalar counts, two wavefronts a SIMD), the products 28, and reading query rows (67 MB) and centroids 18.
template <bool BF16, int DC>
__global__ void __launch_bounds__(512) BlocksRouteKernel(BlocksArgs a, uint32_t groups, uint32_t tokens, uint32_t tiles, const float* __restrict__ summary,
                                                         uint32_t first, uint32_t last, int32_t* __restrict__ probes) {
    TakeWholeRegisterFile();
    constexpr int D = DC * 16, K = D / 4;
    typedef double f64x4_t __attribute__((ext_vector_type(4)));
    extern __shared__ uint64_t s_key[];   // [query row of the workgroup][block]
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    uint32_t pair, tile;
    if (!BlocksPairOf(blockIdx.x, a.B * a.Hkv, tiles, pair, tile)) return;
    const uint32_t b = pair / a.Hkv, h = pair % a.Hkv, parts = 8 / groups, group = wave / parts, part = wave % parts;
    const int n = BlocksKvLen(a, b), m = BlocksQLen(a, b);
    const uint32_t row0 = (tiles - 1 - tile) * groups * tokens, t0 = row0 + group * tokens;
    const uint32_t live = (int)t0 < m ? min(tokens, (uint32_t)m - t0) : 0;
    const uint32_t blocks = live ? (uint32_t)(BlocksVisible(a, n, m, (int)(t0 + live - 1)) + (int)a.bs - 1) / a.bs : 0;
    const float* cen = summary + (uint64_t)pair * a.nblk * D + g * 4;   // this lane's dimensions: 16 i + 4 g ..
    if (part * 16 < blocks && blocks > a.P) {
        double q[K];
#pragma unroll
        for (int i = 0; i < K; ++i) q[i] = 0;
        if (r < live) {
            const uint16_t* p = a.q + b * a.qs[0] + (int64_t)(t0 + r) * a.qs[1] + (int64_t)h * a.G * a.qs[2] + g * 4;
            uint2 y[K / 4];
#pragma unroll
            for (int i = 0; i < K / 4; ++i) y[i] = *reinterpret_cast<const uint2*>(p + i * 16);
            for (uint32_t x = 1;; ++x) {   // the next head's numbers are on their way while one's are added
                uint2 z[K / 4];
                const uint16_t* after = p + min(x, a.G - 1) * a.qs[2];
#pragma unroll
                for (int i = 0; i < K / 4; ++i) z[i] = *reinterpret_cast<const uint2*>(after + i * 16);
#pragma unroll
                for (int i = 0; i < K / 4; ++i) {
                    q[4 * i] += BlocksToDouble((uint16_t)y[i].x, BF16);
                    q[4 * i + 1] += BlocksToDouble((uint16_t)(y[i].x >> 16), BF16);
                    q[4 * i + 2] += BlocksToDouble((uint16_t)y[i].y, BF16);
                    q[4 * i + 3] += BlocksToDouble((uint16_t)(y[i].y >> 16), BF16);
                    y[i] = z[i];
                }
                if (x >= a.G) break;
            }
        }
        float4 c[K / 4], next[K / 4];
        auto load = [&](uint32_t j0, float4(&to)[K / 4]) {
            const float* p = cen + (uint64_t)min(j0 + r, blocks - 1) * D;
#pragma unroll
            for (int i = 0; i < K / 4; ++i) to[i] = *reinterpret_cast<const float4*>(p + i * 16);
        };
        load(part * 16, c);
        for (uint32_t j0 = part * 16; j0 < blocks; j0 += parts * 16) {
            load(j0 + parts * 16, next);   // (of no use behind the last blocks; a load under a branch would be waited for at once)
            f64x4_t x = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < K / 4; ++i) {
                x = __builtin_amdgcn_mfma_f64_16x16x4f64(q[4 * i], (double)c[i].x, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f64_16x16x4f64(q[4 * i + 1], (double)c[i].y, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f64_16x16x4f64(q[4 * i + 2], (double)c[i].z, x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f64_16x16x4f64(q[4 * i + 3], (double)c[i].w, x, 0, 0, 0);
            }
            if (j0 + r < blocks)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (i * 4 + g < live) s_key[(uint64_t)(group * tokens + i * 4 + g) * a.nblk + j0 + r] = BlocksScoreKey(x[i]);
#pragma unroll
            for (int i = 0; i < K / 4; ++i) c[i] = next[i];
        }
    }
    // a wavefront that has all the blocks of its query rows to itself goes on with them; else the workgroup's query rows are divided
    const bool own = parts == 1;
    if (own)
        BlocksWaveSync();
    else
        __syncthreads();
    for (uint32_t i = own ? group * tokens : wave, end = own ? i + tokens : groups * tokens; i < end; i += own ? 1 : 8) {
        const uint32_t t = row0 + i;
        if ((int)t >= m) break;
        const uint32_t nb = (uint32_t)(BlocksVisible(a, n, m, (int)t) + (int)a.bs - 1) / a.bs;
        int32_t* out = probes + (((int64_t)b * a.Tq + t) * a.Hkv + h) * a.P;
        if (nb <= a.P) {
            if (lane < a.P) out[lane] = lane < nb ? (int32_t)lane : -1;
        } else if (nb <= 128) {
            BlocksSelect<2>(s_key + (uint64_t)i * a.nblk, nb, a.P, first, last, lane, out);
        } else if (nb <= 512) {
            BlocksSelect<8>(s_key + (uint64_t)i * a.nblk, nb, a.P, first, last, lane, out);
        } else {
            BlocksSelect<0>(s_key + (uint64_t)i * a.nblk, nb, a.P, first, last, lane, out);
        }
    }
}

// lane ^ 1, ^ 2, and the mirrors of 8 and 16 lanes: a sum over 16 lanes on the vector unit
template <int CTRL>
__device__ __forceinline__ double BlocksAddLane(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return x + __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double BlocksSumOver16(double x) {
    x = BlocksAddLane<0xB1>(x);    // quad_perm 1 0 3 2
    x = BlocksAddLane<0x4E>(x);    // quad_perm 2 3 0 1
    x = BlocksAddLane<0x141>(x);   // row_half_mirror
    return BlocksAddLane<0x140>(x);   // row_mirror
}

// One query row per (sequence, head): a workgroup reads all its blocks' centroids once — bound by that read, so by what is in flight: 64 groups of 16 lanes,
// four blocks each — and one wavefront selects.  64 sequences of up to 512 blocks, 8 heads of 128 dimensions (110 MB of centroids): 24.5 us, 4.5 TB/s.
template <bool BF16, int DC>
__global__ void __launch_bounds__(1024) BlocksRouteRowKernel(BlocksArgs a, const float* __restrict__ summary, uint32_t first, uint32_t last,
                                                             int32_t* __restrict__ probes) {
    constexpr uint32_t D = DC * 16, N = (D + 63) / 64;   // float4 a lane of a 16-lane group: dimensions 64 i + 4 l
    extern __shared__ uint64_t s_key[];
    const uint32_t t = blockIdx.x, pair = blockIdx.y, b = pair / a.Hkv, h = pair % a.Hkv, sub = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int n = BlocksKvLen(a, b), m = BlocksQLen(a, b);
    if ((int)t >= m) return;
    const uint32_t nb = (uint32_t)(BlocksVisible(a, n, m, (int)t) + (int)a.bs - 1) / a.bs;
    int32_t* out = probes + (((int64_t)b * a.Tq + t) * a.Hkv + h) * a.P;
    if (nb <= a.P) {
        if (threadIdx.x < a.P) out[threadIdx.x] = threadIdx.x < nb ? (int32_t)threadIdx.x : -1;
        return;
    }
    const float* cen = summary + (uint64_t)pair * a.nblk * D;
    const uint16_t* p = a.q + b * a.qs[0] + (int64_t)t * a.qs[1] + (int64_t)h * a.G * a.qs[2];
    double q[N][4];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) q[i][0] = q[i][1] = q[i][2] = q[i][3] = 0;
    for (uint32_t j0 = 0; j0 < nb; j0 += 256) {
        float4 c[4][N];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
            for (uint32_t i = 0; i < N; ++i)
                c[u][i] = *reinterpret_cast<const float4*>(cen + (uint64_t)min(j0 + u * 64 + group, nb - 1) * D + min(i * 64 + sub * 4, D - 4));
        if (j0 == 0)
            for (uint32_t x = 0; x < a.G; ++x)
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) {
                    if (i * 64 + sub * 4 >= D) continue;
                    const uint2 y = *reinterpret_cast<const uint2*>(p + x * a.qs[2] + i * 64 + sub * 4);
                    q[i][0] += BlocksToDouble((uint16_t)y.x, BF16);
                    q[i][1] += BlocksToDouble((uint16_t)(y.x >> 16), BF16);
                    q[i][2] += BlocksToDouble((uint16_t)y.y, BF16);
                    q[i][3] += BlocksToDouble((uint16_t)(y.y >> 16), BF16);
                }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            double x = 0;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i)
                if (i * 64 + sub * 4 < D) {
                    x = fma(q[i][0], (double)c[u][i].x, x);
                    x = fma(q[i][1], (double)c[u][i].y, x);
                    x = fma(q[i][2], (double)c[u][i].z, x);
                    x = fma(q[i][3], (double)c[u][i].w, x);
                }
            x = BlocksSumOver16(x);
            const uint32_t j = j0 + u * 64 + group;
            if (sub == 0 && j < nb) s_key[j] = BlocksScoreKey(x);
        }
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    if (nb <= 128)
        BlocksSelect<2>(s_key, nb, a.P, first, last, threadIdx.x, out);
    else if (nb <= 512)
        BlocksSelect<8>(s_key, nb, a.P, first, last, threadIdx.x, out);
    else
        BlocksSelect<0>(s_key, nb, a.P, first, last, threadIdx.x, out);
}

// A workgroup per query row and head, or matrix tiles of up to 16 query rows (512 blocks of 128 dimensions: 8 rows of 64 heads 32 us by row, 26 by tiles, 4 rows
// 22 and 24; 2 rows of 512 heads 30 and 46, 4 rows 48 and 51).  Tiles hold a workgroup's keys in 128 KB: with more blocks they would have fewer than four rows.
static bool BlocksRouteByRow(uint64_t pairs, uint32_t rows, uint32_t blocks) { return rows < 4 || pairs * rows <= 256 || blocks > 128 * 1024 / 8 / 4; }
template <bool BF16, int DC>
static gpann_status Route(const BlocksArgs& a, const float* summary, uint32_t first, uint32_t last, int32_t* probes, hipStream_t st) {
    // keys of a workgroup's query rows in 128 KB; groups are given up while there are not two workgroups per CU
    const uint64_t pairs = (uint64_t)a.B * a.Hkv, room = 128 * 1024 / 8;
    if (BlocksRouteByRow(pairs, a.Tq, a.nblk)) {
        const size_t lds = (size_t)a.nblk * 8;
        auto kernel = BlocksRouteRowKernel<BF16, DC>;
        if (lds > 32 * 1024) GPANN_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kernel, dim3(a.Tq, (uint32_t)pairs), dim3(1024), lds, st, a, summary, first, last, probes);
        GPANN_HIP_TRY(hipGetLastError());
        return GPANN_OK;
    }
    const uint32_t tokens = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(16, a.Tq), std::max<uint64_t>(1, room / std::max(1u, a.nblk)));
    uint32_t groups = 8;
    while (groups > 1 && ((uint64_t)groups * tokens * a.nblk > room || pairs * ((a.Tq + groups * tokens - 1) / (groups * tokens)) < 512)) groups /= 2;
    const uint64_t tiles = ((uint64_t)a.Tq + groups * tokens - 1) / (groups * tokens);
    const size_t lds = std::max<size_t>(8, (size_t)groups * tokens * a.nblk * 8);
    return BlocksLaunch(BlocksRouteKernel<BF16, DC>, BlocksPairGrid(pairs, tiles), lds, st, a, groups, tokens, (uint32_t)tiles, summary, first, last, probes);
}

// ---- eviction -------------------------------------------------------------------------------------------------------------------------------
// binary32 -> unsigned whose order is the numbers' order; NaN is the smallest, both zeros are equal
__device__ __forceinline__ uint32_t BlocksMassKey(float x) {
    if (x != x) return 0;
    return OrderedKey(x + 0.f);
}

constexpr uint32_t kEvictKeys = 32768;   // keys that fit LDS: sequences up to that length are read once
// One workgroup per (head, sequence).  The smallest key that stays is found eleven, eleven and ten bits at a time: a histogram of the keys that agree with the
// bits found so far, summed from its top.  Then one pass in row order: keys above it stay, and of those equal to it the lowest rows.  8 sequences x 8 heads x
// 32768 rows: 57 us, bound by the six passes' instructions on the 64 CUs that have a head.  (Bins over the span of the keys, equal keys counted at once: 64 us.)
template <bool HELD>
__global__ void __launch_bounds__(1024) BlocksEvictSelectKernel(BlocksArgs a, const float* __restrict__ mass, uint32_t keep, uint32_t first, uint32_t last,
                                                                int32_t* __restrict__ rows, int32_t* __restrict__ count) {
    __shared__ uint32_t s_bins[2048], s_gt[16], s_eq[16], s_found[2];
    const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const uint32_t n = (uint32_t)BlocksKvLen(a, b);
    const uint32_t take = min(n, keep);
    const int64_t pair = (int64_t)b * a.Hkv + h;
    const float* ms = mass + pair * a.Tk;
    int32_t* out = rows + pair * keep;
    if (tid == 0) count[pair] = (int32_t)take;
    if (n <= keep) {
        for (uint32_t j = tid; j < n; j += 1024) out[j] = (int32_t)j;
        return;
    }
    // rows first .. n - last compete for what the others leave
    const uint32_t lo_row = first, hi_row = n - last, want = take - first - last;
    // a wavefront has the rows chunk * wave .., 64 at a time: what it keeps lies together in the output
    const uint32_t chunk = (n + 1023) / 1024 * 64, row0 = wave * chunk;
    extern __shared__ uint32_t s_keys[];
    if (HELD)
#pragma unroll 4
        for (uint32_t i = 0; i < chunk; i += 64) {
            const uint32_t j = row0 + i + lane;
            if (j < n) s_keys[j] = BlocksMassKey(ms[j]);
        }
    auto each = [&](auto&& f) {   // f(row, key) of the wavefront's rows, in their order
#pragma unroll 4
        for (uint32_t i = 0; i < chunk; i += 64) {
            const uint32_t j = row0 + i + lane, at = min(j, n - 1);
            f(j, HELD ? s_keys[at] : BlocksMassKey(ms[at]));
        }
    };
    uint32_t v = 0, left = want;   // key bits found; how many of the keys that agree with them stay
    if (want > 0)
        for (int digit = 0; digit < 3; ++digit) {
            const uint32_t shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bins = digit == 2 ? 1024 : 2048;
            const uint32_t above = digit == 0 ? 0 : digit == 1 ? 0xFFE00000u : 0xFFFFFC00u;
            for (uint32_t i = tid; i < bins; i += 1024) s_bins[i] = 0;
            __syncthreads();
            each([&](uint32_t j, uint32_t k) {
                if (j >= lo_row && j < hi_row && (k & above) == v) atomicAdd(&s_bins[(k >> shift) & (bins - 1)], 1u);
            });
            __syncthreads();
            // thread t: bins top - 2 t and top - 2 t - 1 (or one each); sums from the top
            const uint32_t per = bins / 1024, bin = bins - 1 - tid * per;
            const uint32_t c0 = s_bins[bin], c1 = per == 2 ? s_bins[bin - 1] : 0;
            uint32_t sum = c0 + c1;
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t x = __shfl_up(sum, s);
                if ((int)lane >= s) sum += x;
            }
            if (lane == 63) s_gt[wave] = sum;
            __syncthreads();
            uint32_t before = sum - c0 - c1;
            for (uint32_t w = 0; w < wave; ++w) before += s_gt[w];
            if (before < left && before + c0 + c1 >= left) {
                const bool upper = before + c0 >= left;
                s_found[0] = upper ? bin : bin - 1;
                s_found[1] = upper ? before : before + c0;
            }
            __syncthreads();
            v |= s_found[0] << shift;
            left -= s_found[1];
            __syncthreads();
        }
    // `left` of the rows whose key is v stay: how many of either kind the wavefronts before this one have, then where each row goes
    const uint64_t below = (1ull << lane) - 1;
    auto kind = [&](uint32_t j, uint32_t k, bool& gt, bool& eq) {
        const bool free = j >= lo_row && j < hi_row && want > 0;
        gt = (j < n && !(j >= lo_row && j < hi_row)) || (free && k > v);
        eq = free && k == v;
    };
    uint32_t gts = 0, eqs = 0;
    each([&](uint32_t j, uint32_t k) {
        bool gt, eq;
        kind(j, k, gt, eq);
        gts += (uint32_t)__popcll(__ballot(gt));
        eqs += (uint32_t)__popcll(__ballot(eq));
    });
    if (lane == 0) {
        s_gt[wave] = gts;
        s_eq[wave] = eqs;
    }
    __syncthreads();
    uint32_t gt_at = 0, eq_at = 0;
    for (uint32_t w = 0; w < wave; ++w) {
        gt_at += s_gt[w];
        eq_at += s_eq[w];
    }
    each([&](uint32_t j, uint32_t k) {
        bool gt, eq;
        kind(j, k, gt, eq);
        const uint64_t g = __ballot(gt), e = __ballot(eq);
        const uint32_t before = gt_at + (uint32_t)__popcll(g & below), same = eq_at + (uint32_t)__popcll(e & below);
        if (gt || (eq && same < left)) out[before + min(same, left)] = (int32_t)j;
        gt_at += (uint32_t)__popcll(g);
        eq_at += (uint32_t)__popcll(e);
    });
}

// 16 bytes of a kept row per thread: a copy, at a copy's rate (8 x 8192 rows x 8 heads of 128 dimensions, 537 MB moved: 93 us, 5.8 TB/s)
__global__ void __launch_bounds__(256) BlocksEvictCopyKernel(BlocksArgs a, uint32_t chunks, uint32_t keep, uint32_t kept, const int32_t* __restrict__ rows,
                                                             const int32_t* __restrict__ count, const float* __restrict__ mass, uint16_t* __restrict__ k_out,
                                                             uint16_t* __restrict__ v_out, int64_t os0, int64_t os1, int64_t os2, float* __restrict__ mass_out) {
    const uint32_t b = blockIdx.y;
    const uint64_t all = (uint64_t)kept * a.Hkv * chunks;   // (slots that a sequence of this layout can fill: keep may be far more)
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
        const uint32_t c = (uint32_t)(i % chunks), h = (uint32_t)(i / chunks % a.Hkv), r = (uint32_t)(i / chunks / a.Hkv);
        const int64_t pair = (int64_t)b * a.Hkv + h;
        if ((int)r >= count[pair]) continue;
        const int row = rows[pair * keep + r];
        if (c == 0 && mass_out) mass_out[pair * keep + r] = mass[pair * a.Tk + row];
        if (!k_out) continue;
        int64_t ko, vo;
        const int block = row / (int)a.bs, in = row % (int)a.bs;
        uint4 x{}, y{};
        if (BlocksBase(a, b, block, ko, vo)) {
            x = *reinterpret_cast<const uint4*>(a.k + ko + in * a.ks[1] + h * a.ks[2] + c * 8);
            y = *reinterpret_cast<const uint4*>(a.v + vo + in * a.vs[1] + h * a.vs[2] + c * 8);
        }
        const int64_t o = b * os0 + r * os1 + h * os2 + c * 8;
        *reinterpret_cast<uint4*>(k_out + o) = x;
        *reinterpret_cast<uint4*>(v_out + o) = y;
    }
}

}  // namespace gpann

using namespace gpann;

extern "C" {

gpann_status gpann_blocks_summarize(const gpann_blocks_layout* L, const void* k, uint32_t new_rows, float* summary, void* stream) {
    GPANN_TRY(BlocksCheckLayout(L));
    GPANN_REQUIRE(k && summary, "a tensor is null");
    GPANN_REQUIRE(BlocksAligned(16, k) && BlocksAligned(16, summary), "tensors must be 16-byte aligned");
    GPANN_BLOCKS_ENTER(L, stream);
    const BlocksArgs a = BlocksMakeArgs(L, nullptr, k, nullptr, nullptr, 0);
    if (a.B == 0 || a.nblk == 0) return GPANN_OK;
    // the last new_rows rows start anywhere in a block
    const uint32_t touched = new_rows == 0 ? a.nblk : std::min<uint32_t>(a.nblk, (uint32_t)(((uint64_t)new_rows + a.bs - 2) / a.bs + 1));
    const uint32_t d = L->head_dim, groups = 256 / (d / 8);
    const dim3 grid(touched, a.Hkv, a.B);
    const size_t lds = (size_t)groups * d * sizeof(double);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (L->dtype == GPANN_BLOCKS_BF16)
        hipLaunchKernelGGL(BlocksSummarizeKernel<true>, grid, dim3(256), lds, st, a, d, new_rows, summary);
    else
        hipLaunchKernelGGL(BlocksSummarizeKernel<false>, grid, dim3(256), lds, st, a, d, new_rows, summary);
    GPANN_HIP_TRY(hipGetLastError());
    return GPANN_OK;
}

gpann_status gpann_blocks_route(const gpann_blocks_layout* L, const void* q, const float* summary, uint32_t nprobe, uint32_t first, uint32_t last,
                                int32_t* probes, void* workspace, size_t workspace_bytes, void* stream) {
    (void)workspace;
    (void)workspace_bytes;
    GPANN_TRY(BlocksCheckLayout(L));
    GPANN_REQUIRE(q && summary && probes, "a tensor is null");
    GPANN_REQUIRE(BlocksAligned(16, q) && BlocksAligned(16, summary) && BlocksAligned(4, probes), "q and summary must be 16-byte aligned, probes 4-byte aligned");
    GPANN_REQUIRE(nprobe >= 1 && nprobe <= GPANN_BLOCKS_MAX_PROBE, "nprobe must be 1 .. GPANN_BLOCKS_MAX_PROBE");
    GPANN_REQUIRE(first <= nprobe && last <= nprobe - first, "first + last must not exceed nprobe");
    GPANN_REQUIRE(last >= 1 || !(L->flags & GPANN_BLOCKS_CAUSAL), "a causal route needs last >= 1");
    if (BlocksRouteByRow((uint64_t)L->batch * L->kv_heads, L->q_rows, BlocksPerSequence(L))) {
        GPANN_REQUIRE((uint64_t)L->batch * L->kv_heads <= 65535, "more than 65535 (sequence, head) pairs");
        GPANN_REQUIRE(L->q_rows < 1u << 22, "2^22 query rows or more over more than 4096 blocks");
    }
    GPANN_BLOCKS_ENTER(L, stream);
    const BlocksArgs a = BlocksMakeArgs(L, q, nullptr, nullptr, nullptr, nprobe);
    if (a.B == 0 || a.Tq == 0) return GPANN_OK;
    GPANN_BLOCKS_DISPATCH(L, Route, a, summary, first, last, probes, static_cast<hipStream_t>(stream));
}

gpann_status gpann_blocks_evict(const gpann_blocks_layout* L, const void* k, const void* v, const float* mass, uint32_t keep, uint32_t first, uint32_t last,
                                int32_t* rows, int32_t* count, void* k_out, void* v_out, const int64_t out_kv_stride[3], float* mass_out, void* workspace,
                                size_t workspace_bytes, void* stream) {
    (void)workspace;
    (void)workspace_bytes;
    GPANN_TRY(BlocksCheckLayout(L));
    GPANN_REQUIRE(mass && rows && count, "a tensor is null");
    GPANN_REQUIRE((k_out == nullptr) == (v_out == nullptr), "k_out and v_out must be given together");
    GPANN_REQUIRE(k_out == nullptr || (k && v && out_kv_stride), "a tensor is null");
    GPANN_REQUIRE(BlocksAligned(16, k) && BlocksAligned(16, v) && BlocksAligned(16, k_out) && BlocksAligned(16, v_out), "k, v, k_out and v_out must be 16-byte aligned");
    GPANN_REQUIRE(BlocksAligned(4, mass) && BlocksAligned(4, rows) && BlocksAligned(4, count) && BlocksAligned(4, mass_out), "tensors must be 4-byte aligned");
    GPANN_REQUIRE(keep >= 1 && keep <= (1u << 24), "keep must be 1 .. 2^24");
    GPANN_REQUIRE(first <= keep && last <= keep - first, "first + last must not exceed keep");
    GPANN_REQUIRE(mass_out == nullptr || mass_out != mass, "mass_out must not be mass");
    if (k_out) {
        GPANN_REQUIRE(k_out != k && v_out != v && k_out != v_out && k_out != v && v_out != k, "the outputs must not overlap the cache");
        for (int i = 0; i < 3; ++i)
            GPANN_REQUIRE(out_kv_stride[i] >= 0 && out_kv_stride[i] % 8 == 0 && out_kv_stride[i] <= (int64_t)1 << 40, "strides must be non-negative multiples of 8 elements");
        GPANN_REQUIRE(BlocksDisjoint(out_kv_stride, L->batch, keep, L->kv_heads, L->head_dim), "an output tensor overlaps itself");
    }
    GPANN_BLOCKS_ENTER(L, stream);
    const BlocksArgs a = BlocksMakeArgs(L, nullptr, k, v, nullptr, 0);
    if (a.B == 0) return GPANN_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t lds = ((size_t)a.Tk + 64) * 4;
    if (a.Tk <= kEvictKeys) GPANN_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(BlocksEvictSelectKernel<true>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    if (a.Tk <= kEvictKeys)
        hipLaunchKernelGGL(BlocksEvictSelectKernel<true>, dim3(a.Hkv, a.B), dim3(1024), lds, st, a, mass, keep, first, last, rows, count);
    else
        hipLaunchKernelGGL(BlocksEvictSelectKernel<false>, dim3(a.Hkv, a.B), dim3(1024), 0, st, a, mass, keep, first, last, rows, count);
    GPANN_HIP_TRY(hipGetLastError());
    if (!k_out && !mass_out) return GPANN_OK;
    const uint32_t chunks = L->head_dim / 8, kept = std::min(keep, L->kv_rows);
    if (kept == 0) return GPANN_OK;
    const uint64_t threads = (uint64_t)kept * a.Hkv * chunks;
    int64_t zero[3] = {0, 0, 0};
    const int64_t* os = out_kv_stride ? out_kv_stride : zero;
    hipLaunchKernelGGL(BlocksEvictCopyKernel, dim3((uint32_t)std::min<uint64_t>((threads + 255) / 256, 1u << 20), a.B), dim3(256), 0, st, a, chunks, keep, kept, rows, count, mass,
                       static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), os[0], os[1], os[2], mass_out);
    GPANN_HIP_TRY(hipGetLastError());
    return GPANN_OK;
}

}  // extern "C"

// Weight gradient of the gated block for fp32 tensors on the tensor cores:
//   dW[pair (j, C)][c][g | u] = sum over tokens t of x[t, 32 C + c] * [dg | du][t, 32 j ...]
// for the pairs of gate and up blocks of the block-sparse matrix, as many-term sums of exact products.
//
// Arithmetic.  An fp32 value is the sum of three bf16 values exactly (3 x 8 significant bits).  With x = x1 + x2 + x3 and
// d = d1 + d2 + d3 the products down to 2^-16 of the largest are six; the rest, 2^-24, is dropped.  Three instructions per 16
// tokens compute them for both projections at once, each into the columns of its order of magnitude:
//   x1 * [d1 d2 d3] (N = 192)    x2 * [d1 d2] (N = 128, 64 columns further)    x3 * [d1] (N = 64, 128 further)
// so that column set k holds the terms of order 2^-8k and the sets are added once, at the end of a segment of tokens.  The tensor
// core's own accumulation drifts by about 2e-8 per addition; segments of 512 tokens (32 additions) keep that near 5e-7, their
// sums are added in fp32 registers (segments of 1024: 757 us instead of 772 on the case below, error 1.6e-6 instead of 1.05e-6).
//
// The three parts are written beforehand as three bf16 matrices ("planes"), transposed: [features][tokens], for x by
// split_planes_kernel and for [dg | du], which the input gradient reads too, by the activation's backward kernel: tokens are the contraction index, and rows of
// 64 tokens are what TMA and the tensor core move as one 128-byte line.
//
// CTA = one item (up to 4 pairs of one pair-row, which fill the 128 rows of an instruction) x one range of tokens.  Per 64 tokens:
// 48 KiB of x, 24 KiB of [dg | du], 12 instructions.  Bound by the tensor core: 8192 tokens, 4096 -> 4096 at density 0.25 take
// 772 us, 1070 TFLOP/s of the six products together where a large dense bf16 product reaches 1390 under the power limit
// (segments of 1024 tokens: 774 us at that time, without the loads 679, without the instructions 543).  bsmm_sddmm takes 1230 us on the same operands.  Token-major
// planes (MN-major operands, 8 pairs per item) measured the same.
//   warp 0 loads, warp 1 issues, warps 2-5 read the sums out.
// Token ranges write partial results that reduce_kernel adds in order; every result repeats bit by bit.
// Every wait is bounded; on expiry the CTA raises the device status word and drains.
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"
#include "bsmm_ptx.cuh"
#include "bsmm_umma.cuh"

namespace bsmm {
namespace {

using namespace ptx;

constexpr int kItemPairs = 4;
constexpr int kStepTokens = 64;
constexpr int kSegmentSteps = 8;                               // 512 tokens between two promotions
constexpr int kPlanes = 3;
constexpr uint32_t kXBlockBytes = 32 * kStepTokens * 2;        // [32 features][64 tokens] bf16
constexpr uint32_t kXPlaneBytes = kItemPairs * kXBlockBytes;
constexpr uint32_t kDPlaneBytes = 64 * kStepTokens * 2;        // [32 g | 32 u][64 tokens] bf16
constexpr uint32_t kDBytes = kPlanes * kDPlaneBytes;
constexpr uint32_t kOffD = kPlanes * kXPlaneBytes;
constexpr uint32_t kStageBytes = kOffD + kDBytes;
constexpr int kStages = 3;
constexpr uint32_t kTmemCols = 256;                            // 192 in use
constexpr uint32_t kOffBar = kStages * kStageBytes;
constexpr uint32_t kOffMisc = kOffBar + (2 * kStages + 2) * 8;
constexpr uint32_t kSmemBytes = kOffMisc + 16 + 1024;          // + slack to align the base to 1 KiB
static_assert(kSmemBytes <= 232448, "shared memory");
constexpr int kEpilogueWarps = 4, kThreads = 32 * (2 + kEpilogueWarps);

// Plan: header (16 bytes: number of items), items, then the pairs by row: (input block, gate slot, up slot, 0), a slot -1 where
// that projection has no block.  A row's pairs begin where its entries do in the CSR.
struct __align__(16) WgradItem {
    int32_t row, first, count, pad;
};

int64_t max_items(int64_t rows, int64_t nnz) { return nnz / kItemPairs + rows; }

struct WgradParams {
    const int32_t* n_items;
    const WgradItem* items;
    const int4* pairs;
    float* out;               // data layout, or partial results [split][nnz][1024]
    float* block_sumsq;       // may be null
    unsigned int* status;
    int64_t tokens, per_split, split_stride;
};

__global__ void __launch_bounds__(kThreads, 1)
gated_wgrad_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_d, const WgradParams p) {
    if ((int)blockIdx.x >= __ldg(p.n_items)) return;  // fewer items than the grid allows for
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    auto full = [&](int s) { return smem_base + kOffBar + 8u * s; };
    auto empty = [&](int s) { return smem_base + kOffBar + 8u * (kStages + s); };
    const uint32_t acc_full = smem_base + kOffBar + 8u * (2 * kStages), acc_empty = acc_full + 8u;
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem_gen + kOffMisc);  // [0] tensor memory, [1] abort
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2 * kStages + 1; ++s) mbar_init(full(s), 1);
        mbar_init(acc_empty, 32 * kEpilogueWarps);
        misc[1] = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_base + kOffMisc, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    volatile uint32_t* abort_flag = &misc[1];
    bool bad = false;  // alike in all lanes of a warp
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
        if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) bad = true;
    };

    const int4 item = __ldg(reinterpret_cast<const int4*>(p.items) + blockIdx.x);  // row, first pair, pairs
    const int count = item.z;
    const int64_t t0 = (int64_t)blockIdx.y * p.per_split, t1 = min(p.tokens, t0 + p.per_split);
    const int steps = (int)((t1 - t0 + kStepTokens - 1) / kStepTokens);

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        const int mine = lane < count ? __ldg(&p.pairs[item.y + lane].x) : 0;
        int cols[kItemPairs];
#pragma unroll
        for (int i = 0; i < kItemPairs; ++i) cols[i] = __shfl_sync(0xffffffffu, mine, i) * 32;
        int issued = 0;
        for (int step = 0; step < steps && !bad; ++step) {
            const int s = step % kStages;
            wait(empty(s), ((uint32_t)(step / kStages) & 1u) ^ 1u);
            if (bad) break;
            const uint32_t stage = smem_base + s * kStageBytes;
            const int32_t tok = (int32_t)(t0 + (int64_t)step * kStepTokens);
            if (elect_one()) {
                mbar_arrive_expect_tx(full(s), (uint32_t)count * kPlanes * kXBlockBytes + kDBytes);
                tma_load_3d(stage + kOffD, &tmap_d, tok, item.x * 64, 0, full(s));
#pragma unroll
                for (int i = 0; i < kItemPairs; ++i)
                    if (i < count)
#pragma unroll
                        for (int q = 0; q < kPlanes; ++q)
                            tma_load_3d(stage + q * kXPlaneBytes + i * kXBlockBytes, &tmap_x, tok, cols[i], q, full(s));
            }
            ++issued;
        }
        if (bad)  // the copies still in flight land in this CTA's memory: they are waited for, again with a limit
            for (int v = max(0, issued - kStages); v < issued; ++v) {
                const long long c0 = clock64();
                while (!mbar_test_wait(full(v % kStages), (uint32_t)(v / kStages) & 1u) && clock64() - c0 < kWaitCycles / 16) {}
            }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA
        constexpr uint32_t idesc1 = make_idesc(1u, 128u, 192u, false, false);
        constexpr uint32_t idesc2 = make_idesc(1u, 128u, 128u, false, false);
        constexpr uint32_t idesc3 = make_idesc(1u, 128u, 64u, false, false);
        for (int step = 0; step < steps && !bad; ++step) {
            const int s = step % kStages, segment = step / kSegmentSteps;
            if (step % kSegmentSteps == 0) {
                wait(acc_empty, ((uint32_t)segment & 1u) ^ 1u);  // the sums of the segment before have been read
                tc_fence_after();
            }
            wait(full(s), (uint32_t)(step / kStages) & 1u);
            if (bad) break;
            const uint32_t stage = smem_base + s * kStageBytes;
            // K-major tiles of 128-byte rows, eight rows 1024 bytes apart; 16 tokens are 32 bytes of a row
            const uint64_t x = smem_desc_sw128(stage, 16u, 1024u), d = smem_desc_sw128(stage + kOffD, 16u, 1024u);
            const uint32_t first = step % kSegmentSteps == 0 ? 0u : 1u;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kStepTokens / 16; ++k) {
                    const uint64_t a = x + (uint64_t)(2 * k), b = d + (uint64_t)(2 * k);
                    mma_ss_f16(tmem, a, b, idesc1, k == 0 ? first : 1u);
                    mma_ss_f16(tmem + 64, a + (kXPlaneBytes >> 4), b, idesc2, 1u);
                    mma_ss_f16(tmem + 128, a + 2 * (kXPlaneBytes >> 4), b, idesc3, 1u);
                }
                mma_commit(empty(s));
                if (step + 1 == steps || (step + 1) % kSegmentSteps == 0) mma_commit(acc_full);
            }
        }
    } else {
        // ------------------------------------------------------------------ read-out
        const int at = warp & 3;  // the pair whose 32 input features are this warp's lanes
        const bool live = at < count;
        const uint32_t from = tmem + ((uint32_t)(at * 32) << 16);
        float sums[64];  // g | u of this lane's feature
#pragma unroll
        for (int j = 0; j < 64; ++j) sums[j] = 0.f;
        const int segments = (steps + kSegmentSteps - 1) / kSegmentSteps;
        for (int segment = 0; segment < segments; ++segment) {
            wait(acc_full, (uint32_t)segment & 1u);
            if (bad) break;
            tc_fence_after();
            if (live) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t v0[16], v1[16], v2[16];
                    tmem_ld16(from + j * 16, v0);
                    tmem_ld16(from + 64 + j * 16, v1);
                    tmem_ld16(from + 128 + j * 16, v2);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sums[j * 16 + e] += __uint_as_float(v0[e]) + (__uint_as_float(v1[e]) + __uint_as_float(v2[e]));
                }
            }
            tc_fence_before();
            mbar_arrive(acc_empty);
        }
        if (live && !bad) {
            const int4 pair = __ldg(p.pairs + item.y + at);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int slot = half == 0 ? pair.y : pair.z;
                if (slot < 0) continue;
                float4* to = reinterpret_cast<float4*>(p.out + (int64_t)blockIdx.y * p.split_stride + (int64_t)slot * kBlockElems + lane * 32);
                float squares = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float* v = sums + half * 32 + 4 * j;
                    to[j] = make_float4(v[0], v[1], v[2], v[3]);
                    squares += v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3];
                }
                if (p.block_sumsq != nullptr) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
                    if (lane == 0) p.block_sumsq[slot] = squares;
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag != 0) atomicOr(p.status, 1u);
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// out = sum of the token ranges' partial results, in order; block_sumsq of the sums
__global__ void __launch_bounds__(256)
wgrad_reduce_kernel(const float* __restrict__ partial, int splits, int64_t split_stride, float* __restrict__ out,
                    float* __restrict__ block_sumsq) {
    __shared__ float red[8];
    const int64_t at = (int64_t)blockIdx.x * kBlockElems + threadIdx.x * 4;
    float4 sum = *reinterpret_cast<const float4*>(partial + at);
    for (int s = 1; s < splits; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(partial + s * split_stride + at);
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    *reinterpret_cast<float4*>(out + at) = sum;
    if (block_sumsq == nullptr) return;
    float squares = sum.x * sum.x + sum.y * sum.y + sum.z * sum.z + sum.w * sum.w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = squares;
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += red[w];
        block_sumsq[blockIdx.x] = t;
    }
}

// planes[q][c][t] = part q of x[t][c], rows of `pitch` tokens.  A CTA turns a tile of 64 tokens x 64 features (32 at the edge)
// through shared memory.  Memory bound: reads 4, writes 6 bytes per value.
__global__ void __launch_bounds__(256)
split_planes_kernel(const float* __restrict__ x, int64_t m, int64_t k, int64_t pitch, __nv_bfloat16* __restrict__ planes) {
    __shared__ float tile[64][65];
    const int64_t col_tiles = (k + 63) / 64, t0 = blockIdx.x / col_tiles * 64, c0 = blockIdx.x % col_tiles * 64;
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = (threadIdx.x >> 4) + i * 16, c = (threadIdx.x & 15) * 4;
        v[i] = t0 + t < m && c0 + c < k ? __ldg(reinterpret_cast<const float4*>(x + (t0 + t) * k + c0 + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = (threadIdx.x >> 4) + i * 16, c = (threadIdx.x & 15) * 4;
        tile[c][t] = v[i].x; tile[c + 1][t] = v[i].y; tile[c + 2][t] = v[i].z; tile[c + 3][t] = v[i].w;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = (threadIdx.x >> 3) + i * 32, t = (threadIdx.x & 7) * 8;
        if (c0 + c >= k || t0 + t >= pitch) continue;
        store_planes(tile[c] + t, planes + (c0 + c) * pitch + t0 + t, k * pitch);
    }
}

// The pairs of one pair-row per CTA: its entries are dropped into a table by input block, prefix sums give the positions.
__global__ void __launch_bounds__(256)
build_row_pairs_kernel(const int32_t* __restrict__ ptr, const int2* __restrict__ idx, int k_blocks, int32_t* __restrict__ counts,
                       int4* __restrict__ pairs) {
    extern __shared__ int32_t slots[];  // [2][k_blocks] gate and up slot + 1
    __shared__ int chunk[256];
    const int row = blockIdx.x, begin = ptr[2 * row], middle = ptr[2 * row + 1], end = ptr[2 * row + 2];
    for (int c = threadIdx.x; c < 2 * k_blocks; c += 256) slots[c] = 0;
    __syncthreads();
    for (int e = begin + threadIdx.x; e < end; e += 256) slots[(e < middle ? 0 : k_blocks) + idx[e].x] = idx[e].y + 1;
    __syncthreads();
    const int per = (k_blocks + 255) / 256, c0 = min(k_blocks, (int)threadIdx.x * per), c1 = min(k_blocks, c0 + per);
    int n = 0;
    for (int c = c0; c < c1; ++c) n += (slots[c] | slots[k_blocks + c]) != 0;
    chunk[threadIdx.x] = n;
    __syncthreads();
    int at = 0;
    for (int t = 0; t < (int)threadIdx.x; ++t) at += chunk[t];
    if (threadIdx.x == 255) counts[row] = at + n;
    for (int c = c0; c < c1; ++c)
        if ((slots[c] | slots[k_blocks + c]) != 0) pairs[begin + at++] = make_int4(c, slots[c] - 1, slots[k_blocks + c] - 1, 0);
}

// one CTA: the rows' pairs cut into items
__global__ void __launch_bounds__(1024)
build_items_kernel(const int32_t* __restrict__ ptr, const int32_t* __restrict__ counts, int rows, int32_t* __restrict__ n_items,
                   WgradItem* __restrict__ items) {
    __shared__ int chunk[1024];
    const int per = (rows + 1023) / 1024, r0 = min(rows, (int)threadIdx.x * per), r1 = min(rows, r0 + per);
    int n = 0;
    for (int r = r0; r < r1; ++r) n += (counts[r] + kItemPairs - 1) / kItemPairs;
    chunk[threadIdx.x] = n;
    __syncthreads();
    int at = 0;
    for (int t = 0; t < (int)threadIdx.x; ++t) at += chunk[t];
    if (threadIdx.x == 1023) *n_items = at + n;
    for (int r = r0; r < r1; ++r)
        for (int i = 0; i < counts[r]; i += kItemPairs) {
            const WgradItem item = {r, ptr[2 * r] + i, min(kItemPairs, counts[r] - i), 0};
            items[at++] = item;
        }
}

struct PlanPointers {
    int32_t* n_items;
    WgradItem* items;
    int4* pairs;
    int32_t* counts;
};
PlanPointers plan_pointers(void* plan, int64_t hidden, int64_t nnz) {
    PlanPointers at;
    at.n_items = static_cast<int32_t*>(plan);
    at.items = reinterpret_cast<WgradItem*>(at.n_items + 4);
    at.pairs = reinterpret_cast<int4*>(at.items + max_items(hidden / 32, nnz));
    at.counts = reinterpret_cast<int32_t*>(at.pairs + nnz);
    return at;
}

// Token ranges: whole waves of CTAs.  A range costs a partial result (8 KiB written and read per pair); with S of them the
// last wave is filled to items * S mod 148, so the S is taken that minimises waves / S, plus 2 % per range, among ranges of at
// least 512 tokens.  (The number of items is estimated for patterns that gate and up share.)
void choose_splits(int64_t rows, int64_t nnz, int64_t tokens, int64_t* splits, int64_t* per) {
    int64_t items = nnz / (2 * kItemPairs) > rows ? nnz / (2 * kItemPairs) : rows;
    if (items < 1) items = 1;
    double best = 0;
    *splits = 1;
    for (int64_t s = 1; s <= 16 && (s == 1 || tokens / s >= 512); ++s) {
        const double cost = (double)((items * s + 147) / 148) / (double)s * (1.0 + 0.02 * (double)(s - 1));
        if (s == 1 || cost < best) {
            best = cost;
            *splits = s;
        }
    }
    *per = ((tokens + *splits - 1) / *splits + 255) / 256 * 256;
    *splits = (tokens + *per - 1) / *per;
    if (*splits < 1) *splits = 1;
}

}  // namespace

GatedPairs gated_pairs(const void* plan, int64_t hidden, int64_t nnz) {
    const PlanPointers at = plan_pointers(const_cast<void*>(plan), hidden, nnz);
    return {at.pairs, at.counts};
}

int64_t gated_wgrad_plan_bytes(int64_t hidden, int64_t nnz) {
    return 16 + 16 * max_items(hidden / 32, nnz) + 16 * nnz + (hidden / 32 + 1) * 4;
}

cudaError_t launch_build_gated_wgrad_plan(const int32_t* ptr, const int32_t* idx, int64_t hidden, int64_t k, int64_t nnz, void* plan,
                                          cudaStream_t stream) {
    const int rows = (int)(hidden / 32), k_blocks = (int)(k / 32);
    if (rows == 0) return cudaSuccess;
    const PlanPointers at = plan_pointers(plan, hidden, nnz);
    build_row_pairs_kernel<<<rows, 256, (size_t)k_blocks * 8, stream>>>(ptr, reinterpret_cast<const int2*>(idx), k_blocks, at.counts, at.pairs);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    build_items_kernel<<<1, 1024, 0, stream>>>(ptr, at.counts, rows, at.n_items, at.items);
    return cudaGetLastError();
}

cudaError_t launch_split_planes(const float* x, int64_t m, int64_t k, void* planes, cudaStream_t stream) {
    if (m == 0 || k == 0) return cudaSuccess;
    const int64_t ctas = (m + 63) / 64 * ((k + 63) / 64);
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    split_planes_kernel<<<(unsigned)ctas, 256, 0, stream>>>(x, m, k, plane_pitch(m), static_cast<__nv_bfloat16*>(planes));
    return cudaGetLastError();
}

int64_t gated_wgrad_workspace_bytes(int64_t hidden, int64_t nnz, int64_t tokens) {
    int64_t splits, per;
    choose_splits(hidden / 32, nnz, tokens, &splits, &per);
    return splits > 1 ? splits * nnz * (int64_t)kBlockElems * 4 : 0;
}

cudaError_t launch_gated_wgrad(const void* x_planes, const void* d_planes, int64_t tokens, int64_t k, int64_t hidden, int64_t nnz,
                               const void* plan, float* out, float* block_sumsq, void* workspace, cudaStream_t stream) {
    if (nnz == 0) return cudaSuccess;
    constexpr int kMaxDevices = 64;
    static bool ready[kMaxDevices] = {false};  // (two threads racing on the first call set it twice)
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (!ready[dev]) {
        err = cudaFuncSetAttribute(gated_wgrad_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
        if (err != cudaSuccess) return err;
        ready[dev] = true;
    }
    CUtensorMap tmap_x, tmap_d;
    const uint64_t pitch = (uint64_t)plane_pitch(tokens);
    err = make_tmap_3d(&tmap_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x_planes, (uint64_t)tokens, (uint64_t)k, kPlanes, pitch, kStepTokens, 32,
                       1, CU_TENSOR_MAP_SWIZZLE_128B);
    if (err == cudaSuccess)
        err = make_tmap_3d(&tmap_d, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, d_planes, (uint64_t)tokens, (uint64_t)(2 * hidden), kPlanes, pitch,
                           kStepTokens, 64, kPlanes, CU_TENSOR_MAP_SWIZZLE_128B);
    if (err != cudaSuccess) return err;
    int64_t splits, per;
    choose_splits(hidden / 32, nnz, tokens, &splits, &per);
    if (splits > 1 && workspace == nullptr) return cudaErrorInvalidValue;
    const PlanPointers at = plan_pointers(const_cast<void*>(plan), hidden, nnz);
    WgradParams p;
    p.n_items = at.n_items;
    p.items = at.items;
    p.pairs = at.pairs;
    p.out = splits > 1 ? static_cast<float*>(workspace) : out;
    p.block_sumsq = splits > 1 ? nullptr : block_sumsq;
    err = device_status_address(&p.status);
    if (err != cudaSuccess) return err;
    p.tokens = tokens;
    p.per_split = per;
    p.split_stride = nnz * (int64_t)kBlockElems;
    const dim3 grid((unsigned)max_items(hidden / 32, nnz), (unsigned)splits);
    gated_wgrad_kernel<<<grid, kThreads, kSmemBytes, stream>>>(tmap_x, tmap_d, p);
    err = cudaGetLastError();
    if (err != cudaSuccess || splits == 1) return err;
    wgrad_reduce_kernel<<<(unsigned)nnz, 256, 0, stream>>>(static_cast<const float*>(workspace), (int)splits, p.split_stride, out, block_sumsq);
    return cudaGetLastError();
}

}  // namespace bsmm

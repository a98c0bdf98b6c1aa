// Tensor-core forward kernel of the gated feed-forward block: both block-sparse projections, the activation and the
// product in one pass, h = act(x Wg^T + bg) * (x Wu^T + bu), for sm_100a.
//
// Block-rows 2j (gate) and 2j + 1 (up) of the matrix are worked on as ONE row of PAIRS: where either has a block at an
// input block, the two (a missing one as zeros) form one right-hand operand of N = 64.  A tcgen05.mma of M = 128 costs
// max(45, N / 2) cycles, so the pair costs what one of its blocks would cost alone; layers built with one pattern for both
// projections have only full pairs.
//
// Tile: 128 tokens x kGroup pair-rows, accumulators in tensor memory, two sets, so that one tile is read out while the next is
// computed.  A tile visits the input blocks for which the group has a pair (the plan lists them); a visit is one stage of a
// ring in shared memory: the [128 x 32] slab of x (TMA, 64-byte swizzle) and the visit's pair images, which lie behind one
// another in memory (packed in the plan's order) and come with one bulk copy.  One CTA per SM walks its tiles.
//   warp 0     loads: plan -> TMA and bulk copies, and the visit's row mask beside them
//   warp 1     tcgen05.mma, both operands from shared memory: two k-steps of 16 per pair; one commit per visit
//   warps 2-5  epilogue: tcgen05.ld, + bias, act(g) * u, (g and u for a backward pass,) stores
// Every wait is bounded; on expiry the CTA raises the device status word and drains.
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"
#include "bsmm_ptx.cuh"
#include "bsmm_umma.cuh"

namespace bsmm {
namespace {

using namespace ptx;

constexpr int kTileTokens = 128;
constexpr int kGroup = 4;                    // pair-rows of a tile
constexpr int kPairCols = 64;                // tensor-memory columns of a pair-row: g | u
constexpr uint32_t kSlabBytes = kTileTokens * 64;   // [128 tokens][32 k] bf16
constexpr uint32_t kPairBytes = 4096;        // bf16 image of a pair: [64 rows g | u][32 k]
constexpr uint32_t kStageBytes = kSlabBytes + kGroup * kPairBytes;
constexpr int kStages = 9;
constexpr int kBuffers = 2;                  // sets of accumulators
constexpr uint32_t kTmemCols = 512;
static_assert(kBuffers * kGroup * kPairCols <= (int)kTmemCols, "tensor memory");
constexpr uint32_t kOffBar = kStages * kStageBytes;
constexpr uint32_t kOffCmd = kOffBar + (2 * kStages + 2 * kBuffers) * 8;
constexpr uint32_t kOffMisc = kOffCmd + kStages * 4;
constexpr uint32_t kSmemBytes = kOffMisc + 16 + 1024;  // + slack to align the base to 1 KiB
static_assert(kSmemBytes <= 232448, "shared memory");
constexpr int kThreads = 192;

// image of a pair: K-major, un-swizzled canonical layout; 8-k chunks of 64 rows x 16 bytes
constexpr uint32_t kPairLbo = 1024, kPairSbo = 128, kPairStepBytes = 2048;

// Plan: [groups] PlanGroup, [groups][k / 32] visits, [nnz] pairs of slots
struct __align__(16) PlanGroup {
    int32_t visits;      // number of input blocks with a pair
    int32_t first_pair;  // pairs of the group: first_pair, + 1, ...; in visit order, within a visit by row
    int32_t rows;        // bit r: row r of the group has a pair
    int32_t pad;
};
struct __align__(16) PlanVisit {
    int32_t inner;       // input block
    int32_t pair;        // first pair of the visit
    int32_t rows;        // bit r: row r of the group has a pair here
    int32_t count;       // pairs of the visit
};

struct GatedParams {
    const PlanGroup* groups;
    const PlanVisit* visits;
    const uint8_t* images;
    const float* bias;        // [2 hidden] or null
    __nv_bfloat16* h;         // [m, hidden]
    __nv_bfloat16* pre;       // [m, 2 hidden] or null
    unsigned int* status;
    int64_t m, hidden;
    int32_t n_groups, n_tiles, k_blocks, n_rows;
    uint32_t x_bytes;
    int32_t act;
};

// The activation where its result is rounded to bf16 (half a step: 2^-8): exp and the quotient by the hardware's
// approximations, about 2^-20.  (With expf and the exact quotient, out of line, reading a tile out took longer than computing it.)
__device__ __forceinline__ float gate_act_bf16(float g, int kind) {
    if (kind == 0) return __fdividef(g, 1.f + __expf(-g));
    return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
}

__global__ void __launch_bounds__(kThreads, 1)
gated_umma_kernel(const __grid_constant__ CUtensorMap tmap_x, const GatedParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    auto full = [&](int s) { return smem_base + kOffBar + 8u * s; };
    auto empty = [&](int s) { return smem_base + kOffBar + 8u * (kStages + s); };
    auto acc_full = [&](int b) { return smem_base + kOffBar + 8u * (2 * kStages + b); };
    auto acc_empty = [&](int b) { return smem_base + kOffBar + 8u * (2 * kStages + kBuffers + b); };
    auto cmd = [&](int s) { return smem_base + kOffCmd + 4u * s; };
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem_gen + kOffMisc);  // [0] tensor memory, [1] abort
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < kBuffers; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), 128); }
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
    bool bad = false;  // alike in all lanes of a warp: the roles' control flow stays uniform when a wait gives up
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
        if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) bad = true;
    };

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        uint32_t seq = 0;  // visits so far, over all tiles
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int g = tile % p.n_groups;
            const int32_t tok0 = tile / p.n_groups * kTileTokens;
            const int visits = __ldg(&p.groups[g].visits);
            const int4* list = reinterpret_cast<const int4*>(p.visits + (int64_t)g * p.k_blocks);
            int4 ahead = lane < visits ? __ldg(list + lane) : make_int4(0, 0, 0, 0);
            for (int base = 0; base < visits && !bad; base += 32) {
                const int4 mine = ahead;
                ahead = base + 32 + lane < visits ? __ldg(list + base + 32 + lane) : make_int4(0, 0, 0, 0);
                const int n = min(32, visits - base);
                for (int i = 0; i < n; ++i, ++seq) {
                    const int s = (int)(seq % kStages);
                    const int inner = __shfl_sync(0xffffffffu, mine.x, i), pair = __shfl_sync(0xffffffffu, mine.y, i);
                    const int rows = __shfl_sync(0xffffffffu, mine.z, i), count = __shfl_sync(0xffffffffu, mine.w, i);
                    wait(empty(s), ((seq / kStages) & 1u) ^ 1u);
                    const uint32_t stage = smem_base + s * kStageBytes;
                    if (elect_one() && !bad) {
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(cmd(s)), "r"(rows) : "memory");
                        mbar_arrive_expect_tx(full(s), p.x_bytes + (uint32_t)count * kPairBytes);
                        tma_load_2d(stage, &tmap_x, inner * 32, tok0, full(s));
                        bulk_load(stage + kSlabBytes, p.images + (int64_t)pair * kPairBytes, (uint32_t)count * kPairBytes, full(s));
                    }
                }
            }
        }
        if (bad) {  // the copies still in flight land in this CTA's memory: they are waited for, again with a limit
            for (uint32_t v = seq > kStages ? seq - kStages : 0; v < seq; ++v) {
                const long long t0 = clock64();
                while (!mbar_test_wait(full((int)(v % kStages)), (v / kStages) & 1u) && clock64() - t0 < kWaitCycles / 16) {}
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA
        constexpr uint32_t idesc = make_idesc(1u, 128u, 64u, false, false);
        uint32_t seq = 0, turn = 0;
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x, ++turn) {
            const int g = tile % p.n_groups, b = (int)(turn % kBuffers);
            const int visits = __ldg(&p.groups[g].visits);
            const uint32_t acc = tmem + (uint32_t)(b * kGroup * kPairCols);
            wait(acc_empty(b), ((turn / kBuffers) & 1u) ^ 1u);
            tc_fence_after();
            uint32_t started = 0;
            for (int i = 0; i < visits && !bad; ++i, ++seq) {
                const int s = (int)(seq % kStages);
                wait(full(s), (seq / kStages) & 1u);
                uint32_t rows;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(rows) : "r"(cmd(s)) : "memory");
                const uint32_t stage = smem_base + s * kStageBytes;
                const uint64_t a = smem_desc_sw64(stage, 16u, 512u);
                uint64_t w = smem_desc_noswizzle(stage + kSlabBytes, kPairLbo, kPairSbo);
                if (elect_one() && !bad) {
#pragma unroll
                    for (int r = 0; r < kGroup; ++r)
                        if ((rows >> r) & 1u) {
                            mma_ss_f16(acc + r * kPairCols, a, w, idesc, (started >> r) & 1u);
                            mma_ss_f16(acc + r * kPairCols, a + 2, w + (kPairStepBytes >> 4), idesc, 1u);
                            w += kPairBytes >> 4;
                        }
                    mma_commit(empty(s));
                }
                started |= rows;
            }
            if (elect_one() && !bad) mma_commit(acc_full(b));
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3;
        const uint32_t tmem_lane = tmem + ((uint32_t)(quarter * 32) << 16);
        uint32_t turn = 0;
        for (int tile = blockIdx.x; tile < p.n_tiles; tile += gridDim.x, ++turn) {
            const int g = tile % p.n_groups, b = (int)(turn % kBuffers);
            const int64_t tok = (int64_t)(tile / p.n_groups) * kTileTokens + quarter * 32 + lane;
            const uint32_t rows = (uint32_t)__ldg(&p.groups[g].rows);
            wait(acc_full(b), (turn / kBuffers) & 1u);
            if (bad) break;
            tc_fence_after();
            for (int r = 0; r < kGroup; ++r) {
                const int row = g * kGroup + r;
                if (row >= p.n_rows) break;
                uint32_t gate[32], up[32];
                if ((rows >> r) & 1u) {
                    tmem_ld32(tmem_lane + (uint32_t)((b * kGroup + r) * kPairCols), gate);
                    tmem_ld32(tmem_lane + (uint32_t)((b * kGroup + r) * kPairCols + 32), up);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) gate[j] = up[j] = 0;
                }
                if (p.bias != nullptr) {
                    const float4* bias = reinterpret_cast<const float4*>(p.bias + (int64_t)row * 64);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 bg = __ldg(bias + j), bu = __ldg(bias + 8 + j);
                        gate[4 * j] = __float_as_uint(__uint_as_float(gate[4 * j]) + bg.x);
                        gate[4 * j + 1] = __float_as_uint(__uint_as_float(gate[4 * j + 1]) + bg.y);
                        gate[4 * j + 2] = __float_as_uint(__uint_as_float(gate[4 * j + 2]) + bg.z);
                        gate[4 * j + 3] = __float_as_uint(__uint_as_float(gate[4 * j + 3]) + bg.w);
                        up[4 * j] = __float_as_uint(__uint_as_float(up[4 * j]) + bu.x);
                        up[4 * j + 1] = __float_as_uint(__uint_as_float(up[4 * j + 1]) + bu.y);
                        up[4 * j + 2] = __float_as_uint(__uint_as_float(up[4 * j + 2]) + bu.z);
                        up[4 * j + 3] = __float_as_uint(__uint_as_float(up[4 * j + 3]) + bu.w);
                    }
                }
                if (p.pre != nullptr && tok < p.m) {
                    __nv_bfloat16* pre = p.pre + tok * 2 * p.hidden + (int64_t)row * 64;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v[8], w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) { v[e] = __uint_as_float(gate[8 * j + e]); w[e] = __uint_as_float(up[8 * j + e]); }
                        store8(pre + 8 * j, v);
                        store8(pre + 32 + 8 * j, w);
                    }
                }
                __nv_bfloat16* h = p.h + tok * p.hidden + (int64_t)row * 32;
                auto finish = [&](int kind) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            v[e] = gate_act_bf16(__uint_as_float(gate[8 * j + e]), kind) * __uint_as_float(up[8 * j + e]);
                        if (tok < p.m) store8(h + 8 * j, v);
                    }
                };
                if (p.act == 0) finish(0); else finish(1);
            }
            tc_fence_before();
            mbar_arrive(acc_empty(b));
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

// ---------------------------------------------------------------------------------------------------------------- plan
// One CTA per group: the group's entries are dropped into a table by input block; its prefix sums give the visits and the
// pairs' positions.  The group's pairs begin where its entries do in the CSR (there are no more pairs than entries).
__global__ void __launch_bounds__(256)
build_gated_plan_kernel(const int32_t* __restrict__ ptr, const int2* __restrict__ idx, int n_rows, int k_blocks,
                        PlanGroup* __restrict__ groups, PlanVisit* __restrict__ visits, int2* __restrict__ pairs) {
    extern __shared__ uint32_t table[];  // [k_blocks] row mask, then first pair of the visit
    uint32_t* first = table + k_blocks;
    __shared__ int chunk_visits[256], chunk_pairs[256];
    const int g = blockIdx.x, row0 = g * kGroup, rows = min(kGroup, n_rows - row0);
    const int begin = ptr[2 * row0], end = ptr[2 * (row0 + rows)];
    for (int c = threadIdx.x; c < k_blocks; c += 256) table[c] = 0;
    for (int e = begin + threadIdx.x; e < end; e += 256) pairs[e] = make_int2(-1, -1);
    __syncthreads();
    auto row_of = [&](int e) {  // block-row (of 2 * rows) of an entry
        int r = 0;
        while (r + 1 < 2 * rows && ptr[2 * row0 + r + 1] <= e) ++r;
        return r;
    };
    for (int e = begin + threadIdx.x; e < end; e += 256) atomicOr(table + idx[e].x, 1u << (row_of(e) >> 1));
    __syncthreads();
    // thread t takes the columns [t * per, (t + 1) * per)
    const int per = (k_blocks + 255) / 256, c0 = min(k_blocks, (int)threadIdx.x * per), c1 = min(k_blocks, c0 + per);
    int nv = 0, np = 0;
    for (int c = c0; c < c1; ++c) {
        nv += table[c] != 0;
        np += __popc(table[c]);
    }
    chunk_visits[threadIdx.x] = nv;
    chunk_pairs[threadIdx.x] = np;
    __syncthreads();
    int v = 0, q = begin;
    uint32_t seen = 0;
    for (int t = 0; t < (int)threadIdx.x; ++t) {
        v += chunk_visits[t];
        q += chunk_pairs[t];
    }
    for (int c = c0; c < c1; ++c) {
        const uint32_t mask = table[c];
        if (mask == 0) continue;
        PlanVisit visit = {c, q, (int32_t)mask, __popc(mask)};
        visits[(int64_t)g * k_blocks + v] = visit;
        first[c] = (uint32_t)q;
        q += visit.count;
        ++v;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < k_blocks; c += 256) seen |= table[c];
    seen = __reduce_or_sync(0xffffffffu, seen);
    __shared__ uint32_t warp_seen[8];
    if ((threadIdx.x & 31) == 0) warp_seen[threadIdx.x >> 5] = seen;
    __syncthreads();
    if (threadIdx.x == 255) {
        uint32_t all = 0;
        for (int w = 0; w < 8; ++w) all |= warp_seen[w];
        PlanGroup group = {v, begin, (int32_t)all, 0};
        groups[g] = group;
    }
    for (int e = begin + threadIdx.x; e < end; e += 256) {
        const int r = row_of(e), c = idx[e].x;
        int* half = reinterpret_cast<int*>(pairs + first[c] + __popc(table[c] & ((1u << (r >> 1)) - 1u)));
        half[r & 1] = idx[e].y;
    }
}

// ---------------------------------------------------------------------------------------------------------------- pack
// The bf16 image of every pair, [gate rows | up rows] x k, from the two blocks' T[c][r] = W[r][c].  Memory bound.
__global__ void __launch_bounds__(256)
pack_pairs_kernel(const float* __restrict__ data, const int2* __restrict__ pairs, uint8_t* __restrict__ images) {
    __shared__ float T[2][32][33];
    const int2 slots = pairs[blockIdx.x];
    if (slots.x < 0 && slots.y < 0) return;  // fewer pairs than entries
    const int tid = threadIdx.x, c = tid >> 3, r4 = (tid & 7) * 4;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int slot = half == 0 ? slots.x : slots.y;
        const float4 v = slot < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                                  : __ldg(reinterpret_cast<const float4*>(data + (int64_t)slot * kBlockElems) + tid);
        T[half][c][r4 + 0] = v.x;
        T[half][c][r4 + 1] = v.y;
        T[half][c][r4 + 2] = v.z;
        T[half][c][r4 + 3] = v.w;
    }
    __syncthreads();
    // 16 bytes per thread: chunk of 8 k, one of 64 rows
    const int chunk = tid >> 6, row = tid & 63, half = row >> 5, r = row & 31;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = T[half][chunk * 8 + j][r];
    store8(reinterpret_cast<__nv_bfloat16*>(images + (int64_t)blockIdx.x * kPairBytes + tid * 16), v);
}

int64_t group_count(int64_t hidden) { return (hidden / 32 + kGroup - 1) / kGroup; }

struct PlanPointers {
    PlanGroup* groups;
    PlanVisit* visits;
    int2* pairs;
};
PlanPointers plan_pointers(void* plan, int64_t hidden, int64_t k) {
    PlanPointers at;
    at.groups = static_cast<PlanGroup*>(plan);
    at.visits = reinterpret_cast<PlanVisit*>(at.groups + group_count(hidden));
    at.pairs = reinterpret_cast<int2*>(at.visits + group_count(hidden) * (k / 32));
    return at;
}

}  // namespace

int64_t gated_plan_bytes(int64_t hidden, int64_t k, int64_t nnz) {
    return group_count(hidden) * (1 + k / 32) * 16 + (nnz > 0 ? nnz : 1) * 8;
}

int64_t gated_images_bytes(int64_t nnz) { return nnz * (int64_t)kPairBytes; }

cudaError_t launch_build_gated_plan(const int32_t* ptr, const int32_t* idx, int64_t hidden, int64_t k, void* plan,
                                    cudaStream_t stream) {
    if (hidden == 0) return cudaSuccess;
    const PlanPointers at = plan_pointers(plan, hidden, k);
    build_gated_plan_kernel<<<(unsigned)group_count(hidden), 256, (size_t)(2 * (k / 32) * 4), stream>>>(
        ptr, reinterpret_cast<const int2*>(idx), (int)(hidden / 32), (int)(k / 32), at.groups, at.visits, at.pairs);
    return cudaGetLastError();
}

cudaError_t launch_pack_pairs(const float* data, const void* plan, int64_t hidden, int64_t k, int64_t nnz, void* images,
                              cudaStream_t stream) {
    if (nnz == 0) return cudaSuccess;
    const PlanPointers at = plan_pointers(const_cast<void*>(plan), hidden, k);
    pack_pairs_kernel<<<(unsigned)nnz, 256, 0, stream>>>(data, at.pairs, static_cast<uint8_t*>(images));
    return cudaGetLastError();
}

cudaError_t launch_gated_umma(const void* x, int64_t m, int64_t k, const void* plan, const void* images, int64_t hidden,
                              const float* bias, void* h, void* pre, int act, cudaStream_t stream) {
    if (m == 0 || hidden == 0) return cudaSuccess;
    constexpr int kMaxDevices = 64;
    static int sm_count[kMaxDevices] = {0};  // (two threads racing on the first call store the same value)
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (sm_count[dev] == 0) {
        err = cudaFuncSetAttribute(gated_umma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
        if (err != cudaSuccess) return err;
        int count = 0;
        err = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
        if (err != cudaSuccess) return err;
        sm_count[dev] = count;
    }
    const int64_t groups = group_count(hidden), tiles = (m + kTileTokens - 1) / kTileTokens;
    if (groups * tiles > 0x7fffffffll || m > 0x7fffffffll) return cudaErrorInvalidValue;
    const uint32_t box_rows = (uint32_t)(m < kTileTokens ? m : kTileTokens);  // (rows behind m hold stale values: not stored)
    CUtensorMap tmap;
    err = make_tmap_2d(&tmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, (uint64_t)k, (uint64_t)m, 32, box_rows, CU_TENSOR_MAP_SWIZZLE_64B);
    if (err != cudaSuccess) return err;
    const PlanPointers at = plan_pointers(const_cast<void*>(plan), hidden, k);
    GatedParams p;
    p.groups = at.groups;
    p.visits = at.visits;
    p.images = static_cast<const uint8_t*>(images);
    p.bias = bias;
    p.h = static_cast<__nv_bfloat16*>(h);
    p.pre = static_cast<__nv_bfloat16*>(pre);
    err = device_status_address(&p.status);
    if (err != cudaSuccess) return err;
    p.m = m;
    p.hidden = hidden;
    p.n_groups = (int32_t)groups;
    p.n_tiles = (int32_t)(groups * tiles);
    p.k_blocks = (int32_t)(k / 32);
    p.n_rows = (int32_t)(hidden / 32);
    p.x_bytes = box_rows * 64u;
    p.act = act;
    const int64_t n_tiles = groups * tiles;
    gated_umma_kernel<<<(unsigned)(n_tiles < sm_count[dev] ? n_tiles : sm_count[dev]), kThreads, kSmemBytes, stream>>>(tmap, p);
    return cudaGetLastError();
}

}  // namespace bsmm

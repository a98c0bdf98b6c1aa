// Tensor-core forward kernel of the gated feed-forward block: both block-sparse projections, the activation and the
// product in one pass, h = act(x Wg^T + bg) * (x Wu^T + bu), for sm_100a.
//
// Block-rows 2j (gate) and 2j + 1 (up) of the matrix are worked on as ONE row of PAIRS: where either has a block at an
// input block, the two (a missing one as zeros) form one right-hand operand of N = 64.  A tcgen05.mma of M = 128 costs
// max(45, N / 2) cycles, so the pair costs what one of its blocks would cost alone; layers built with one pattern for both
// projections have only full pairs.
//
// Tile: 256 tokens (two instructions' M) x two pair-rows, accumulators in tensor memory.  A tile visits the input blocks for
// which the group has a pair (the plan lists them); a visit is one stage of a ring in shared memory: the [256 x 32] slab of x
// (TMA, 64-byte swizzle) and the visit's pair images, which lie behind one another in memory (packed in the plan's order) and
// come with one bulk copy.  One CTA per SM walks its tiles in two pipelines, each with its own half of the ring, of tensor
// memory and of the warps, a tile at a time each: while one reads its tile out the other computes.
// What bounds it is L2 -> shared memory: 20.6 KB per visit, 2.36 GB on a prompt of 4001 tokens, 4096 -> 8192 at density 0.25, in 166 us are
// 14.2 TB/s, which no kernel here exceeds.  (A tile of 128 tokens x four pair-rows, the same memory: 224 us; one pipeline with all of the
// ring: 227 us; rings of five slabs and six images per pipeline instead of four stages: 167.  Without any load, store or read-out
// the same walk takes 126 us, its MMAs alone 90 us.)
//   warps 0-3    loads, two per pipeline: plan -> TMA and bulk copies
//   warps 4-5    tcgen05.mma, both operands from shared memory: two k-steps of 16 per pair; one commit per visit
//   warps 6-21   epilogue, eight per pipeline: tcgen05.ld, + bias, act(g) * u, (g and u for a backward pass,) stores
// Every wait is bounded; on expiry the CTA raises the device status word and drains.
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"
#include "bsmm_ptx.cuh"
#include "bsmm_umma.cuh"

namespace bsmm {
namespace {

using namespace ptx;

constexpr int kHalves = 2;                   // a tile's tokens, 128 at a time (the M of an instruction)
constexpr int kTileTokens = 128 * kHalves;
constexpr int kGroup = 2;                    // pair-rows of a tile
constexpr int kPairCols = 64;                // tensor-memory columns of a pair-row and half: g | u
constexpr uint32_t kHalfSlabBytes = 128 * 64;
constexpr uint32_t kSlabBytes = kTileTokens * 64;   // [256 tokens][32 k] bf16
constexpr uint32_t kPairBytes = 4096;        // bf16 image of a pair: [64 rows g | u][32 k]
constexpr uint32_t kStageBytes = kSlabBytes + kGroup * kPairBytes;
constexpr int kPipelines = 2;
constexpr int kStages = 4;                   // of a pipeline
constexpr int kLoaders = 2;                  // loading warps of a pipeline; a stage stays with one of them
static_assert(kStages % kLoaders == 0, "a stage stays with one loading warp");
constexpr uint32_t kTmemCols = 512;
constexpr int kAccCols = kHalves * kGroup * kPairCols;  // of a pipeline: [half][row][g | u]
static_assert(kPipelines * kAccCols <= (int)kTmemCols, "tensor memory");
constexpr int kBars = 2 * kStages + 2;       // of a pipeline
constexpr uint32_t kOffBar = kPipelines * kStages * kStageBytes;
constexpr uint32_t kOffMisc = kOffBar + kPipelines * kBars * 8;
constexpr uint32_t kSmemBytes = kOffMisc + 16 + 1024;  // + slack to align the base to 1 KiB
static_assert(kSmemBytes <= 232448, "shared memory");
constexpr int kFirstMmaWarp = kPipelines * kLoaders, kFirstEpilogueWarp = kFirstMmaWarp + kPipelines;
constexpr int kEpilogueWarps = 4 * kHalves;  // of a pipeline: every half has its four
constexpr int kThreads = 32 * (kFirstEpilogueWarp + kEpilogueWarps * kPipelines);

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

// The MMAs of a visit.  One case per row mask: within it every operand is a constant step from the visit's first, and the
// single jump costs what one of several conditional branches would.
template <uint32_t kRows>
__device__ __forceinline__ void issue_rows(uint32_t acc, uint64_t a, uint64_t w, uint32_t started, int halves) {
    constexpr uint32_t idesc = make_idesc(1u, 128u, 64u, false, false);
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {
        if (half == 1 && halves == 1) break;
        const uint64_t tokens = a + (uint64_t)(half * (int)(kHalfSlabBytes >> 4));
        int at = 0;
#pragma unroll
        for (int r = 0; r < kGroup; ++r)
            if ((kRows >> r) & 1u) {
                const uint32_t d = acc + (uint32_t)((half * kGroup + r) * kPairCols);
                const uint64_t image = w + (uint64_t)(at * (int)(kPairBytes >> 4));
                mma_ss_f16(d, tokens, image, idesc, (started >> r) & 1u);
                mma_ss_f16(d, tokens + 2, image + (kPairStepBytes >> 4), idesc, 1u);
                ++at;
            }
    }
}
__device__ __forceinline__ void issue_visit(uint32_t rows, uint32_t acc, uint64_t a, uint64_t w, uint32_t started, int halves) {
    switch (rows) {
        case 1: issue_rows<1>(acc, a, w, started, halves); break;
        case 2: issue_rows<2>(acc, a, w, started, halves); break;
        default: issue_rows<3>(acc, a, w, started, halves); break;
    }
}

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
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pl = warp < kFirstMmaWarp ? warp / kLoaders
                   : warp < kFirstEpilogueWarp ? warp - kFirstMmaWarp : (warp - kFirstEpilogueWarp) / kEpilogueWarps;  // pipeline
    const uint32_t bars = smem_base + kOffBar + (uint32_t)(pl * kBars) * 8u;
    const uint32_t ring = smem_base + (uint32_t)(pl * kStages) * kStageBytes;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kStages + s); };
    const uint32_t acc_full = bars + 8u * (2 * kStages), acc_empty = acc_full + 8u;
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem_gen + kOffMisc);  // [0] tensor memory, [1] abort

    if (threadIdx.x == 0) {
        for (int q = 0; q < kPipelines; ++q) {
            const uint32_t at = smem_base + kOffBar + (uint32_t)(q * kBars) * 8u;
            for (int i = 0; i <= 2 * kStages; ++i) mbar_init(at + 8u * i, 1);
            mbar_init(at + 8u * (2 * kStages + 1), 32 * kEpilogueWarps);
        }
        misc[1] = 0;
        fence_mbar_init();
    }
    if (warp == kFirstMmaWarp) {
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

    const int tile0 = (int)blockIdx.x + pl * (int)gridDim.x, tile_step = kPipelines * (int)gridDim.x;
    if (warp < kFirstMmaWarp) {
        // ------------------------------------------------------------------ loads
        const int part = warp % kLoaders;
        int done = 0;              // visits of earlier tiles
        int s = part;              // stage of this warp's next visit, and the parity of its release
        uint32_t parity = 1;
        uint32_t issued = 0;
        for (int tile = tile0; tile < p.n_tiles && !bad; tile += tile_step) {
            const int g = tile % p.n_groups;
            const int32_t tok0 = tile / p.n_groups * kTileTokens;
            const int visits = __ldg(&p.groups[g].visits);
            const int4* list = reinterpret_cast<const int4*>(p.visits + (int64_t)g * p.k_blocks);
            // this warp's visits: those whose number over all tiles is `part` mod kLoaders; lane i holds the i-th of a chunk
            const int begin = (part + kLoaders - done % kLoaders) % kLoaders;
            auto fetch = [&](int i) { return i < visits ? __ldg(list + i) : make_int4(0, 0, 0, 0); };
            int4 ahead = fetch(begin + lane * kLoaders);
            for (int base = begin; base < visits && !bad; base += 32 * kLoaders) {
                const int4 mine = ahead;
                ahead = fetch(base + (32 + lane) * kLoaders);
                const int n = min(32, (visits - base + kLoaders - 1) / kLoaders);
                for (int i = 0; i < n; ++i) {
                    const int inner = __shfl_sync(0xffffffffu, mine.x, i), pair = __shfl_sync(0xffffffffu, mine.y, i);
                    const int count = __shfl_sync(0xffffffffu, mine.w, i);
                    wait(empty(s), parity);
                    const uint32_t stage = ring + s * kStageBytes;
                    if (elect_one() && !bad) {
                        mbar_arrive_expect_tx(full(s), p.x_bytes + (uint32_t)count * kPairBytes);
                        tma_load_2d(stage, &tmap_x, inner * 32, tok0, full(s));
                        bulk_load(stage + kSlabBytes, p.images + (int64_t)pair * kPairBytes, (uint32_t)count * kPairBytes, full(s));
                    }
                    if (!bad) ++issued;
                    s += kLoaders;
                    if (s >= kStages) { s -= kStages; parity ^= 1u; }
                }
            }
            done += visits;
        }
        if (bad) {  // the copies still in flight land in this CTA's memory: they are waited for, again with a limit
            constexpr uint32_t kMine = kStages / kLoaders;
            for (uint32_t v = issued > kMine ? issued - kMine : 0; v < issued; ++v) {
                const long long t0 = clock64();
                while (!mbar_test_wait(full((int)(v % kMine) * kLoaders + part), (v / kMine) & 1u) && clock64() - t0 < kWaitCycles / 16) {}
            }
        }
    } else if (warp < kFirstEpilogueWarp) {
        // ------------------------------------------------------------------ MMA
        const uint64_t a0 = smem_desc_sw64(ring, 16u, 512u);
        const uint64_t w0 = smem_desc_noswizzle(ring + kSlabBytes, kPairLbo, kPairSbo);
        const uint32_t acc = tmem + (uint32_t)(pl * kAccCols);
        int s = 0;
        uint32_t parity = 0, acc_parity = 1;
        for (int tile = tile0; tile < p.n_tiles && !bad; tile += tile_step) {
            const int visits = __ldg(&p.groups[tile % p.n_groups].visits);
            const int halves = (int64_t)(tile / p.n_groups) * kTileTokens + 128 < p.m ? 2 : 1;  // the second one may lie behind the tokens
            wait(acc_empty, acc_parity);
            acc_parity ^= 1u;
            tc_fence_after();
            // lane i holds the row mask of visit base + i; a visit's mask is made warp-uniform (a reduction) one visit ahead, and
            // the next stage's barrier is tested before the current visit is issued, so that both answers arrive on the way
            const int4* list = reinterpret_cast<const int4*>(p.visits + (int64_t)(tile % p.n_groups) * p.k_blocks);
            auto fetch = [&](int i) { return i < visits ? (uint32_t)__ldg(&list[i].z) : 0u; };
            uint32_t masks = fetch(lane), ahead = fetch(32 + lane);
            uint32_t started = 0;  // bit r: row r holds a sum of this tile
            uint32_t rows = __reduce_or_sync(0xffffffffu, lane == 0 ? masks : 0u);
            bool arrived = mbar_test_wait(full(s), parity);
            for (int i = 0; i < visits; ++i) {
                if (!__all_sync(0xffffffffu, arrived)) {
                    wait(full(s), parity);
                    if (bad) break;
                }
                const int now = s;
                if (++s == kStages) { s = 0; parity ^= 1u; }
                arrived = mbar_test_wait(full(s), parity);
                const int next = (i + 1) & 31;
                if (next == 0) {
                    masks = ahead;
                    ahead = fetch(i + 33 + lane);
                }
                const uint32_t rows_next = __reduce_or_sync(0xffffffffu, lane == next ? masks : 0u);
                const uint64_t a = a0 + (uint64_t)(now * (int)(kStageBytes >> 4)), w = w0 + (uint64_t)(now * (int)(kStageBytes >> 4));
                if (elect_one()) {
                    issue_visit(rows, acc, a, w, started, halves);
                    mma_commit(empty(now));
                }
                started |= rows;
                rows = rows_next;
            }
            if (elect_one() && !bad) mma_commit(acc_full);
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3, half = (warp - kFirstEpilogueWarp) / 4 % kHalves;
        const uint32_t tmem_lane = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(pl * kAccCols + half * kGroup * kPairCols);
        uint32_t parity = 0;
        for (int tile = tile0; tile < p.n_tiles; tile += tile_step) {
            const int g = tile % p.n_groups;
            const int64_t tok = (int64_t)(tile / p.n_groups) * kTileTokens + half * 128 + quarter * 32 + lane;
            const uint32_t rows = (uint32_t)__ldg(&p.groups[g].rows);
            wait(acc_full, parity);
            parity ^= 1u;
            if (bad) break;
            tc_fence_after();
            for (int part = 0; part < 2 * kGroup; ++part) {  // 16 hidden units of a row
                const int r = part >> 1, c = (part & 1) * 16, row = g * kGroup + r;
                if (row >= p.n_rows || tok - lane >= p.m) continue;
                uint32_t gate[16], up[16];
                if ((rows >> r) & 1u) {
                    tmem_ld16(tmem_lane + (uint32_t)(r * kPairCols + c), gate);
                    tmem_ld16(tmem_lane + (uint32_t)(r * kPairCols + 32 + c), up);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) gate[j] = up[j] = 0;
                }
                if (p.bias != nullptr) {
                    const float4* bias = reinterpret_cast<const float4*>(p.bias + (int64_t)row * 64 + c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
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
                    __nv_bfloat16* pre = p.pre + tok * 2 * p.hidden + (int64_t)row * 64 + c;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float v[8], w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) { v[e] = __uint_as_float(gate[8 * j + e]); w[e] = __uint_as_float(up[8 * j + e]); }
                        store8(pre + 8 * j, v);
                        store8(pre + 32 + 8 * j, w);
                    }
                }
                __nv_bfloat16* h = p.h + tok * p.hidden + (int64_t)row * 32 + c;
                auto finish = [&](int kind) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
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
            mbar_arrive(acc_empty);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag != 0) atomicOr(p.status, 1u);
    if (warp == kFirstMmaWarp) {
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
// The bf16 image of every pair, [gate rows | up rows] x k, from the two blocks' T[c][r] = W[r][c].  Memory bound; a CTA takes
// kPackPairs pairs and asks for all of their blocks at once (one pair per CTA: 23 us for 67 MB of blocks, four: the same; what is left is the
// ramp of a short kernel: the floor is 15 us).
constexpr int kPackPairs = 4;
__global__ void __launch_bounds__(256)
pack_pairs_kernel(const float* __restrict__ data, const int2* __restrict__ pairs, int64_t count, uint8_t* __restrict__ images) {
    __shared__ float T[kPackPairs][2][32][33];
    const int tid = threadIdx.x, c = tid >> 3, r4 = (tid & 7) * 4;
    const int64_t first = (int64_t)blockIdx.x * kPackPairs;
    int2 slots[kPackPairs];
    float4 v[kPackPairs][2];
#pragma unroll
    for (int i = 0; i < kPackPairs; ++i) slots[i] = first + i < count ? __ldg(pairs + first + i) : make_int2(-1, -1);
#pragma unroll
    for (int i = 0; i < kPackPairs; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int slot = half == 0 ? slots[i].x : slots[i].y;
            v[i][half] = slot < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                                  : __ldg(reinterpret_cast<const float4*>(data + (int64_t)slot * kBlockElems) + tid);
        }
#pragma unroll
    for (int i = 0; i < kPackPairs; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            T[i][half][c][r4 + 0] = v[i][half].x;
            T[i][half][c][r4 + 1] = v[i][half].y;
            T[i][half][c][r4 + 2] = v[i][half].z;
            T[i][half][c][r4 + 3] = v[i][half].w;
        }
    __syncthreads();
    // 16 bytes per thread and pair: chunk of 8 k, one of 64 rows
    const int chunk = tid >> 6, row = tid & 63, half = row >> 5, r = row & 31;
#pragma unroll
    for (int i = 0; i < kPackPairs; ++i) {
        if (slots[i].x < 0 && slots[i].y < 0) continue;  // fewer pairs than entries
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = T[i][half][chunk * 8 + j][r];
        store8(reinterpret_cast<__nv_bfloat16*>(images + (first + i) * kPairBytes + tid * 16), w);
    }
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
    pack_pairs_kernel<<<(unsigned)((nnz + kPackPairs - 1) / kPackPairs), 256, 0, stream>>>(data, at.pairs, nnz,
                                                                                           static_cast<uint8_t*>(images));
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

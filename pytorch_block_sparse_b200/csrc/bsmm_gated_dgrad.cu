// Input gradient of the gated block for fp32 tensors on the tensor cores, dx = [dg | du] W, from the planes that the weight
// gradient reads: three bf16 matrices [features][tokens] that add up to [dg | du] exactly (bsmm_gated_wgrad.cu).
//
// Arithmetic as there: the six products down to 2^-16 of the largest, three instructions per 16 rows of W for a block of 32 columns,
//   d1 * [w1 w2 w3] (N = 96)    d2 * [w1 w2] (N = 64, 32 columns further)    d3 * [w1] (N = 32, 64 further)
// An instruction of M = 128 costs max(45, N / 2) cycles, 138 in all.  The tensor core's accumulation drifts by about 2e-8 per
// addition: after kSegment blocks (32 additions) the sums move to fp32 registers.
//
// Tile: 128 tokens x a group of 2 or 4 block-columns.  A tile visits the block-rows in which the group has a block (the plan
// lists them) and loads their slab of the planes once: [3][32 features][128 tokens], 24 KiB, rows of tokens as they lie, which is
// the tensor core's MN-major operand.  The blocks' images, [w1 w2 w3] x 32 rows, 6 KiB, lie in the order of the visits, so that a
// visit's come with one copy (two where their ring wraps around).
// A block's six instructions are so few that what surrounds them -- a wait of ~85 cycles, commits -- takes longer: four warps
// issue, each into sums of its own, a column's blocks (of a group of 2: every other block of one) each.
// Persistent, one CTA per SM:
//   warp 0 loads slabs, warp 1 images, warps 2-5 issue, warps 6-13 read out (two of the four sums, 32 tokens each)
// Bound by the tensor cores and, beside them, the loads: 8192 tokens, 4096 -> 2 x 4096 at density 0.25 take 920 us and 12 for the
// images, 895 TFLOP/s of the six products together; without loads 790, without instructions 690, neither 525.  (One issuing warp:
// 1650 us.  Images with barriers of their own: 950.  bsmm_dsd in TF32x3, relative error 3.7e-6 instead of 0.9e-6: 872 and 27 for its
// images, and 35 more for writing its operand in fp32.)  1001 tokens, 768 -> 2 x 2048 at 0.5: 39 us and 4; bsmm_dsd 56 and 7.
// Every wait is bounded; on expiry the CTA raises the device status word and drains.
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"
#include "bsmm_ptx.cuh"
#include "bsmm_umma.cuh"

namespace bsmm {
namespace {

using namespace ptx;

constexpr int kMaxGroup = 4, kGroups = 2;              // groups of 2 and 4 block-columns
constexpr int kIssuers = 4;
constexpr int kTileTokens = 128, kPlanes = 3;
constexpr int kSegment = 16;
constexpr uint32_t kPlaneBytes = 32 * 128;             // [32 features][64 tokens] bf16
constexpr uint32_t kHalfBytes = kPlanes * kPlaneBytes; // of 64 tokens
constexpr uint32_t kSlabBytes = 2 * kHalfBytes;
constexpr uint32_t kImageBytes = 96 * 32 * 2;          // [w1 w2 w3][32 rows] bf16
constexpr int kSlabs = 6, kImages = 10;
constexpr uint32_t kOffImages = kSlabs * kSlabBytes;
constexpr uint32_t kOffOut = kOffImages + kImages * kImageBytes;
constexpr int kEpilogueWarps = 8, kThreads = 32 * (2 + kIssuers + kEpilogueWarps);
constexpr int kOutPitch = 20;                          // floats: 16 columns of 32 tokens, read and written without bank conflicts
constexpr uint32_t kOffBar = kOffOut + kEpilogueWarps * 32 * kOutPitch * 4;
constexpr uint32_t kOffMisc = kOffBar + (2 * kSlabs + 2 * kIssuers) * 8;
constexpr uint32_t kSmemBytes = kOffMisc + 16 + 1024;  // + slack to align the base to 1 KiB
static_assert(kSmemBytes <= 232448, "shared memory");
constexpr uint32_t kCols = 96, kTmemCols = 512;        // 4 * 96 in use

// image: K-major, un-swizzled canonical layout; 8-row chunks of 96 columns x 16 bytes
constexpr uint32_t kImageLbo = 96 * 16, kImageSbo = 128, kImageStepBytes = 2 * kImageLbo;

// Plan, for each size of a group: [groups] number of visits, [nnz] visits (block-row | columns << 28), [nnz] slots in the
// order of the visits, within one by column.  A group's begin where its first column's entries do in the CSC.
struct GroupPlan {
    int32_t* visits;
    int32_t* keys;
    int32_t* slots;
};
int64_t groups_of(int64_t cols, int g) { return (cols + (2 << g) - 1) / (2 << g); }
int64_t plan_ints(int64_t cols, int64_t nnz, int g) { return groups_of(cols, g) + 2 * nnz; }
GroupPlan group_plan(void* plan, int64_t cols, int64_t nnz, int g) {
    int32_t* at = static_cast<int32_t*>(plan);
    for (int i = 0; i < g; ++i) at += plan_ints(cols, nnz, i);
    return {at + 2 * nnz, at, at + nnz};
}

struct DgradParams {
    const int32_t* col_ptr;   // CSC offsets
    const int32_t* visits;
    const int32_t* keys;
    const uint8_t* images;
    float* dx;                // [m, k]
    unsigned int* status;
    int64_t m, k;
    int32_t cols, group, n_groups, n_tiles;
};

__global__ void __launch_bounds__(kThreads, 1)
gated_dgrad_kernel(const __grid_constant__ CUtensorMap tmap, const DgradParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars = smem_base + kOffBar;
    auto slab_full = [&](uint32_t s) { return bars + 8u * s; };
    auto slab_empty = [&](uint32_t s) { return bars + 8u * (kSlabs + s); };
    auto acc_full = [&](int a) { return bars + 8u * (2 * kSlabs + a); };
    auto acc_empty = [&](int a) { return bars + 8u * (2 * kSlabs + kIssuers + a); };
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem_gen + kOffMisc);  // [0] tensor memory, [1] abort
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlabs; ++i) {
            mbar_init(slab_full(i), 2);  // the slab, the images
            mbar_init(slab_empty(i), kIssuers);
        }
        for (int i = 0; i < kIssuers; ++i) {
            mbar_init(acc_full(i), 1);
            mbar_init(acc_empty(i), 32 * kEpilogueWarps / 2);
        }
        misc[1] = 0;
        fence_mbar_init();
    }
    if (warp == 2) {
        tmem_alloc(smem_base + kOffMisc, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    const int share = kIssuers / p.group;  // issuing warps of a column
    volatile uint32_t* abort_flag = &misc[1];
    bool bad = false;  // alike in all lanes of a warp
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
        if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) bad = true;
    };

    // The end of the visit in stage s, `parity` of its phase.  A wait costs ~85 cycles also where there is nothing to wait for: the
    // stages from s on are tested at once, and the next `ready` of them are known to have ended.
    auto finished = [&](uint32_t s, uint32_t parity, int& ready) {
        if (ready == 0) ready = mbar_ring_ready(slab_empty(0), kSlabs, (int)s, parity, lane);
        if (ready == 0) {
            wait(slab_empty(s), parity);
            ready = 1;
        }
        --ready;
    };
    // A loader that gave up waits for the copies still in flight, which land in this CTA's memory, again with a limit.
    auto settle = [&](uint32_t seq) {
        if (!bad) return;
        for (uint32_t v = seq > kSlabs ? seq - kSlabs : 0; v < seq; ++v) {
            const long long t0 = clock64();
            while (!mbar_test_wait(slab_full(v % kSlabs), (v / kSlabs) & 1u) && clock64() - t0 < kWaitCycles / 16) {}
        }
    };

    if (warp == 0) {
        // ------------------------------------------------------------------ slabs
        uint32_t s = 0, open = 1, seq = 0;  // stage, parity of its last use's end
        int ready = 0;
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int group = tile % p.n_groups;
            const int32_t tok = tile / p.n_groups * kTileTokens;
            const int first = __ldg(p.col_ptr + group * p.group), count = __ldg(p.visits + group);
            auto fetch = [&](int i) { return i < count ? (__ldg(p.keys + first + i) & 0x0fffffff) * 32 : 0; };
            int ahead = fetch(lane);
            for (int base = 0; base < count && !bad; base += 32) {
                const int mine = ahead, n = min(32, count - base);
                ahead = fetch(base + 32 + lane);
                for (int i = 0; i < n; ++i) {
                    const int32_t row = __shfl_sync(0xffffffffu, mine, i);
                    finished(s, open, ready);
                    if (bad) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(slab_full(s), kSlabBytes);
                        tma_load_3d(smem_base + s * kSlabBytes, &tmap, tok, row, 0, slab_full(s));
                        tma_load_3d(smem_base + s * kSlabBytes + kHalfBytes, &tmap, tok + 64, row, 0, slab_full(s));
                    }
                    if (++s == kSlabs) { s = 0; open ^= 1u; }
                    ++seq;
                }
            }
        }
        settle(seq);
    } else if (warp == 1) {
        // ------------------------------------------------------------------ images
        uint32_t s = 0, seq = 0;                // stage of the visit, and its number
        uint32_t end = 0, open = 0, done = 0;   // the same of the oldest visit in flight
        int ready = 0;
        uint32_t image = 0, in_use = 0;         // next place in the ring of images, and how many of the visits in flight
        uint32_t counts = 0;                    // images of the visits in flight, the oldest lowest, four bits each
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int group = tile % p.n_groups;
            const int first = __ldg(p.col_ptr + group * p.group), count = __ldg(p.visits + group);
            const uint8_t* from = p.images + (int64_t)first * kImageBytes;
            auto fetch = [&](int i) { return i < count ? __popc((uint32_t)__ldg(p.keys + first + i) >> 28) : 0; };
            int ahead = fetch(lane);
            for (int base = 0; base < count && !bad; base += 32) {
                const int mine = ahead, n = min(32, count - base);
                ahead = fetch(base + 32 + lane);
                for (int i = 0; i < n; ++i) {
                    const uint32_t blocks = (uint32_t)__shfl_sync(0xffffffffu, mine, i);
                    while (!bad && (seq - done >= kSlabs || in_use + blocks > kImages)) {
                        finished(end, open, ready);
                        if (++end == kSlabs) { end = 0; open ^= 1u; }
                        in_use -= counts & 15u;
                        counts >>= 4;
                        ++done;
                    }
                    if (bad) break;
                    if (elect_one()) {
                        const uint32_t head = min(blocks, kImages - image), full = slab_full(s);
                        mbar_arrive_expect_tx(full, blocks * kImageBytes);
                        bulk_load(smem_base + kOffImages + image * kImageBytes, from, head * kImageBytes, full);
                        if (head < blocks) bulk_load(smem_base + kOffImages, from + head * kImageBytes, (blocks - head) * kImageBytes, full);
                    }
                    from += blocks * kImageBytes;
                    image = image + blocks < kImages ? image + blocks : image + blocks - kImages;
                    counts |= blocks << (4 * (seq - done));
                    in_use += blocks;
                    if (++s == kSlabs) s = 0;
                    ++seq;
                }
            }
        }
        settle(seq);
    } else if (warp < 2 + kIssuers) {
        // ------------------------------------------------------------------ MMA
        constexpr uint32_t idesc1 = make_idesc(1u, 128u, 96u, true, false);
        constexpr uint32_t idesc2 = make_idesc(1u, 128u, 64u, true, false);
        constexpr uint32_t idesc3 = make_idesc(1u, 128u, 32u, true, false);
        const int issuer = warp - 2, column = issuer & (p.group - 1);
        const uint32_t acc = tmem + issuer * kCols, before = (1u << column) - 1u;  // the columns whose images come before in a visit
        uint32_t s = 0, open = 0, images = 0, turn = 0;
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int group = tile % p.n_groups, col = group * p.group + column;
            const int first = __ldg(p.col_ptr + group * p.group), count = __ldg(p.visits + group);
            // this warp takes blocks issuer / group, + share, ... of its column
            int next = issuer / p.group, at = 0, left = col < p.cols ? __ldg(p.col_ptr + col + 1) - __ldg(p.col_ptr + col) : 0;
            left = (left - next + share - 1) / share;
            int in_segment = 0;
            auto fetch = [&](int i) { return i < count ? __ldg(p.keys + first + i) : 0; };
            int ahead = fetch(lane);
            for (int base = 0; base < count && !bad; base += 32) {
                const int mine = ahead, n = min(32, count - base);
                ahead = fetch(base + 32 + lane);
                for (int i = 0; i < n; ++i) {
                    const uint32_t columns = (uint32_t)__shfl_sync(0xffffffffu, mine, i) >> 28;
                    const bool has = ((columns >> column) & 1u) != 0, takes = has && at == next;
                    wait(slab_full(s), open);
                    if (bad) break;
                    if (takes) {
                        const uint32_t image = images + __popc(columns & before), place = image < kImages ? image : image - kImages;
                        if (in_segment == 0) {
                            wait(acc_empty(issuer), (turn & 1u) ^ 1u);  // the sums before have been read
                            ++turn;
                            tc_fence_after();
                        }
                        if (bad) break;
                        // token-major operand: 64-token halves by the leading offset, groups of eight features by the stride offset
                        const uint64_t d = smem_desc_sw128(smem_base + s * kSlabBytes, kHalfBytes, 1024u);
                        const uint64_t w = smem_desc_noswizzle(smem_base + kOffImages + place * kImageBytes, kImageLbo, kImageSbo);
                        const uint32_t sum = in_segment != 0 ? 1u : 0u;
                        --left;
                        const bool read = ++in_segment == kSegment || left == 0;
                        if (elect_one()) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {  // 16 rows of W
                                const uint64_t a = d + (uint64_t)(h * (2048 >> 4)), b = w + (uint64_t)(h * (int)(kImageStepBytes >> 4));
                                mma_ss_f16(acc, a, b, idesc1, h == 0 ? sum : 1u);
                                mma_ss_f16(acc + 32, a + (kPlaneBytes >> 4), b, idesc2, 1u);
                                mma_ss_f16(acc + 64, a + 2 * (kPlaneBytes >> 4), b, idesc3, 1u);
                            }
                            mma_commit(slab_empty(s));
                            if (read) mma_commit(acc_full(issuer));
                        }
                        if (read) in_segment = 0;
                        next += share;
                    } else if (lane == 0) {
                        mbar_arrive(slab_empty(s));
                    }
                    at += has ? 1 : 0;
                    images += __popc(columns);  // the next visit's first place
                    if (images >= kImages) images -= kImages;
                    if (++s == kSlabs) { s = 0; open ^= 1u; }
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ read-out
        const int quarter = warp & 3, half = (warp - 2 - kIssuers) / 4;  // the sums of issuers half and half + 2
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)half * kCols;
        float* out = reinterpret_cast<float*>(smem_gen + kOffOut) + (warp - 2 - kIssuers) * 32 * kOutPitch;
        uint32_t turn[2] = {0, 0};
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int group = tile % p.n_groups;
            const int64_t tok0 = (int64_t)(tile / p.n_groups) * kTileTokens + quarter * 32;
            const bool live = tok0 < p.m;
            float sums[2][32];
            int segments[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int issuer = half + 2 * c, col = group * p.group + (issuer & (p.group - 1));
                const int blocks = col < p.cols ? __ldg(p.col_ptr + col + 1) - __ldg(p.col_ptr + col) : 0;
                segments[c] = ((blocks - issuer / p.group + share - 1) / share + kSegment - 1) / kSegment;
#pragma unroll
                for (int j = 0; j < 32; ++j) sums[c][j] = 0.f;
            }
            // whichever of the two is ready: neither may hold up the other's issuer, or both would wait for ever
            long long t0 = clock64();
            while (segments[0] + segments[1] > 0 && !bad) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t bar = acc_full(half + 2 * c);
                    if (segments[c] == 0 || !__all_sync(0xffffffffu, mbar_test_wait(bar, turn[c] & 1u))) continue;
                    tc_fence_after();
                    if (live) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t at = from + c * 2 * kCols + j * 16;
                            uint32_t v0[16], v1[16], v2[16];
                            tmem_ld16(at, v0);
                            tmem_ld16(at + 32, v1);
                            tmem_ld16(at + 64, v2);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                sums[c][j * 16 + e] += __uint_as_float(v0[e]) + (__uint_as_float(v1[e]) + __uint_as_float(v2[e]));
                        }
                    }
                    tc_fence_before();
                    mbar_arrive(acc_empty(half + 2 * c));
                    ++turn[c];
                    --segments[c];
                    t0 = clock64();
                }
                if (__any_sync(0xffffffffu, *abort_flag != 0 || clock64() - t0 > kWaitCycles)) {
                    *abort_flag = 1;
                    bad = true;
                }
            }
            if (p.group == 2) {  // one column, shared by two issuers
#pragma unroll
                for (int j = 0; j < 32; ++j) sums[0][j] += sums[1][j];
            }
            if (bad || !live) continue;
            // 16 columns at a time through shared memory: four lanes write 64 bytes of a token
            const int n_live = (int)min((int64_t)32, p.m - tok0);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int j = half + 2 * c, col = group * p.group + j;
                if (j >= p.group || col >= p.cols) continue;  // (the same for all lanes)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float* v = sums[c] + h * 16 + 4 * e;
                        *reinterpret_cast<float4*>(out + lane * kOutPitch + 4 * e) = make_float4(v[0], v[1], v[2], v[3]);
                    }
                    __syncwarp();
                    float* to = p.dx + tok0 * p.k + (int64_t)col * 32 + h * 16 + (lane & 3) * 4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = e * 8 + (lane >> 2);
                        if (t < n_live)
                            *reinterpret_cast<float4*>(to + t * p.k) = *reinterpret_cast<const float4*>(out + t * kOutPitch + (lane & 3) * 4);
                    }
                    __syncwarp();
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag != 0) atomicOr(p.status, 1u);
    if (warp == 2) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// The images, [w1 w2 w3] columns x 32 rows, in the plan's order from data[slot][column][row]: eight rows of a column per thread.
// Memory bound: reads 4, writes 6 bytes per value.
__global__ void __launch_bounds__(256)
pack_block_planes_kernel(const float* __restrict__ data, int64_t nnz, const int32_t* __restrict__ slots, uint8_t* __restrict__ images) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, image = i >> 7;
    if (image >= nnz) return;
    const int c = (int)(i >> 2) & 31, chunk = (int)i & 3;
    float v[8];
    load8(data + (int64_t)__ldg(slots + image) * kBlockElems + c * 32 + chunk * 8, v);
    store_planes(v, reinterpret_cast<__nv_bfloat16*>(images + image * kImageBytes + chunk * kImageLbo + c * 16), 32 * 8);
}

// The visits of one group per CTA, kRange block-rows at a time: the group's entries are dropped into a table by block-row, prefix
// sums give the positions.
constexpr int kRange = 2048;
__global__ void __launch_bounds__(256)
build_visits_kernel(const int32_t* __restrict__ col_ptr, const int2* __restrict__ col_idx, int cols, int rows, int group_size,
                    int32_t* __restrict__ visits, int32_t* __restrict__ keys, int32_t* __restrict__ slots) {
    __shared__ int32_t table[kRange][kMaxGroup];  // slot + 1
    __shared__ int2 chunk[256];                   // visits, blocks
    const int group = blockIdx.x, c0 = group * group_size, first = col_ptr[c0];
    int n_visits = 0, n_slots = 0;
    for (int r0 = 0; r0 < rows; r0 += kRange) {
        for (int i = threadIdx.x; i < kRange * kMaxGroup; i += 256) (&table[0][0])[i] = 0;
        __syncthreads();
        for (int j = 0; j < group_size && c0 + j < cols; ++j)
            for (int e = col_ptr[c0 + j] + threadIdx.x; e < col_ptr[c0 + j + 1]; e += 256) {
                const int2 entry = col_idx[e];
                if (entry.x >= r0 && entry.x < r0 + kRange) table[entry.x - r0][j] = entry.y + 1;
            }
        __syncthreads();
        constexpr int kPer = kRange / 256;
        int2 mine = make_int2(0, 0);
        for (int i = 0; i < kPer; ++i) {
            int blocks = 0;
            for (int j = 0; j < kMaxGroup; ++j) blocks += table[threadIdx.x * kPer + i][j] != 0;
            mine.x += blocks != 0;
            mine.y += blocks;
        }
        chunk[threadIdx.x] = mine;
        __syncthreads();
        int2 at = make_int2(n_visits, n_slots), all = at;
        for (int t = 0; t < 256; ++t) {
            const int2 c = chunk[t];
            if (t < (int)threadIdx.x) at = make_int2(at.x + c.x, at.y + c.y);
            all = make_int2(all.x + c.x, all.y + c.y);
        }
        for (int i = 0; i < kPer; ++i) {
            int columns = 0;
            for (int j = 0; j < kMaxGroup; ++j) {
                const int slot = table[threadIdx.x * kPer + i][j];
                if (slot == 0) continue;
                columns |= 1 << j;
                slots[first + at.y++] = slot - 1;
            }
            if (columns != 0) keys[first + at.x++] = (int32_t)((uint32_t)(r0 + threadIdx.x * kPer + i) | (uint32_t)columns << 28);
        }
        n_visits = all.x;
        n_slots = all.y;
        __syncthreads();  // the table and the sums have been read
    }
    if (threadIdx.x == 0) visits[group] = n_visits;
}

// The size of the group: a block costs its instructions or, where a slab serves few, its share of the loads (71 bytes per cycle and
// SM); a tile a few thousand cycles besides; wider groups fill fewer SMs.  Groups of 2 / 4, us with the images: 8192 tokens, 4096 ->
// 2 x 4096 at density 0.25 1035 / 930; 1001 tokens 177 / 155; 1001 tokens, 768 -> 2 x 2048 at 0.5 43 / 63; 2048 tokens 73 / 68;
// 8192 tokens, 2048 -> 2 x 8192 at 0.1 464 / 422; 300 tokens, 4096 -> 2 x 4096 at 0.1 50 / 45.
int choose_group(int64_t m, int64_t cols, int64_t rows, int64_t nnz) {
    const double density = (double)nnz / ((double)cols * (double)rows);
    int best = 0;
    double least = 0;
    double empty = 1;  // share of the rows in which the group has no block
    for (int g = 0, done = 0; g < kGroups; ++g) {
        const int size = 2 << g;
        for (; done < size; ++done) empty *= 1 - density;
        const double loads = ((1 - empty) * kSlabBytes + size * density * kImageBytes) / 71, instructions = size * density * 276;
        const int64_t tiles = (m + kTileTokens - 1) / kTileTokens * groups_of(cols, g);
        const double cost = (double)((tiles + 147) / 148) * ((double)rows * (loads > instructions ? loads : instructions) + 3000);
        if (g == 0 || cost < least) {
            best = g;
            least = cost;
        }
    }
    return best;
}

}  // namespace

int64_t gated_dgrad_plan_bytes(int64_t k, int64_t nnz) {
    int64_t ints = 0;
    for (int g = 0; g < kGroups; ++g) ints += plan_ints(k / 32, nnz, g);
    return ints * 4;
}

cudaError_t launch_build_gated_dgrad_plan(const int32_t* col_ptr, const int32_t* col_idx, int64_t hidden, int64_t k, int64_t nnz, void* plan,
                                          cudaStream_t stream) {
    const int cols = (int)(k / 32), rows = (int)(hidden / 16);
    if (cols == 0) return cudaSuccess;
    for (int g = 0; g < kGroups; ++g) {
        const GroupPlan at = group_plan(plan, cols, nnz, g);
        build_visits_kernel<<<(unsigned)groups_of(cols, g), 256, 0, stream>>>(col_ptr, reinterpret_cast<const int2*>(col_idx), cols, rows, 2 << g,
                                                                              at.visits, at.keys, at.slots);
        const cudaError_t err = cudaGetLastError();
        if (err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

int64_t gated_dgrad_workspace_bytes(int64_t nnz) { return nnz * (int64_t)kImageBytes; }

cudaError_t launch_gated_dgrad(const void* d_planes, int64_t m, int64_t k, int64_t hidden, int64_t nnz, const float* data,
                               const int32_t* col_ptr, const void* plan, float* dx, void* workspace, cudaStream_t stream) {
    if (m == 0 || k == 0) return cudaSuccess;
    constexpr int kMaxDevices = 64;
    static int sm_count[kMaxDevices] = {0};  // (two threads racing on the first call store the same value)
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (sm_count[dev] == 0) {
        err = cudaFuncSetAttribute(gated_dgrad_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
        if (err != cudaSuccess) return err;
        int count = 0;
        err = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
        if (err != cudaSuccess) return err;
        sm_count[dev] = count;
    }
    const int64_t cols = k / 32;
    const int g = choose_group(m, cols, hidden / 16, nnz);
    const int64_t groups = groups_of(cols, g), tiles = (m + kTileTokens - 1) / kTileTokens * groups, pieces = (nnz + 1) / 2;
    if (tiles > 0x7fffffffll || m > 0x7fffffffll - kTileTokens || hidden / 16 > 0x0fffffffll) return cudaErrorInvalidValue;
    uint8_t* images = static_cast<uint8_t*>(workspace);
    const GroupPlan at = group_plan(const_cast<void*>(plan), cols, nnz, g);
    pack_block_planes_kernel<<<(unsigned)pieces, 256, 0, stream>>>(data, nnz, at.slots, images);
    err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    CUtensorMap tmap;
    err = make_tmap_3d(&tmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, d_planes, (uint64_t)m, (uint64_t)(2 * hidden), kPlanes,
                       (uint64_t)plane_pitch(m), 64, 32, kPlanes, CU_TENSOR_MAP_SWIZZLE_128B);
    if (err != cudaSuccess) return err;
    DgradParams p;
    p.col_ptr = col_ptr;
    p.visits = at.visits;
    p.keys = at.keys;
    p.images = images;
    p.dx = dx;
    err = device_status_address(&p.status);
    if (err != cudaSuccess) return err;
    p.m = m;
    p.k = k;
    p.cols = (int32_t)cols;
    p.group = 2 << g;
    p.n_groups = (int32_t)groups;
    p.n_tiles = (int32_t)tiles;
    gated_dgrad_kernel<<<(unsigned)(tiles < sm_count[dev] ? tiles : sm_count[dev]), kThreads, kSmemBytes, stream>>>(tmap, p);
    return cudaGetLastError();
}

}  // namespace bsmm

// Forward kernel of the gated block for fp32 tensors in the fp32-class precisions: both block-sparse projections, the activation
// and the product in one pass on the tensor cores, h = act(x Wg^T + bg) * (x Wu^T + bu).
//
// Arithmetic, as in bsmm_gated_wgrad.cu: every value is the sum of three bf16 values exactly, and the six products down to 2^-16
// of the largest are added, three instructions per 16 inputs for both projections at once,
//   x1 * [g1 u1 g2 u2 g3 u3] (N = 192)    x2 * [g1 u1 g2 u2] (N = 128, 64 columns further)    x3 * [g1 u1] (N = 64, 128 further)
// so that column set k holds the terms of order 2^-8k.  The tensor core's accumulation drifts by about 2e-8 per addition: after
// every kSegment pairs of a row (two additions of the main term each) the sums move to fp32 registers.
//
// x comes as three bf16 matrices [m][k] (split_rows_kernel), the weights as one 12 KiB image per pair of gate and up blocks, in
// the order of the rows' pairs.  Tile: 256 tokens (two instructions' M) x one pair-row, 2 x 192 accumulator columns.  A visit is one
// pair: 48 KiB of x (three TMA boxes, 64-byte swizzle) and its image, 12 instructions, ~840 cycles at the nominal rate; with 128
// tokens per tile it moves 36 KiB for half of that and is bound by L2 -> shared memory.  Persistent, one CTA per SM:
//   warp 0 loads, warp 1 issues, warps 2-9 read out (four per half), the sums and h through shared memory in whole lines.
// Bound by the tensor cores.  8192 tokens, 4096 -> 2 x 4096 at density 0.25 with g and u kept: 720 us, 1145 TFLOP/s (713 with
// segments of 32 pairs, but a relative error of 1.8e-6 instead of 0.9e-6; 759 with each lane storing its own token) + 52 to split
// x + 19 for the images; bsmm_dsd in TF32x3 and
// bsmm_gated_act as kernels of their own take 941.
// Without g and u kept, TF32x3 products before -> this kernel, us (device, images and split included):
//   4096 tokens, 1024 -> 2 x 4096 at 0.5: 230 -> 185   512: 70 -> 41   64: 39 -> 23
//   4096 tokens, 8192 -> 2 x 2048 at 0.25: 414 -> 400  512: 93 -> 81   64: 91 -> 53
//   4096 tokens, 512 -> 2 x 512 at 0.5: 40 -> 28       512: 19 -> 16   64: 20 -> 16
// The relative error falls from about 4e-6 to 8e-7 throughout.
// Every wait is bounded; on expiry the CTA raises the device status word and drains.
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"
#include "bsmm_ptx.cuh"
#include "bsmm_umma.cuh"

namespace bsmm {
namespace {

using namespace ptx;

constexpr int kHalves = 2, kTileTokens = 128 * kHalves, kPlanes = 3;
constexpr int kSegment = 16;
constexpr uint32_t kPlaneBytes = kTileTokens * 64;     // [256 tokens][32 k] bf16
constexpr uint32_t kXBytes = kPlanes * kPlaneBytes;
constexpr uint32_t kImageBytes = 192 * 32 * 2;         // [g1 u1 g2 u2 g3 u3][32 k] bf16
constexpr uint32_t kStageBytes = kXBytes + kImageBytes;
constexpr int kStages = 3;
constexpr uint32_t kHalfCols = 192, kTmemCols = 512;
constexpr uint32_t kOffBar = kStages * kStageBytes;
constexpr uint32_t kOffMisc = kOffBar + (2 * kStages + 2) * 8;
constexpr int kEpilogueWarps = 4 * kHalves, kThreads = 32 * (2 + kEpilogueWarps);
constexpr int kOutPitch = 36;                          // floats: 32 columns of 32 tokens, read and written without bank conflicts
constexpr uint32_t kOffOut = kOffMisc + 16;
constexpr uint32_t kSmemBytes = kOffOut + kEpilogueWarps * 32 * kOutPitch * 4 + 1024;  // + slack to align the base to 1 KiB
static_assert(kOffOut % 16 == 0 && kSmemBytes <= 232448, "shared memory");

// image: K-major, un-swizzled canonical layout; 8-k chunks of 192 rows x 16 bytes
constexpr uint32_t kImageLbo = 192 * 16, kImageSbo = 128, kImageStepBytes = 2 * kImageLbo;

struct ForwardParams {
    const int32_t* row_first;  // first pair of a pair-row: the CSR offset of its gate's block-row (every other offset)
    const int32_t* row_count;
    const int4* pairs;         // (input block, gate slot, up slot, 0)
    const uint8_t* images;
    const float* bias;         // [2 hidden] or null
    float* h;                  // [m, hidden]
    float* pre;                // [m, 2 hidden] or null
    unsigned int* status;
    int64_t m, hidden;
    int32_t n_rows, n_tiles, tile_tokens;  // 128 or 256 tokens per tile
    uint32_t x_bytes;          // what a visit's boxes of x deliver
    int32_t act;
};

__global__ void __launch_bounds__(kThreads, 1)
gated_f32_kernel(const __grid_constant__ CUtensorMap tmap_x, const ForwardParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    auto full = [&](int s) { return smem_base + kOffBar + 8u * s; };
    auto empty = [&](int s) { return smem_base + kOffBar + 8u * (kStages + s); };
    const uint32_t acc_full = smem_base + kOffBar + 8u * (2 * kStages), acc_empty = acc_full + 8u;
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem_gen + kOffMisc);  // [0] tensor memory, [1] abort
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * kStages + 1; ++i) mbar_init(full(i), 1);
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

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        uint32_t seq = 0;
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int row = tile % p.n_rows;
            const int32_t tok = tile / p.n_rows * p.tile_tokens;
            const int first = __ldg(p.row_first + 2 * row), count = __ldg(p.row_count + row);
            auto fetch = [&](int i) { return i < count ? __ldg(&p.pairs[first + i].x) : 0; };
            int ahead = fetch(lane);
            for (int base = 0; base < count && !bad; base += 32) {
                const int mine = ahead;
                ahead = fetch(base + 32 + lane);
                const int n = min(32, count - base);
                for (int i = 0; i < n; ++i) {
                    const int s = (int)(seq % kStages), col = __shfl_sync(0xffffffffu, mine, i) * 32;
                    wait(empty(s), ((seq / kStages) & 1u) ^ 1u);
                    if (bad) break;
                    const uint32_t stage = smem_base + s * kStageBytes;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(full(s), p.x_bytes + kImageBytes);
                        bulk_load(stage + kXBytes, p.images + (int64_t)(first + base + i) * kImageBytes, kImageBytes, full(s));
#pragma unroll
                        for (int q = 0; q < kPlanes; ++q) tma_load_3d(stage + q * kPlaneBytes, &tmap_x, col, tok, q, full(s));
                    }
                    ++seq;
                }
            }
        }
        if (bad)  // the copies still in flight land in this CTA's memory: they are waited for, again with a limit
            for (uint32_t v = seq > kStages ? seq - kStages : 0; v < seq; ++v) {
                const long long t0 = clock64();
                while (!mbar_test_wait(full((int)(v % kStages)), (v / kStages) & 1u) && clock64() - t0 < kWaitCycles / 16) {}
            }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA
        constexpr uint32_t idesc1 = make_idesc(1u, 128u, 192u, false, false);
        constexpr uint32_t idesc2 = make_idesc(1u, 128u, 128u, false, false);
        constexpr uint32_t idesc3 = make_idesc(1u, 128u, 64u, false, false);
        uint32_t seq = 0, turn = 0;
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int count = __ldg(p.row_count + tile % p.n_rows);
            const bool both = p.tile_tokens > 128 && (int64_t)(tile / p.n_rows) * kTileTokens + 128 < p.m;  // (or none in the second half)
            for (int i = 0; i < count; ++i, ++seq) {
                const int s = (int)(seq % kStages);
                if (i % kSegment == 0) {
                    wait(acc_empty, (turn & 1u) ^ 1u);  // the sums before have been read
                    ++turn;
                    tc_fence_after();
                }
                wait(full(s), (seq / kStages) & 1u);
                if (bad) break;
                const uint32_t stage = smem_base + s * kStageBytes;
                const uint64_t x = smem_desc_sw64(stage, 16u, 512u), w = smem_desc_noswizzle(stage + kXBytes, kImageLbo, kImageSbo);
                const uint32_t acc = i % kSegment == 0 ? 0u : 1u;
                if (elect_one()) {
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        if (half == 1 && !both) break;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t d = tmem + half * kHalfCols;
                            const uint64_t a = x + (uint64_t)(half * (int)((128 * 64) >> 4) + 2 * k), b = w + (uint64_t)(k * (int)(kImageStepBytes >> 4));
                            mma_ss_f16(d, a, b, idesc1, k == 0 ? acc : 1u);
                            mma_ss_f16(d + 64, a + (kPlaneBytes >> 4), b, idesc2, 1u);
                            mma_ss_f16(d + 128, a + 2 * (kPlaneBytes >> 4), b, idesc3, 1u);
                        }
                    }
                    mma_commit(empty(s));
                    if (i + 1 == count || (i + 1) % kSegment == 0) mma_commit(acc_full);
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ read-out
        const int quarter = warp & 3, half = (warp - 2) / 4;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)half * kHalfCols;
        uint32_t turn = 0;
        for (int tile = blockIdx.x; tile < p.n_tiles && !bad; tile += gridDim.x) {
            const int row = tile % p.n_rows, count = __ldg(p.row_count + row);
            const int64_t tok0 = (int64_t)(tile / p.n_rows) * p.tile_tokens + half * 128 + quarter * 32;
            const bool live = tok0 < p.m && half * 128 < p.tile_tokens;
            float sums[64];  // g | u of token tok0 + lane
#pragma unroll
            for (int j = 0; j < 64; ++j) sums[j] = 0.f;
            if (p.bias != nullptr) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + (int64_t)row * 64) + j);
                    sums[4 * j] = b.x; sums[4 * j + 1] = b.y; sums[4 * j + 2] = b.z; sums[4 * j + 3] = b.w;
                }
            }
            for (int i = 0; i < count; i += kSegment, ++turn) {
                wait(acc_full, turn & 1u);
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
            if (bad || !live) continue;
            // 32 columns of 32 tokens at a time through shared memory: eight lanes write a token's 128 bytes
            float* out = reinterpret_cast<float*>(smem_gen + kOffOut) + (warp - 2) * 32 * kOutPitch;
            const int n_live = (int)min((int64_t)32, p.m - tok0);
            auto store = [&](const float* v, float* to, int64_t pitch) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *reinterpret_cast<float4*>(out + lane * kOutPitch + 4 * j) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int t = j * 4 + (lane >> 3);
                    if (t < n_live)
                        *reinterpret_cast<float4*>(to + (tok0 + t) * pitch + (lane & 7) * 4) =
                            *reinterpret_cast<const float4*>(out + t * kOutPitch + (lane & 7) * 4);
                }
                __syncwarp();
            };
            if (p.pre != nullptr) {
                store(sums, p.pre + (int64_t)row * 64, 2 * p.hidden);
                store(sums + 32, p.pre + (int64_t)row * 64 + 32, 2 * p.hidden);
            }
            if (p.act == 0) {
#pragma unroll
                for (int j = 0; j < 32; ++j) sums[j] = gate_act(sums[j], 0) * sums[32 + j];
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) sums[j] = gate_act(sums[j], 1) * sums[32 + j];
            }
            store(sums, p.h + (int64_t)row * 32, p.hidden);
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

// planes[q][i] = part q of x[i], eight values per thread.  Memory bound: reads 4, writes 6 bytes per value.
__global__ void __launch_bounds__(256)
split_rows_kernel(const float* __restrict__ x, int64_t n, __nv_bfloat16* __restrict__ planes) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= n) return;
    float v[8];
    load8(x + i, v);
    store_planes(v, planes + i, n);
}

// The image of every pair, [g1 u1 g2 u2 g3 u3] x k, from the two blocks' T[c][r] = W[r][c].  Memory bound.
__global__ void __launch_bounds__(256)
pack_pair_planes_kernel(const float* __restrict__ data, const int32_t* __restrict__ row_first, const int32_t* __restrict__ row_count,
                        const int4* __restrict__ pairs, uint8_t* __restrict__ images) {
    __shared__ float T[2][32][33];
    const int row = blockIdx.x, first = __ldg(row_first + 2 * row), count = __ldg(row_count + row);
    const int tid = threadIdx.x, c = tid >> 3, r4 = (tid & 7) * 4;
    for (int i = blockIdx.y; i < count; i += gridDim.y) {
        const int4 pair = __ldg(pairs + first + i);
        float4 v[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int slot = half == 0 ? pair.y : pair.z;
            v[half] = slot < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                               : __ldg(reinterpret_cast<const float4*>(data + (int64_t)slot * kBlockElems) + tid);
        }
        __syncthreads();  // the block before has been read
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            T[half][c][r4] = v[half].x; T[half][c][r4 + 1] = v[half].y; T[half][c][r4 + 2] = v[half].z; T[half][c][r4 + 3] = v[half].w;
        }
        __syncthreads();
        // eight k of one of the 64 rows, in three parts: 16 bytes each
        const int chunk = tid >> 6, r = tid & 63;
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = T[r >> 5][chunk * 8 + j][r & 31];
        store_planes(w, reinterpret_cast<__nv_bfloat16*>(images + (int64_t)(first + i) * kImageBytes + chunk * kImageLbo + r * 16), 64 * 8);
    }
}

}  // namespace

int64_t gated_f32_workspace_bytes(int64_t m, int64_t k, int64_t nnz) { return (6 * m * k + 255) / 256 * 256 + nnz * (int64_t)kImageBytes; }

cudaError_t launch_gated_f32(const float* x, int64_t m, int64_t k, const float* data, int64_t nnz, const int32_t* ptr,
                             const void* pairs_plan, int64_t hidden, const float* bias, float* h, float* pre, int act, void* workspace,
                             cudaStream_t stream) {
    if (m == 0 || hidden == 0) return cudaSuccess;
    constexpr int kMaxDevices = 64;
    static int sm_count[kMaxDevices] = {0};  // (two threads racing on the first call store the same value)
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (sm_count[dev] == 0) {
        err = cudaFuncSetAttribute(gated_f32_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
        if (err != cudaSuccess) return err;
        int count = 0;
        err = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
        if (err != cudaSuccess) return err;
        sm_count[dev] = count;
    }
    const int64_t rows = hidden / 32, pieces = (m * k / 8 + 255) / 256;
    // Tiles of 128 tokens where those of 256 leave SMs idle: a visit takes about 3/5 of the time for half the tokens.
    // (256 tokens, 8192 -> 2 x 2048 at density 0.25: 59 us, 77 in tiles of 256; 4096 -> 2 x 1024 at 0.5: 45 and 63.)
    const int64_t sms = sm_count[dev], whole = (m + kTileTokens - 1) / kTileTokens * rows, halves = (m + 127) / 128 * rows;
    const bool small = 3 * ((halves + sms - 1) / sms) < 5 * ((whole + sms - 1) / sms);
    const int64_t tiles = small ? halves : whole;
    if (halves > 0x7fffffffll || pieces > 0x7fffffffll || m > 0x7fffffffll) return cudaErrorInvalidValue;
    uint8_t* planes = static_cast<uint8_t*>(workspace);
    uint8_t* images = planes + (6 * m * k + 255) / 256 * 256;
    const GatedPairs at = gated_pairs(pairs_plan, hidden, nnz);
    split_rows_kernel<<<(unsigned)pieces, 256, 0, stream>>>(x, m * k, reinterpret_cast<__nv_bfloat16*>(planes));
    err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    // a row's pairs are dealt to as many CTAs as give the GPU enough of them
    const int64_t per_row = nnz / rows / 2 > 0 ? nnz / rows / 2 : 1, want = (8 * 148 + rows - 1) / rows;
    const int64_t split = want < per_row ? want : per_row;
    pack_pair_planes_kernel<<<dim3((unsigned)rows, (unsigned)split), 256, 0, stream>>>(data, ptr, at.counts, at.pairs, images);
    err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    const uint32_t tile_tokens = small ? 128 : kTileTokens, box_rows = (uint32_t)(m < tile_tokens ? m : tile_tokens);  // (rows behind m hold stale values: not stored)
    CUtensorMap tmap;
    err = make_tmap_3d(&tmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, planes, (uint64_t)k, (uint64_t)m, kPlanes, (uint64_t)k, 32, box_rows, 1,
                       CU_TENSOR_MAP_SWIZZLE_64B);
    if (err != cudaSuccess) return err;
    ForwardParams p;
    p.row_first = ptr;
    p.row_count = at.counts;
    p.pairs = at.pairs;
    p.images = images;
    p.bias = bias;
    p.h = h;
    p.pre = pre;
    err = device_status_address(&p.status);
    if (err != cudaSuccess) return err;
    p.m = m;
    p.hidden = hidden;
    p.n_rows = (int32_t)rows;
    p.n_tiles = (int32_t)tiles;
    p.tile_tokens = (int32_t)tile_tokens;
    p.x_bytes = kPlanes * box_rows * 64u;
    p.act = act;
    gated_f32_kernel<<<(unsigned)(tiles < sm_count[dev] ? tiles : sm_count[dev]), kThreads, kSmemBytes, stream>>>(tmap, p);
    return cudaGetLastError();
}

}  // namespace bsmm

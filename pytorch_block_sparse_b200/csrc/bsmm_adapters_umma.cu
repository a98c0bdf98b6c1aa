// Shrink kernel of the low-rank adapters for prompts of bf16 tensors on the fifth-generation tensor cores: v = x D_a^T for up to
// 128 tokens of one request, [128 x K] x [K x rank] with tcgen05.mma.  Both operands arrive by TMA in stages of 64 features
// and are used as they lie; the CTAs of a cluster take a part of the features each and add their sums through distributed
// shared memory.  Bound by reading x.  6001 tokens in 24 requests, 4096 features, rank 64: 17 us against 26 for mma.sync with
// cp.async (the form of fp32 tensors and higher ranks), whose eight warps spend their time on fragment loads and barriers.  (The
// expand kernel stays with mma.sync: from registers its sums meet the base where they are, while tensor memory's rows
// have to pass through shared memory to be stored in lines: measured 42 against 28 us.)
// A tile that ends inside the 128 rows computes the rows behind it along and does not store them.
// Every wait is bounded; on expiry the CTA raises the device status word and drains.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "bsmm_adapters.cuh"
#include "bsmm_ptx.cuh"
#include "bsmm_umma.cuh"

namespace bsmm {
namespace {

namespace cg = cooperative_groups;
using namespace adapters;
using namespace ptx;

constexpr uint32_t kXBytes = kTileTokens * 128;   // [128 tokens][64 features] bf16, 128-byte swizzle

// A wait that gives up makes `bad` true in all lanes of the warp alike.
struct Waiter {
    volatile uint32_t* abort_flag;
    bool bad = false;
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
        if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) bad = true;
    }
    // copies in flight when a role gave up land in this CTA's memory: waited for, again with a limit
    __device__ __forceinline__ void settle(uint32_t bar, uint32_t parity) {
        const long long t0 = clock64();
        while (!mbar_test_wait(bar, parity) && clock64() - t0 < kWaitCycles / 16) {}
    }
};

// ---------------------------------------------------------------------------------------------------------------- shrink
template <int kRank>
struct Shrink {
    static constexpr uint32_t kDBytes = kRank * 128;
    static constexpr uint32_t kStage = kXBytes + kDBytes;
    static constexpr int kStages = kRank <= 64 ? 4 : 3;             // two CTAs per SM
    static constexpr uint32_t kTmemCols = kRank < 32 ? 32 : kRank;
    static constexpr uint32_t kPitch = kRank + 4;                   // floats of a row of sums: four rows apart, another bank
    static constexpr uint32_t kOffBar = kStages * kStage;
    static constexpr uint32_t kOffMisc = kOffBar + (2 * kStages + 1) * 8;
    static constexpr uint32_t kSmem = kOffMisc + 16 + 1024;
    static_assert(kTileTokens * kPitch * 4 <= kOffBar, "the sums reuse the ring");
    static_assert(2 * (kSmem + 1024) <= 233472, "two CTAs per SM");
};
constexpr int kShrinkThreads = 192;  // warp 0 loads, 1 issues, all sum up; 2-5 read tensor memory

template <int kRank>
__global__ void __launch_bounds__(kShrinkThreads, 2)
shrink_umma_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_down, const AdapterCall p,
                   const Units units, unsigned int* status) {
    using S = Shrink<kRank>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const int parts = (int)units.parts, part = (int)blockIdx.x % parts;
    Tile tile;
    if (!tile.find(p, (int)blockIdx.x / parts) || tile.id == kNone) return;  // (the whole cluster alike)

    auto full = [&](int s) { return smem_base + S::kOffBar + 8u * s; };
    auto empty = [&](int s) { return smem_base + S::kOffBar + 8u * (S::kStages + s); };
    const uint32_t acc_full = smem_base + S::kOffBar + 8u * (2 * S::kStages);
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem_gen + S::kOffMisc);  // [0] tensor memory, [1] abort
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * S::kStages + 1; ++i) mbar_init(full(i), 1);
        misc[1] = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_base + S::kOffMisc, S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    let_expand_start();
    const uint32_t tmem = misc[0];
    Waiter wait = {&misc[1]};
    const int64_t k0 = min(p.inner, part * units.per_part), k1 = min(p.inner, k0 + units.per_part);
    const int steps = (int)((k1 - k0 + 63) / 64);

    if (warp == 0) {
        int issued = 0;
        for (int i = 0; i < steps; ++i) {
            const int s = i % S::kStages;
            wait(empty(s), ((uint32_t)(i / S::kStages) & 1u) ^ 1u);
            if (wait.bad) break;
            if (elect_one()) {
                mbar_arrive_expect_tx(full(s), S::kStage);
                tma_load_2d(smem_base + s * S::kStage, &tmap_x, (int32_t)(k0 + i * 64), tile.first, full(s));
                tma_load_2d(smem_base + s * S::kStage + kXBytes, &tmap_down, (int32_t)(k0 + i * 64), tile.id * kRank, full(s));
            }
            ++issued;
        }
        if (wait.bad)
            for (int v = max(0, issued - S::kStages); v < issued; ++v) wait.settle(full(v % S::kStages), (uint32_t)(v / S::kStages) & 1u);
    } else if (warp == 1) {
        constexpr uint32_t idesc = make_idesc(1u, 128u, (uint32_t)kRank, false, false);
        for (int i = 0; i < steps; ++i) {
            const int s = i % S::kStages;
            wait(full(s), (uint32_t)(i / S::kStages) & 1u);
            if (wait.bad) break;
            const uint64_t a = smem_desc_sw128(smem_base + s * S::kStage, 16u, 1024u);
            const uint64_t b = smem_desc_sw128(smem_base + s * S::kStage + kXBytes, 16u, 1024u);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_ss_f16(tmem, a + (uint64_t)(2 * k), b + (uint64_t)(2 * k), idesc, i > 0 || k > 0 ? 1u : 0u);
                mma_commit(empty(s));
                if (i + 1 == steps) mma_commit(acc_full);
            }
        }
    } else {
        // the sums to shared memory: a lane is a token; the ring's last reader has finished with acc_full
        float* row = reinterpret_cast<float*>(smem_gen) + ((warp & 3) * 32 + lane) * S::kPitch;
        if (steps > 0) {
            wait(acc_full, 0);
            tc_fence_after();
        }
        if (!wait.bad) {
#pragma unroll
            for (int c = 0; c < kRank; c += 16) {
                uint32_t v[16];
                if (steps > 0) {
                    tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c, v);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<uint4*>(row + c + 4 * j) =
                        steps > 0 ? make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]) : make_uint4(0u, 0u, 0u, 0u);
            }
        }
        tc_fence_before();
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (parts > 1) cluster.sync(); else __syncthreads();
    tc_fence_after();
    // every CTA adds up a share of the tile's rows, in the order of the parts
    const float* sums = reinterpret_cast<const float*>(smem_gen);
    for (int i = part * kShrinkThreads + threadIdx.x; i < tile.rows * (kRank / 4); i += parts * kShrinkThreads) {
        const int at = i / (kRank / 4) * (int)S::kPitch + i % (kRank / 4) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < parts; ++c) {
            const float4 w = *reinterpret_cast<const float4*>((parts > 1 ? cluster.map_shared_rank(sums, c) : sums) + at);
            sum.x += w.x; sum.y += w.y; sum.z += w.z; sum.w += w.w;
        }
        *reinterpret_cast<float4*>(p.workspace + (int64_t)(tile.first + i / (kRank / 4)) * kRank + i % (kRank / 4) * 4) = sum;
    }
    if (parts > 1) cluster.sync(); else __syncthreads();  // the sums have been read
    if (threadIdx.x == 0 && misc[1] != 0) atomicOr(status, 1u);
    if (warp == 1) tmem_dealloc(tmem, S::kTmemCols);
}

template <int kRank>
cudaError_t launch(const AdapterCall& p, const Units& units, cudaStream_t stream) {
    static bool ready[64] = {false};
    cudaError_t err = allow_smem(shrink_umma_kernel<kRank>, (int)Shrink<kRank>::kSmem, ready);
    if (err != cudaSuccess) return err;
    CUtensorMap tmap_x, tmap_down;
    err = make_tmap_2d(&tmap_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.x, (uint64_t)p.inner, (uint64_t)p.tokens, 64, kTileTokens,
                       CU_TENSOR_MAP_SWIZZLE_128B);
    if (err == cudaSuccess)
        err = make_tmap_2d(&tmap_down, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.down, (uint64_t)p.inner, (uint64_t)(p.count * kRank), 64, kRank,
                           CU_TENSOR_MAP_SWIZZLE_128B);
    unsigned int* status = nullptr;
    if (err == cudaSuccess) err = device_status_address(&status);
    if (err != cudaSuccess) return err;
    return launch_with(shrink_umma_kernel<kRank>, units.tiles * units.parts, kShrinkThreads, (int)Shrink<kRank>::kSmem, (int)units.parts, false,
                       stream, tmap_x, tmap_down, p, units, status);
}

}  // namespace

bool adapters::shrink_on_umma(const AdapterCall& p, bool bf16) {
    // (tensor maps count rows in 31 bits, and a box may not exceed its tensor)
    return bf16 && p.rank <= 128 && p.inner >= 64 && p.tokens >= kTileTokens && p.tokens <= 0x7fffffffll && p.count * p.rank <= 0x7fffffffll;
}

cudaError_t adapters::launch_shrink_umma(const AdapterCall& p, const Units& units, cudaStream_t stream) {
    switch (p.rank) {
        case 16: return launch<16>(p, units, stream);
        case 32: return launch<32>(p, units, stream);
        case 64: return launch<64>(p, units, stream);
        case 128: return launch<128>(p, units, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace bsmm

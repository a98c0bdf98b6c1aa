// What the kernels of the low-rank adapters share: cutting a batch into tiles of one request's tokens, and launching.
#pragma once
#include "bsmm_feedforward.cuh"

namespace bsmm {
namespace adapters {

constexpr int kNone = -1;
constexpr int kTileTokens = 128;

// The expand kernel is launched while the shrink kernel still runs (programmatic dependent launch): what it does before
// this wait -- finding its work, the first loads of U and of the base -- overlaps the other's tail.  Every thread waits before
// it leaves, so that the expand grid never completes before the shrink grid.
__device__ __forceinline__ void wait_for_shrink() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_expand_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct Units {
    int64_t tiles;      // of 128 tokens
    int64_t parts;      // ranges of input features (shrink) or of output features (expand)
    int64_t per_part;   // features of a part, a multiple of 32
};

// Up to 128 tokens of one request.  The requests' tokens are cut into such tiles from each request's start; the tokens before
// the first request and behind the last one count as requests without an adapter.
struct Tile {
    int first, rows, id;
    // Each warp finds the tile by itself, 32 requests at a time.  False: there are fewer tiles.
    __device__ __forceinline__ bool find(const AdapterCall& p, int tile) {
        const int lane = threadIdx.x & 31, requests = (int)p.requests, tokens = (int)p.tokens;
        int before = 0;
        for (int r0 = -1; r0 <= requests; r0 += 32) {
            const int r = r0 + lane;
            int start = 0, end = 0, adapter = kNone;
            if (r <= requests) {
                start = r < 0 ? 0 : min(max(__ldg(p.offsets + r), 0), tokens);
                end = r == requests ? tokens : min(max(__ldg(p.offsets + r + 1), 0), tokens);
                if (r >= 0 && r < requests) adapter = __ldg(p.ids + r);
                if (adapter < 0 || adapter >= p.count) adapter = kNone;
            }
            const int tiles = (max(end - start, 0) + kTileTokens - 1) / kTileTokens;
            int sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int below = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += below;
            }
            const uint32_t reached = __ballot_sync(0xffffffffu, before + sum > tile);
            if (reached != 0) {
                const int src = __ffs(reached) - 1;
                const int skipped = tile - before - __shfl_sync(0xffffffffu, sum - tiles, src);
                first = __shfl_sync(0xffffffffu, start, src) + skipped * kTileTokens;
                rows = min(kTileTokens, __shfl_sync(0xffffffffu, end, src) - first);
                id = __shfl_sync(0xffffffffu, adapter, src);
                return true;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        return false;
    }
};

// Tokens without an adapter keep their base, columns n0 ... n1 - 1 of a tile: eight pieces in flight per thread.
template <typename O, int kThreads>
__device__ __forceinline__ void keep_base(const AdapterCall& p, const Tile& tile, int64_t n0, int64_t n1) {
    if (p.base == p.out) return;
    const int per_row = (int)(n1 - n0) / 8, pieces = tile.rows * per_row;
    for (int i0 = threadIdx.x; i0 < pieces; i0 += 8 * kThreads) {
        Raw8<O> v[8];
        int64_t at[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + j * kThreads;
            at[j] = (tile.first + i / per_row) * p.outer + n0 + i % per_row * 8;
            if (i < pieces && p.base != nullptr) v[j].load(static_cast<const O*>(p.base) + at[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (p.base != nullptr) v[j].unpack(f);
            if (i0 + j * kThreads < pieces) store8(static_cast<O*>(p.out) + at[j], f);
        }
    }
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How the input features are cut: CTAs of a cluster (a power of two up to 8), two per SM, at least 256 features each.  Tiles
// start at each request's start, so that there may be one more for every request and for the tokens around them; half that is expected.
inline Units tile_units(const AdapterCall& p) {
    Units u;
    u.tiles = ceil_div(p.tokens, kTileTokens) + p.requests + 2;
    const int64_t expected = ceil_div(p.tokens, kTileTokens) + p.requests / 2;
    u.parts = 1;
    while (u.parts < 8 && expected * u.parts * 2 <= 2 * 148 && u.parts * 2 * 256 <= p.inner) u.parts *= 2;
    u.per_part = ceil_div(ceil_div(p.inner, u.parts), 64) * 64;
    return u;
}

// A launch in clusters of `cluster` CTAs, or one that may begin while the kernel before it still runs.
template <typename... Params, typename... Args>
cudaError_t launch_with(void (*kernel)(Params...), int64_t ctas, int threads, int smem, int cluster, bool early,
                        cudaStream_t stream, Args... args) {
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)ctas);
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = (size_t)smem;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    if (early) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
    } else {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    }
    config.attrs = attr;
    config.numAttrs = early || cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, bool (&ready)[64]) {  // per device; racing first calls set it twice
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (ready[dev]) return cudaSuccess;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess) ready[dev] = true;
    return err;
}

// the expand kernel's ranges of output features, in multiples of `unit`, for `wanted` CTAs or warps in all
inline void cut_outputs(Units& u, int64_t outer, int64_t unit, int64_t wanted_parts) {
    const int64_t most = ceil_div(outer, unit);
    int64_t parts = wanted_parts < most ? wanted_parts : most;
    parts = parts < 1 ? 1 : parts;
    u.per_part = ceil_div(most, parts) * unit;
    u.parts = ceil_div(outer, u.per_part);
}

// the shrink kernel of tiles on the fifth-generation tensor cores (bsmm_adapters_umma.cu), and whether it takes the call
bool shrink_on_umma(const AdapterCall& p, bool bf16);
cudaError_t launch_shrink_umma(const AdapterCall& p, const Units& units, cudaStream_t stream);

}  // namespace adapters
}  // namespace bsmm

// The gated feed-forward block's own arithmetic, h = act(g) * u with g = x Wg^T + bg and u = x Wu^T + bu, around
// pre-activations whose columns alternate in blocks of 32: columns 64 j ... 64 j + 31 of `pre` [m, 2 hidden] are g of the
// hidden units 32 j ... 32 j + 31, the next 32 their u.  (Wg and Wu are one block-sparse matrix of 2 hidden rows whose
// block-rows alternate the same way, so one product computes `pre`, and the gradients with respect to the input and to
// both weights are one product each.)
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"

namespace bsmm {
namespace {

namespace cg = cooperative_groups;

constexpr int kRowsPerChunk = 256;  // rows whose bias gradient one CTA adds up

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&v)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xFFFF0000u);
    v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xFFFF0000u);
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// Memory bound: reads 2, writes 1 value per hidden unit and token (8192 x 4096 fp32, 403 MB: 61 us, 6.6 TB/s).
template <typename P, typename H>
__global__ void __launch_bounds__(256)
gated_act_kernel(const P* __restrict__ pre, int64_t quads, int64_t quads_per_row, H* __restrict__ h, int act) {
    const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (q >= quads) return;
    const int64_t row = q / quads_per_row, c = (q - row * quads_per_row) * 4;
    const P* gate = pre + row * quads_per_row * 8 + (c / 32) * 64 + (c % 32);
    float g[4], u[4];
    load4<P>(gate, g);
    load4<P>(gate + 32, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = gate_act(g[j], act) * u[j];
    store4(h + q * 4, g);
}

// dpre = [dh * u * act'(g) | dh * act(g)], column-interleaved like pre.  Memory bound: reads 3, writes 2 values per hidden
// unit and token.  A CTA takes one block of 32 hidden units and kRowsPerChunk rows and also adds up its columns of dpre
// (the bias gradient) in fp32, in a fixed order; sum_chunks_kernel adds the chunks in order, so results repeat bit by bit.
// kPlanes: dpre goes to its planes instead, the operand of both gradients' products (8192 x 4096 fp32, 805 MB: 157 us, 5.1 TB/s;
// a bank-conflict-free turn through shared memory between).
template <typename P, typename H, bool kPlanes>
__global__ void __launch_bounds__(256)
gated_act_backward_kernel(const P* __restrict__ pre, const H* __restrict__ dh, int64_t m, int64_t hidden,
                          H* __restrict__ dpre, float* __restrict__ partial, int act,
                          __nv_bfloat16* __restrict__ planes) {
    const int64_t blocks = hidden / 32;
    const int64_t chunk = blockIdx.x / blocks, block = blockIdx.x - chunk * blocks;
    const int lane8 = threadIdx.x & 7, row32 = threadIdx.x >> 3;
    const int64_t end = min(m, (chunk + 1) * kRowsPerChunk);
    float sum_g[4] = {0.f, 0.f, 0.f, 0.f}, sum_u[4] = {0.f, 0.f, 0.f, 0.f};
    __shared__ float turned[kPlanes ? 64 : 1][33];  // 32 rows of the CTA's columns of dpre
    for (int64_t row = chunk * kRowsPerChunk + row32; row - row32 < end; row += 32) {
        const int64_t at = row * 2 * hidden + block * 64 + lane8 * 4;
        float g[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
        if (row < end) {
            float d[4];
            load4<P>(pre + at, g);
            load4<P>(pre + at + 32, u);
            load4<H>(dh + row * hidden + block * 32 + lane8 * 4, d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float value, slope;
                gate_act_grad(g[j], act, value, slope);
                g[j] = d[j] * u[j] * slope;
                u[j] = d[j] * value;
                sum_g[j] += g[j];
                sum_u[j] += u[j];
            }
            if (!kPlanes) {
                store4(dpre + at, g);
                store4(dpre + at + 32, u);
            }
        }
        if (kPlanes) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                turned[lane8 * 4 + j][row32] = g[j];
                turned[32 + lane8 * 4 + j][row32] = u[j];
            }
            __syncthreads();
            const int64_t pitch = plane_pitch(m), t = row - row32 + (threadIdx.x & 3) * 8, c = threadIdx.x >> 2;
            if (t < pitch)
                store_planes(turned[c] + (threadIdx.x & 3) * 8, planes + (block * 64 + c) * pitch + t, 2 * hidden * pitch);
            __syncthreads();
        }
    }
    if (partial == nullptr) return;
    __shared__ float sums[32][64];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        sums[row32][lane8 * 4 + j] = sum_g[j];
        sums[row32][32 + lane8 * 4 + j] = sum_u[j];
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) s += sums[r][threadIdx.x];
        partial[chunk * 2 * hidden + block * 64 + threadIdx.x] = s;
    }
}

__global__ void __launch_bounds__(256)
sum_chunks_kernel(const float* __restrict__ partial, int64_t chunks, int64_t cols, float* __restrict__ out) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.f;
    for (int64_t i = 0; i < chunks; ++i) s += partial[i * cols + c];
    out[c] = s;
}

// Few tokens: h straight from the stored fp32 blocks, exact fp32 products, no weight images.  Bound by reading the
// blocks (4 KiB each) once.  A cluster of `parts` CTAs takes one block-row of hidden units; in each CTA warps 0-3 walk the
// gate's blocks, 4-7 the up projection's, a block per warp and step.  data[slot][c][r]: lane (q, r4) of a warp holds the
// four outputs r = 4 r4 ... of the inputs c = 8 q ... 8 q + 7.  Every warp has a ring of its own in shared memory, filled by
// cp.async (16 bytes per lane, a lane reads back the weights it copied itself) kStages - 1 blocks ahead, because a warp that
// waits for its block before it asks for the next keeps only 4 KiB in flight.  The four q, the warps and the CTAs of the
// cluster (through distributed shared memory) are added up at the end in a fixed order.
// 4096 -> 8192 at density 0.25, 8 tokens, 67 MB of blocks: 16.0 us, 4.2 TB/s; the first and last 4 us are launch, the chain from row
// to index to block, and the sums (1024 -> 2048 at 0.5, one token, 8 MB: 4.1 us).
constexpr int kSmallStages = 3;

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename X, int kTok>
struct SmallSmem {
    static constexpr int kXBytes = kTok * 32 * (int)sizeof(X);  // a block's inputs, [token][32]
    static constexpr int kStage = 4096 + kXBytes;
    static constexpr int kRing = kSmallStages * kStage;         // per warp
    static constexpr int kTotal = 8 * kRing;                    // at the end [8 warps][kTok][32] fp32 and [2][kTok][32]
    static_assert(kTotal >= (8 + 2) * kTok * 128, "the sums reuse the rings");
};

// How a warp multiplies a block with its tokens' inputs, and where its sums lie.  Weights in the ring: row c at c * 128, its
// 16-byte piece r4 at position r4 ^ (2 (c / 8)), so that the four c / 8 of a quarter-warp's loads never share a bank.
//
// CUDA cores, exact fp32: acc[t][j] of lane (q, r4) belongs to output 4 r4 + j and this lane's inputs 8 q ... 8 q + 7.
template <typename X, int kTok>
struct SmallFma {
    float acc[kTok][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < kTok; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
    }
    __device__ __forceinline__ void block(const float4 (&w)[8], const X* xs, int nt, int lane) {
        const X* mine = xs + (lane & 3) * 8;
#pragma unroll
        for (int t = 0; t < kTok; ++t) {
            if (t < nt) {
                float xv[8];
                load8(mine + t * 32, xv);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    acc[t][0] = fmaf(w[j].x, xv[j], acc[t][0]);
                    acc[t][1] = fmaf(w[j].y, xv[j], acc[t][1]);
                    acc[t][2] = fmaf(w[j].z, xv[j], acc[t][2]);
                    acc[t][3] = fmaf(w[j].w, xv[j], acc[t][3]);
                }
            }
        }
    }
    __device__ __forceinline__ void store(float* sums, int lane) {  // [kTok][32]
#pragma unroll
        for (int t = 0; t < kTok; ++t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[t][j] += __shfl_xor_sync(0xffffffffu, acc[t][j], 1);
                acc[t][j] += __shfl_xor_sync(0xffffffffu, acc[t][j], 2);
            }
            if ((lane & 3) == 0)
                *reinterpret_cast<float4*>(sums + t * 32 + (lane >> 2) * 4) = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
        }
    }
};
// Tensor cores, bf16 inputs: the block transposed is the 32 x 32 left operand of mma.m16n8k16, eight tokens the right one.
// A weight is the sum of three bf16 values exactly, so that every product is exact and only the fp32 sums round, as with
// fused multiply-adds.  Rows of a fragment are outputs 4 r4 + 2 i, + 1 and its contraction indices this lane's
// inputs 8 q + 4 s ... + 3 (both operands permuted alike): the lane already holds them.
template <int kTok>
struct SmallMma {
    float acc[kTok / 8][2][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < kTok / 8; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
    }
    __device__ __forceinline__ void block(const float4 (&w)[8], const __nv_bfloat16* xs, int nt, int lane) {
        uint4 b[kTok / 8];
#pragma unroll
        for (int n = 0; n < kTok / 8; ++n) b[n] = *reinterpret_cast<const uint4*>(xs + (n * 8 + (lane >> 2)) * 32 + (lane & 3) * 8);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint32_t low[4][3], high[4][3];  // output 4 r4 + e: pairs of inputs 4 s, 4 s + 1 and 4 s + 2, 4 s + 3
            split3_bf16x2(w[4 * s].x, w[4 * s + 1].x, low[0]);
            split3_bf16x2(w[4 * s].y, w[4 * s + 1].y, low[1]);
            split3_bf16x2(w[4 * s].z, w[4 * s + 1].z, low[2]);
            split3_bf16x2(w[4 * s].w, w[4 * s + 1].w, low[3]);
            split3_bf16x2(w[4 * s + 2].x, w[4 * s + 3].x, high[0]);
            split3_bf16x2(w[4 * s + 2].y, w[4 * s + 3].y, high[1]);
            split3_bf16x2(w[4 * s + 2].z, w[4 * s + 3].z, high[2]);
            split3_bf16x2(w[4 * s + 2].w, w[4 * s + 3].w, high[3]);
#pragma unroll
            for (int n = 0; n < kTok / 8; ++n) {
                const uint32_t b0 = s == 0 ? b[n].x : b[n].z, b1 = s == 0 ? b[n].y : b[n].w;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int part = 0; part < 3; ++part)
                        mma16816(acc[n][i], low[2 * i][part], low[2 * i + 1][part], high[2 * i][part], high[2 * i + 1][part], b0, b1);
            }
        }
    }
    __device__ __forceinline__ void store(float* sums, int lane) {
        const int r = (lane >> 2) * 4, t = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < kTok / 8; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float* to = sums + (n * 8 + t) * 32 + r + 2 * i;
                *reinterpret_cast<float2*>(to) = make_float2(acc[n][i][0], acc[n][i][2]);
                *reinterpret_cast<float2*>(to + 32) = make_float2(acc[n][i][1], acc[n][i][3]);
            }
    }
};

template <typename X, typename H, int kTok, typename Math>
__global__ void __launch_bounds__(256)
gated_small_kernel(const X* __restrict__ x, int64_t m, int64_t k, const int32_t* __restrict__ ptr,
                   const int2* __restrict__ idx, const float* __restrict__ data, int64_t hidden,
                   const float* __restrict__ bias, H* __restrict__ h, int act, int parts) {
    using S = SmallSmem<X, kTok>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, r4 = lane >> 2;
    const int64_t block = blockIdx.x / parts, t0 = (int64_t)blockIdx.y * kTok;
    const int part = (int)(blockIdx.x % parts);
    const int nt = (int)min((int64_t)kTok, m - t0);
    const int64_t row = 2 * block + (warp >> 2);
    const int begin = ptr[row] + part * 4 + (warp & 3), stride = 4 * parts;
    const int count = max(0, (ptr[row + 1] - begin + stride - 1) / stride);
    uint8_t* ring = smem + warp * S::kRing;
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
    const int place = ((r4 ^ (2 * q)) << 4) + q * 1024;  // of this lane's first piece in a stage

    int2 ents = make_int2(0, 0);  // entry i of this warp is held by lane i mod 32
    auto issue = [&](int i) {
        if (i < count) {
            if ((i & 31) == 0) ents = i + lane < count ? __ldg(idx + begin + (i + lane) * stride) : make_int2(0, 0);
            const int col = __shfl_sync(0xffffffffu, ents.x, i & 31), slot = __shfl_sync(0xffffffffu, ents.y, i & 31);
            const uint32_t stage = ring_addr + (i % kSmallStages) * S::kStage;
            const float* w = data + (int64_t)slot * kBlockElems + q * 256 + r4 * 4;
#pragma unroll
            for (int j = 0; j < 8; ++j) copy16(stage + place + j * 128, w + j * 32);
            constexpr int kPieces = S::kXBytes / kTok / 16;  // of a token
#pragma unroll
            for (int piece = lane; piece < kTok * kPieces; piece += 32) {
                const int t = piece / kPieces, o = piece % kPieces;
                if (t < nt)
                    copy16(stage + 4096 + piece * 16, reinterpret_cast<const uint8_t*>(x + (t0 + t) * k + (int64_t)col * 32) + o * 16);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    Math math;
    math.clear();
#pragma unroll
    for (int i = 0; i < kSmallStages - 1; ++i) issue(i);
    for (int i = 0; i < count; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kSmallStages - 2) : "memory");
        __syncwarp();  // every lane's part of the block's inputs has arrived, and the stage of the next copy has been read
        issue(i + kSmallStages - 1);
        const uint8_t* stage = ring + (i % kSmallStages) * S::kStage;
        float4 w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const float4*>(stage + place + j * 128);
        math.block(w, reinterpret_cast<const X*>(stage + 4096), nt, lane);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the rings have been read: their memory takes the sums
    float* sums = reinterpret_cast<float*>(smem);
    math.store(sums + warp * kTok * 32, lane);
    __syncthreads();
    float* both = sums + 8 * kTok * 32;  // this CTA's sums: [gate, up][kTok][32]
    for (int i = threadIdx.x; i < 2 * kTok * 32; i += 256) {
        const float* s = sums + (i / (kTok * 32)) * 4 * kTok * 32 + i % (kTok * 32);
        both[i] = s[0] + s[kTok * 32] + s[2 * kTok * 32] + s[3 * kTok * 32];
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (parts > 1) cluster.sync(); else __syncthreads();
    // the cluster's CTAs share the outputs among them
    for (int i = part * 256 + threadIdx.x; i < nt * 32; i += parts * 256) {
        float g = 0.f, u = 0.f;
        for (int c = 0; c < parts; ++c) {
            const float* theirs = parts > 1 ? cluster.map_shared_rank(both, c) : both;
            g += theirs[i];
            u += theirs[kTok * 32 + i];
        }
        const int t = i >> 5, r = i & 31;
        if (bias != nullptr) {
            g += bias[block * 64 + r];
            u += bias[block * 64 + 32 + r];
        }
        h[(t0 + t) * hidden + block * 32 + r] = from_float<H>(gate_act(g, act) * u);
    }
    if (parts > 1) cluster.sync();  // nobody leaves while its sums are read
}

template <typename X, typename H, int kTok, typename Math>
cudaError_t small(const void* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx, const float* data, int64_t nnz,
                  int64_t hidden, const float* bias, void* h, int act, cudaStream_t stream) {
    constexpr int kBytes = SmallSmem<X, kTok>::kTotal;
    constexpr int kMaxDevices = 64;
    static bool ready[kMaxDevices] = {false};  // the attribute is per device; threads racing on the first call set it twice
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (!ready[dev]) {
        err = cudaFuncSetAttribute(gated_small_kernel<X, H, kTok, Math>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (err != cudaSuccess) return err;
        ready[dev] = true;
    }
    const int64_t rows = hidden / 32, tiles = (m + kTok - 1) / kTok;
    if (tiles > 65535) return cudaErrorInvalidValue;
    // CTAs per block-row: as many as the SMs hold at one each, while every warp has a block of its own.  1, 2, 4, 8 CTAs, us, bf16,
    // 8 tokens: 1024 -> 512 at density 0.5 (16 rows) 5.4, 5.0, 4.4, 4.7; 4096 -> 1024 (32 rows) 13.7, 10.2, 8.6, 9.0; 1024 -> 2048
    // (64 rows) 6.0, 5.4, 5.8, 9.3; 1024 -> 4096 (128 rows) 8.0, 9.0, 12.8, 21.8; 4096 -> 8192 at 0.25 (256 rows) 16.6, 20.9, 27, 45
    int parts = 1;
    while (parts < 8 && rows * tiles * parts * 2 <= 148 && nnz / rows >= parts * 2 * 8) parts *= 2;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * parts), (unsigned)tiles);
    config.blockDim = dim3(256);
    config.dynamicSmemBytes = kBytes;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, gated_small_kernel<X, H, kTok, Math>, static_cast<const X*>(x), m, k, ptr,
                              reinterpret_cast<const int2*>(idx), data, hidden, bias, static_cast<H*>(h), act, parts);
}

// Tokens per pass over the blocks.  bf16, CUDA cores / tensor cores, us: 1024 -> 2048 at density 0.5, one token 4.6 / 5.5, two 4.9 /
// 5.5, four 5.3 / 5.5, eight 6.9 / 6.0; 4096 -> 8192 at 0.25: 9.4 / 12.6, 10.6 / 12.6, 12.4 / 12.6, 17.9 / 12.8 (blocks in L2).
template <typename H>
cudaError_t small_fp32(const void* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx, const float* data,
                       int64_t nnz, int64_t hidden, const float* bias, void* h, int act, cudaStream_t stream) {
    if (m == 1) return small<float, H, 1, SmallFma<float, 1>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
    if (m <= 4) return small<float, H, 4, SmallFma<float, 4>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
    return small<float, H, 8, SmallFma<float, 8>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
}

template <typename H>
cudaError_t small_bf16(const void* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx, const float* data,
                       int64_t nnz, int64_t hidden, const float* bias, void* h, int act, cudaStream_t stream) {
    using X = __nv_bfloat16;
    if (m == 1) return small<X, H, 1, SmallFma<X, 1>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
    if (m <= 4) return small<X, H, 4, SmallFma<X, 4>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
    if (m <= 8) return small<X, H, 8, SmallMma<8>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
    if (m <= 16) return small<X, H, 16, SmallMma<16>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
    return small<X, H, 32, SmallMma<32>>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
}

template <typename P, typename H>
cudaError_t act_forward(const void* pre, int64_t m, int64_t hidden, void* h, int act, cudaStream_t stream) {
    const int64_t quads = m * hidden / 4;
    gated_act_kernel<P, H><<<(unsigned)((quads + 255) / 256), 256, 0, stream>>>(static_cast<const P*>(pre), quads, hidden / 4,
                                                                                static_cast<H*>(h), act);
    return cudaGetLastError();
}

template <typename P, typename H, bool kPlanes = false>
cudaError_t act_backward(const void* pre, const void* dh, int64_t m, int64_t hidden, void* dpre, float* partial, int act,
                         unsigned grid, cudaStream_t stream, void* planes = nullptr) {
    gated_act_backward_kernel<P, H, kPlanes><<<grid, 256, 0, stream>>>(
        static_cast<const P*>(pre), static_cast<const H*>(dh), m, hidden, static_cast<H*>(dpre), partial, act,
        static_cast<__nv_bfloat16*>(planes));
    return cudaGetLastError();
}

int64_t row_chunks(int64_t m) { return (m + kRowsPerChunk - 1) / kRowsPerChunk; }

}  // namespace

cudaError_t launch_gated_act(const void* pre, int64_t m, int64_t hidden, void* h, int act, bool pre_bf16, bool io_bf16,
                             cudaStream_t stream) {
    if (m == 0 || hidden == 0) return cudaSuccess;
    if (m * hidden / 4 / 256 >= 0x7fffffffll) return cudaErrorInvalidValue;
    if (!io_bf16) return act_forward<float, float>(pre, m, hidden, h, act, stream);
    return pre_bf16 ? act_forward<__nv_bfloat16, __nv_bfloat16>(pre, m, hidden, h, act, stream)
                    : act_forward<float, __nv_bfloat16>(pre, m, hidden, h, act, stream);
}

int64_t gated_act_workspace_bytes(int64_t m, int64_t hidden) { return row_chunks(m) * 2 * hidden * 4; }

cudaError_t launch_gated_act_backward(const void* pre, const void* dh, int64_t m, int64_t hidden, void* dpre,
                                      float* dbias, float* workspace, int act, bool pre_bf16, bool io_bf16,
                                      void* planes, cudaStream_t stream) {
    if (hidden == 0) return cudaSuccess;
    if (m > 0) {
        const int64_t ctas = row_chunks(m) * (hidden / 32);
        if (ctas >= 0x7fffffffll) return cudaErrorInvalidValue;
        float* partial = dbias != nullptr ? workspace : nullptr;
        const unsigned grid = (unsigned)ctas;
        const cudaError_t err =
            !io_bf16 && planes != nullptr ? act_backward<float, float, true>(pre, dh, m, hidden, dpre, partial, act, grid, stream, planes)
            : !io_bf16 ? act_backward<float, float>(pre, dh, m, hidden, dpre, partial, act, grid, stream)
            : pre_bf16 ? act_backward<__nv_bfloat16, __nv_bfloat16>(pre, dh, m, hidden, dpre, partial, act, grid, stream)
                       : act_backward<float, __nv_bfloat16>(pre, dh, m, hidden, dpre, partial, act, grid, stream);
        if (err != cudaSuccess) return err;
    }
    if (dbias == nullptr) return cudaSuccess;
    sum_chunks_kernel<<<(unsigned)((2 * hidden + 255) / 256), 256, 0, stream>>>(workspace, row_chunks(m), 2 * hidden, dbias);
    return cudaGetLastError();
}

cudaError_t launch_gated_small(const void* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx,
                               const float* data, int64_t nnz, int64_t hidden, const float* bias, void* h, int act,
                               bool x_bf16, bool h_bf16, cudaStream_t stream) {
    if (m == 0 || hidden == 0) return cudaSuccess;
    if (hidden / 32 * 8 > 0x7fffffffll) return cudaErrorInvalidValue;
    if (!x_bf16) return small_fp32<float>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
    return h_bf16 ? small_bf16<__nv_bfloat16>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream)
                  : small_bf16<float>(x, m, k, ptr, idx, data, nnz, hidden, bias, h, act, stream);
}

}  // namespace bsmm

// The gated feed-forward block's own arithmetic, h = act(g) * u with g = x Wg^T + bg and u = x Wu^T + bu, around
// pre-activations whose columns alternate in blocks of 32: columns 64 j ... 64 j + 31 of `pre` [m, 2 hidden] are g of the
// hidden units 32 j ... 32 j + 31, the next 32 their u.  (Wg and Wu are one block-sparse matrix of 2 hidden rows whose
// block-rows alternate the same way, so one product computes `pre`, and the gradients with respect to the input and to
// both weights are one product each.)
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"

namespace bsmm {
namespace {

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

// Memory bound: reads 2, writes 1 value per hidden unit and token.
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
template <typename P, typename H>
__global__ void __launch_bounds__(256)
gated_act_backward_kernel(const P* __restrict__ pre, const H* __restrict__ dh, int64_t m, int64_t hidden,
                          H* __restrict__ dpre, float* __restrict__ partial, int act) {
    const int64_t blocks = hidden / 32;
    const int64_t chunk = blockIdx.x / blocks, block = blockIdx.x - chunk * blocks;
    const int lane8 = threadIdx.x & 7, row32 = threadIdx.x >> 3;
    const int64_t end = min(m, (chunk + 1) * kRowsPerChunk);
    float sum_g[4] = {0.f, 0.f, 0.f, 0.f}, sum_u[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t row = chunk * kRowsPerChunk + row32; row < end; row += 32) {
        const int64_t at = row * 2 * hidden + block * 64 + lane8 * 4;
        float g[4], u[4], d[4];
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
        store4(dpre + at, g);
        store4(dpre + at + 32, u);
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
// blocks (4 KiB each) once.  A CTA takes one block-row of hidden units: warps 0-3 walk the gate's blocks, 4-7 the up
// projection's.  data[slot][c][r]: lane (q, r4) of a warp holds the four outputs r = 4 r4 ... of the inputs c = 8 q ... 8 q + 7
// of a block, so that it loads eight 16-byte pieces of weights (each warp load covers four 128-byte rows) and eight
// consecutive inputs of a token; the four q and four warps are added up at the end, in a fixed order.
constexpr int kSmallTokens = 8;

template <typename X, typename H>
__global__ void __launch_bounds__(256, 2)
gated_small_kernel(const X* __restrict__ x, int64_t m, int64_t k, const int32_t* __restrict__ ptr,
                   const int2* __restrict__ idx, const float* __restrict__ data, int64_t hidden,
                   const float* __restrict__ bias, H* __restrict__ h, int act) {
    __shared__ float sums[8][kSmallTokens][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane >> 3, r4 = lane & 7;
    const int64_t block = blockIdx.x, t0 = (int64_t)blockIdx.y * kSmallTokens;
    const int nt = (int)min((int64_t)kSmallTokens, m - t0);
    const int64_t row = 2 * block + (warp >> 2);
    float acc[kSmallTokens][4];
#pragma unroll
    for (int t = 0; t < kSmallTokens; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][j] = 0.f;
    const int end = ptr[row + 1];
    for (int e = ptr[row] + (warp & 3); e < end; e += 4) {
        const int2 entry = __ldg(idx + e);
        const float4* w4 = reinterpret_cast<const float4*>(data + (int64_t)entry.y * kBlockElems + q * 256) + r4;
        float4 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __ldg(w4 + i * 8);
        const X* xe = x + t0 * k + (int64_t)entry.x * 32 + q * 8;
#pragma unroll
        for (int t = 0; t < kSmallTokens; ++t) {
            if (t < nt) {
                float xv[8];
                load8(xe + t * k, xv);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    acc[t][0] = fmaf(w[i].x, xv[i], acc[t][0]);
                    acc[t][1] = fmaf(w[i].y, xv[i], acc[t][1]);
                    acc[t][2] = fmaf(w[i].z, xv[i], acc[t][2]);
                    acc[t][3] = fmaf(w[i].w, xv[i], acc[t][3]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kSmallTokens; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[t][j] += __shfl_xor_sync(0xffffffffu, acc[t][j], 8);
            acc[t][j] += __shfl_xor_sync(0xffffffffu, acc[t][j], 16);
        }
        if (q == 0) *reinterpret_cast<float4*>(&sums[warp][t][r4 * 4]) = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
    }
    __syncthreads();
    const int t = threadIdx.x >> 5;  // one output per thread
    if (t < nt) {
        float g = sums[0][t][lane] + sums[1][t][lane] + sums[2][t][lane] + sums[3][t][lane];
        float u = sums[4][t][lane] + sums[5][t][lane] + sums[6][t][lane] + sums[7][t][lane];
        if (bias != nullptr) {
            g += bias[block * 64 + lane];
            u += bias[block * 64 + 32 + lane];
        }
        h[(t0 + t) * hidden + block * 32 + lane] = from_float<H>(gate_act(g, act) * u);
    }
}

template <typename P, typename H>
cudaError_t act_forward(const void* pre, int64_t m, int64_t hidden, void* h, int act, cudaStream_t stream) {
    const int64_t quads = m * hidden / 4;
    gated_act_kernel<P, H><<<(unsigned)((quads + 255) / 256), 256, 0, stream>>>(static_cast<const P*>(pre), quads, hidden / 4,
                                                                                static_cast<H*>(h), act);
    return cudaGetLastError();
}

template <typename P, typename H>
cudaError_t act_backward(const void* pre, const void* dh, int64_t m, int64_t hidden, void* dpre, float* partial, int act,
                         unsigned grid, cudaStream_t stream) {
    gated_act_backward_kernel<P, H><<<grid, 256, 0, stream>>>(static_cast<const P*>(pre), static_cast<const H*>(dh), m, hidden,
                                                              static_cast<H*>(dpre), partial, act);
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
                                      cudaStream_t stream) {
    if (hidden == 0) return cudaSuccess;
    if (m > 0) {
        const int64_t ctas = row_chunks(m) * (hidden / 32);
        if (ctas >= 0x7fffffffll) return cudaErrorInvalidValue;
        float* partial = dbias != nullptr ? workspace : nullptr;
        const unsigned grid = (unsigned)ctas;
        const cudaError_t err =
            !io_bf16 ? act_backward<float, float>(pre, dh, m, hidden, dpre, partial, act, grid, stream)
            : pre_bf16 ? act_backward<__nv_bfloat16, __nv_bfloat16>(pre, dh, m, hidden, dpre, partial, act, grid, stream)
                       : act_backward<float, __nv_bfloat16>(pre, dh, m, hidden, dpre, partial, act, grid, stream);
        if (err != cudaSuccess) return err;
    }
    if (dbias == nullptr) return cudaSuccess;
    sum_chunks_kernel<<<(unsigned)((2 * hidden + 255) / 256), 256, 0, stream>>>(workspace, row_chunks(m), 2 * hidden, dbias);
    return cudaGetLastError();
}

cudaError_t launch_gated_small(const void* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx,
                               const float* data, int64_t hidden, const float* bias, void* h, int act, bool x_bf16,
                               bool h_bf16, cudaStream_t stream) {
    if (m == 0 || hidden == 0) return cudaSuccess;
    const int64_t tiles = (m + kSmallTokens - 1) / kSmallTokens;
    if (tiles > 65535 || hidden / 32 > 0x7fffffffll) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)(hidden / 32), (unsigned)tiles);
    const int2* idx2 = reinterpret_cast<const int2*>(idx);
    if (x_bf16) {
        const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(x);
        if (h_bf16)
            gated_small_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, stream>>>(
                xb, m, k, ptr, idx2, data, hidden, bias, static_cast<__nv_bfloat16*>(h), act);
        else
            gated_small_kernel<__nv_bfloat16, float><<<grid, 256, 0, stream>>>(xb, m, k, ptr, idx2, data, hidden, bias,
                                                                               static_cast<float*>(h), act);
    } else {
        gated_small_kernel<float, float><<<grid, 256, 0, stream>>>(static_cast<const float*>(x), m, k, ptr, idx2, data, hidden,
                                                                   bias, static_cast<float*>(h), act);
    }
    return cudaGetLastError();
}

}  // namespace bsmm

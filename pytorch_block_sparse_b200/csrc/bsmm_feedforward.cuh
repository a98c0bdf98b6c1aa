// Shared declarations of the operators around a block-sparse projection: the gated feed-forward block, dropout with the
// residual add, and low-rank adapters.
#pragma once
#include <cuda_bf16.h>

#include "bsmm_common.cuh"

namespace bsmm {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// eight consecutive values, 16-byte aligned
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint32_t pack_bf16x2(float low, float high) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    unpack8(*reinterpret_cast<const uint4*>(p), v);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// w = parts[0] + parts[1] + parts[2] exactly (3 x 8 significant bits), for a pair of values
__device__ __forceinline__ void split3_bf16x2(float w0, float w1, uint32_t (&parts)[3]) {
    asm("{\n\t.reg .b16 h0, h1, m1;\n\t.reg .f32 d0, d1;\n\t"
        "mov.b16 m1, 0xBF80;\n\t"
        "cvt.rn.bf16x2.f32 %0, %4, %3;\n\t"
        "mov.b32 {h0, h1}, %0;\n\t"
        "fma.rn.f32.bf16 d0, h0, m1, %3;\n\t"
        "fma.rn.f32.bf16 d1, h1, m1, %4;\n\t"
        "cvt.rn.bf16x2.f32 %1, d1, d0;\n\t"
        "mov.b32 {h0, h1}, %1;\n\t"
        "fma.rn.f32.bf16 d0, h0, m1, d0;\n\t"
        "fma.rn.f32.bf16 d1, h1, m1, d1;\n\t"
        "cvt.rn.bf16x2.f32 %2, d1, d0;\n\t}"
        : "=&r"(parts[0]), "=&r"(parts[1]), "=r"(parts[2])
        : "f"(w0), "f"(w1));
}

// Planes: an fp32 matrix [tokens][features] as three bf16 matrices [features][pitch] that add up to it exactly.
__host__ __device__ constexpr int64_t plane_pitch(int64_t tokens) { return (tokens + 7) / 8 * 8; }  // rows of whole 16-byte pieces
// eight consecutive tokens of a feature to the three planes, `plane` elements apart
__device__ __forceinline__ void store_planes(const float* v, __nv_bfloat16* to, int64_t plane) {
    uint32_t parts[4][3];
#pragma unroll
    for (int j = 0; j < 4; ++j) split3_bf16x2(v[2 * j], v[2 * j + 1], parts[j]);
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(to + q * plane) = make_uint4(parts[0][q], parts[1][q], parts[2][q], parts[3][q]);
}

// the same as loaded, not yet widened: what a thread holds while loads are in flight
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ void load_pieces(const uint8_t* p, int pitch) {  // 16-byte pieces `pitch` bytes apart
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + pitch);
    }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <>
struct Raw8<__nv_bfloat16> {
    uint4 a;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void load_pieces(const uint8_t* p, int) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const { unpack8(a, v); }
};

// The gate's activation, in fp32.  kind: 0 SiLU g / (1 + exp(-g)), 1 GELU (erf form).
__device__ __forceinline__ float gate_act(float g, int kind) {
    if (kind == 0) return g / (1.f + expf(-g));
    return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
}
// value and derivative
__device__ __forceinline__ void gate_act_grad(float g, int kind, float& value, float& slope) {
    if (kind == 0) {
        const float s = 1.f / (1.f + expf(-g));
        value = g * s;
        slope = s * (1.f + g * (1.f - s));
    } else {
        const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        value = g * cdf;
        slope = cdf + g * expf(-0.5f * g * g) * 0.39894228040143268f;
    }
}

// launchers
cudaError_t launch_dropout(const void* x, const void* residual, void* out, int64_t n, uint32_t cut, const int64_t* rng,
                           bool bf16, cudaStream_t stream);
cudaError_t launch_rng_next(int64_t* state, int64_t* used, cudaStream_t stream);

cudaError_t launch_gated_act(const void* pre, int64_t m, int64_t hidden, void* h, int act, bool pre_bf16, bool io_bf16,
                             cudaStream_t stream);
int64_t gated_act_workspace_bytes(int64_t m, int64_t hidden);
cudaError_t launch_gated_act_backward(const void* pre, const void* dh, int64_t m, int64_t hidden, void* dpre,
                                      float* dbias, float* workspace, int act, bool pre_bf16, bool io_bf16,
                                      void* planes, cudaStream_t stream);  // planes of dpre in its place, or null (fp32 only)
cudaError_t launch_gated_small(const void* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx,
                               const float* data, int64_t nnz, int64_t hidden, const float* bias, void* h, int act,
                               bool x_bf16, bool h_bf16, cudaStream_t stream);

// the tensor-core forward on bf16 tensors (bsmm_gated_umma.cu)
int64_t gated_plan_bytes(int64_t hidden, int64_t k, int64_t nnz);
int64_t gated_images_bytes(int64_t nnz);
cudaError_t launch_build_gated_plan(const int32_t* ptr, const int32_t* idx, int64_t hidden, int64_t k, void* plan,
                                    cudaStream_t stream);
cudaError_t launch_pack_pairs(const float* data, const void* plan, int64_t hidden, int64_t k, int64_t nnz, void* images,
                              cudaStream_t stream);
cudaError_t launch_gated_umma(const void* x, int64_t m, int64_t k, const void* plan, const void* images, int64_t hidden,
                              const float* bias, void* h, void* pre, int act, cudaStream_t stream);

// the forward pass of fp32 tensors from planes of three bf16 parts (bsmm_gated_f32.cu)
int64_t gated_f32_workspace_bytes(int64_t m, int64_t k, int64_t nnz);
cudaError_t launch_gated_f32(const float* x, int64_t m, int64_t k, const float* data, int64_t nnz, const int32_t* ptr,
                             const void* pairs_plan, int64_t hidden, const float* bias, float* h, float* pre, int act, void* workspace,
                             cudaStream_t stream);

// The rows' pairs in the plan of the weight gradient: a row's begin where its entries do in the CSR.
struct GatedPairs {
    const int4* pairs;       // (input block, gate slot, up slot, 0), a slot -1 where that projection has no block
    const int32_t* counts;   // per pair-row
};
GatedPairs gated_pairs(const void* plan, int64_t hidden, int64_t nnz);

// the weight gradient of fp32 tensors from planes of three bf16 parts (bsmm_gated_wgrad.cu)
int64_t gated_wgrad_plan_bytes(int64_t hidden, int64_t nnz);
cudaError_t launch_build_gated_wgrad_plan(const int32_t* ptr, const int32_t* idx, int64_t hidden, int64_t k, int64_t nnz, void* plan,
                                          cudaStream_t stream);
cudaError_t launch_split_planes(const float* x, int64_t m, int64_t k, void* planes, cudaStream_t stream);
int64_t gated_wgrad_workspace_bytes(int64_t hidden, int64_t nnz, int64_t tokens);
cudaError_t launch_gated_wgrad(const void* x_planes, const void* d_planes, int64_t tokens, int64_t k, int64_t hidden, int64_t nnz,
                               const void* plan, float* out, float* block_sumsq, void* workspace, cudaStream_t stream);

// the input gradient of fp32 tensors from the same planes (bsmm_gated_dgrad.cu)
int64_t gated_dgrad_plan_bytes(int64_t k, int64_t nnz);
cudaError_t launch_build_gated_dgrad_plan(const int32_t* col_ptr, const int32_t* col_idx, int64_t hidden, int64_t k, int64_t nnz, void* plan,
                                          cudaStream_t stream);
int64_t gated_dgrad_workspace_bytes(int64_t nnz);
cudaError_t launch_gated_dgrad(const void* d_planes, int64_t m, int64_t k, int64_t hidden, int64_t nnz, const float* data,
                               const int32_t* col_ptr, const void* plan, float* dx, void* workspace, cudaStream_t stream);

struct AdapterCall {
    const void* x;           // [tokens, inner]
    const void* down;        // [count, rank, inner], rank padded to a multiple of 16 with zero rows
    const void* up;          // [count, outer, rank]
    const float* scaling;    // [count]
    const int32_t* offsets;  // [requests + 1]
    const int32_t* ids;      // [requests]
    const void* base;        // [tokens, outer] or null (zeros); may be `out`
    void* out;               // [tokens, outer]
    float* workspace;
    int64_t tokens, inner, outer, requests, count, rank;
};
int64_t adapters_workspace_bytes(int64_t tokens, int64_t inner, int64_t rank);
// in_bf16: x, down and up; out_bf16: base and out
cudaError_t launch_adapters(const AdapterCall& call, bool in_bf16, bool out_bf16, cudaStream_t stream);

}  // namespace bsmm

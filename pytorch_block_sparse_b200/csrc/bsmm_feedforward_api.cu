// extern "C" entry points of the operators around a block-sparse projection: argument validation and launches.
#include "bsmm_feedforward.cuh"

namespace bsmm {
int report_cuda(cudaError_t err);  // bsmm_api.cu: status code, and the error bsmm_last_cuda_error returns
}

namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// rows x cols elements of at most 4 bytes stay addressable, and every product of sizes below fits 63 bits
bool too_large(int64_t rows, int64_t cols) { return rows > 0x7fffffffll || cols > 0x7fffffffll || (cols > 0 && rows > (1ll << 40) / cols); }

int gated_types(uint32_t flags) {
    if ((flags & ~(BSMM_GATED_GELU | BSMM_GATED_IO_BF16 | BSMM_GATED_PRE_BF16 | BSMM_GATED_X_BF16)) != 0) return BSMM_ERR_UNSUPPORTED;
    if ((flags & BSMM_GATED_PRE_BF16) != 0 && (flags & BSMM_GATED_IO_BF16) == 0) return BSMM_ERR_UNSUPPORTED;
    return BSMM_OK;
}

}  // namespace

extern "C" {

int bsmm_gated_act(const void* pre, int64_t m, int64_t hidden, void* h, uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (m < 0 || hidden < 0 || (hidden % 32) != 0) return BSMM_ERR_INVALID_ARGUMENT;
    const int status = gated_types(flags);
    if (status != BSMM_OK || (flags & BSMM_GATED_X_BF16) != 0) return BSMM_ERR_UNSUPPORTED;
    if (m == 0 || hidden == 0) return BSMM_OK;
    if (pre == nullptr || h == nullptr || !aligned(pre, 16) || !aligned(h, 16)) return BSMM_ERR_INVALID_ARGUMENT;
    if (too_large(m, 2 * hidden)) return BSMM_ERR_TOO_LARGE;
    return bsmm::report_cuda(bsmm::launch_gated_act(pre, m, hidden, h, (flags & BSMM_GATED_GELU) != 0,
                                                    (flags & BSMM_GATED_PRE_BF16) != 0, (flags & BSMM_GATED_IO_BF16) != 0,
                                                    static_cast<cudaStream_t>(stream)));
}

int64_t bsmm_gated_act_workspace_bytes(int64_t m, int64_t hidden) {
    if (m < 0 || hidden < 0 || too_large(m, 2 * hidden)) return -1;
    return bsmm::gated_act_workspace_bytes(m, hidden);
}

int bsmm_gated_act_backward(const void* pre, const void* dh, int64_t m, int64_t hidden, void* dpre, float* dbias,
                            void* workspace, uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (m < 0 || hidden < 0 || (hidden % 32) != 0) return BSMM_ERR_INVALID_ARGUMENT;
    const int status = gated_types(flags);
    if (status != BSMM_OK || (flags & BSMM_GATED_X_BF16) != 0) return BSMM_ERR_UNSUPPORTED;
    if (hidden == 0) return BSMM_OK;
    if (m > 0 && (pre == nullptr || dh == nullptr || dpre == nullptr || (dbias != nullptr && workspace == nullptr)))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (!aligned(pre, 16) || !aligned(dh, 16) || !aligned(dpre, 16) || !aligned(dbias, 4) || !aligned(workspace, 16))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (too_large(m, 2 * hidden)) return BSMM_ERR_TOO_LARGE;
    return bsmm::report_cuda(bsmm::launch_gated_act_backward(
        pre, dh, m, hidden, dpre, dbias, static_cast<float*>(workspace), (flags & BSMM_GATED_GELU) != 0,
        (flags & BSMM_GATED_PRE_BF16) != 0, (flags & BSMM_GATED_IO_BF16) != 0, nullptr, static_cast<cudaStream_t>(stream)));
}

int bsmm_gated_small(const void* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx, int64_t nnz,
                     const float* data, int64_t hidden, const float* bias, void* h, uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (m < 0 || k < 0 || hidden < 0 || nnz < 0 || (hidden % 32) != 0 || (k % 32) != 0) return BSMM_ERR_INVALID_ARGUMENT;
    if (gated_types(flags) != BSMM_OK || (flags & BSMM_GATED_PRE_BF16) != 0) return BSMM_ERR_UNSUPPORTED;
    if (m == 0 || hidden == 0) return BSMM_OK;
    if (ptr == nullptr || h == nullptr || (nnz > 0 && (x == nullptr || idx == nullptr || data == nullptr)))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (!aligned(x, 16) || !aligned(ptr, 4) || !aligned(idx, 8) || !aligned(data, 16) || !aligned(bias, 4) || !aligned(h, 16))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (nnz > 0x7fffffff || too_large(m, k) || too_large(m, hidden) || (m + 7) / 8 > 65535) return BSMM_ERR_TOO_LARGE;
    const bool io16 = (flags & BSMM_GATED_IO_BF16) != 0;
    return bsmm::report_cuda(bsmm::launch_gated_small(x, m, k, ptr, idx, data, nnz, hidden, bias, h, (flags & BSMM_GATED_GELU) != 0,
                                                      io16 || (flags & BSMM_GATED_X_BF16) != 0, io16,
                                                      static_cast<cudaStream_t>(stream)));
}

// The fp32-class precisions multiply planes of bf16 parts.
static bool from_planes(int64_t nnz, uint32_t precision) {
    return nnz > 0 && (precision == BSMM_PREC_TF32X3 || precision == BSMM_PREC_BF16X3);
}
static int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int64_t bsmm_gated_forward_workspace_bytes(int64_t m, int64_t k, int64_t hidden, int64_t nnz, uint32_t flags) {
    if (m < 0 || k < 0 || hidden < 0 || nnz < 0 || nnz > 0x7fffffff || too_large(m, k)) return -1;
    return from_planes(nnz, flags & BSMM_PREC_MASK) ? bsmm::gated_f32_workspace_bytes(m, k, nnz) : 0;
}

int bsmm_gated_pass_forward(const float* x, int64_t m, int64_t k, const int32_t* ptr, const int32_t* idx, int64_t nnz,
                            const float* data, void* packed, const void* plan, const void* f32_plan, int64_t hidden,
                            const float* bias, float* pre, void* h, void* workspace, uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    const uint32_t precision = flags & BSMM_PREC_MASK, pass = (flags >> 16) & 0xFu;
    if ((flags & ~(BSMM_PREC_MASK | BSMM_DSD_GROUP(0xFF) | BSMM_GATED_PASS(0xF))) != 0 || (pass & BSMM_GATED_PRE_BF16) != 0)
        return BSMM_ERR_UNSUPPORTED;
    if (f32_plan != nullptr && pass == (pass & BSMM_GATED_GELU) && from_planes(nnz, precision)) {
        if (m < 0 || k <= 0 || hidden < 0 || (hidden % 32) != 0 || (k % 32) != 0) return BSMM_ERR_INVALID_ARGUMENT;
        if (m == 0 || hidden == 0) return BSMM_OK;
        if (x == nullptr || ptr == nullptr || data == nullptr || h == nullptr || workspace == nullptr) return BSMM_ERR_INVALID_ARGUMENT;
        if (!aligned(x, 16) || !aligned(ptr, 4) || !aligned(data, 16) || !aligned(f32_plan, 16) || !aligned(bias, 16) ||
            !aligned(pre, 16) || !aligned(h, 16) || !aligned(workspace, 256))
            return BSMM_ERR_INVALID_ARGUMENT;
        if (nnz > 0x7fffffff || k > BSMM_GATED_MAX_K || too_large(m, k) || too_large(m, 2 * hidden)) return BSMM_ERR_TOO_LARGE;
        return bsmm::report_cuda(bsmm::launch_gated_f32(x, m, k, data, nnz, ptr, f32_plan, hidden, bias, static_cast<float*>(h), pre,
                                                        (pass & BSMM_GATED_GELU) != 0, workspace, static_cast<cudaStream_t>(stream)));
    }
    if (pre == nullptr && m > 0 && hidden > 0) return BSMM_ERR_INVALID_ARGUMENT;
    if (precision != BSMM_PREC_FP32_SIMT) {
        const int status = bsmm_pack_weights(data, nnz, precision, packed, nullptr, stream);
        if (status != BSMM_OK) return status;
    }
    const int status = bsmm_dsd(x, m, k, ptr, idx, nnz, data, packed, plan, 2 * hidden, pre, bias,
                                flags & (BSMM_PREC_MASK | BSMM_DSD_GROUP(0xFF)), stream);
    return status != BSMM_OK ? status : bsmm_gated_act(pre, m, hidden, h, pass, stream);
}

// [planes of x][planes of dpre][the bias gradient's partial sums and the weight gradient's: one after the other, in the same memory]
int64_t bsmm_gated_backward_workspace_bytes(int64_t m, int64_t k, int64_t hidden, int64_t nnz, uint32_t flags) {
    const uint32_t precision = flags & BSMM_PREC_MASK;
    const int64_t a = bsmm_gated_act_workspace_bytes(m, hidden);
    if (k < 0 || too_large(m, k) || nnz < 0 || nnz > 0x7fffffff) return -1;
    if (a >= 0 && m > 0 && from_planes(nnz, precision)) {
        const int64_t b = bsmm::gated_wgrad_workspace_bytes(hidden, nnz, m), c = bsmm::gated_dgrad_workspace_bytes(nnz);
        return padded(6 * bsmm::plane_pitch(m) * k) + padded(12 * bsmm::plane_pitch(m) * hidden) + (a > b ? (a > c ? a : c) : b > c ? b : c);
    }
    const int64_t b = bsmm_sddmm_workspace_bytes(2 * hidden, k, m, nnz, precision);
    return a < 0 || b < 0 ? -1 : a > b ? a : b;
}

int64_t bsmm_gated_f32_plan_bytes(int64_t hidden, int64_t k, int64_t nnz) {
    if (bsmm_gated_plan_bytes(hidden, k, nnz) < 0) return -1;
    return padded(bsmm::gated_wgrad_plan_bytes(hidden, nnz)) + bsmm::gated_dgrad_plan_bytes(k, nnz);
}

int bsmm_build_gated_f32_plan(const int32_t* ptr, const int32_t* idx, const int32_t* csc_ptr, const int32_t* csc_idx, int64_t hidden,
                              int64_t k, int64_t nnz, void* plan, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (bsmm_gated_plan_bytes(hidden, k, nnz) < 0 || ptr == nullptr || csc_ptr == nullptr || plan == nullptr ||
        (nnz > 0 && (idx == nullptr || csc_idx == nullptr)) || !aligned(ptr, 4) || !aligned(idx, 8) || !aligned(csc_ptr, 4) ||
        !aligned(csc_idx, 8) || !aligned(plan, 16))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (k > BSMM_GATED_MAX_K) return BSMM_ERR_TOO_LARGE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t err = bsmm::launch_build_gated_wgrad_plan(ptr, idx, hidden, k, nnz, plan, s);
    if (err == cudaSuccess)
        err = bsmm::launch_build_gated_dgrad_plan(csc_ptr, csc_idx, hidden, k, nnz,
                                                  static_cast<uint8_t*>(plan) + padded(bsmm::gated_wgrad_plan_bytes(hidden, nnz)), s);
    return bsmm::report_cuda(err);
}

int bsmm_gated_pass_backward(const void* x, const void* pre, const void* dh, int64_t m, int64_t k, const int32_t* idx,
                             const int32_t* csc_ptr, const int32_t* csc_idx, const int32_t* blocks, int64_t nnz,
                             const float* data, const void* packed, const void* csc_plan, const void* sddmm_plan,
                             const void* f32_plan, int64_t hidden, void* dpre, void* dx, float* dw, float* dbias,
                             float* block_sumsq, void* workspace, uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    const uint32_t precision = flags & BSMM_PREC_MASK, pass = (flags >> 16) & 0xFu;
    if ((flags & ~(BSMM_PREC_MASK | BSMM_DSD_GROUP(0xFF) | BSMM_GATED_PASS(0xF))) != 0) return BSMM_ERR_UNSUPPORTED;
    // bf16 tensors: the products take them as they are, which the CUDA-core kernels of few tokens or no blocks do not
    const bool io16 = (pass & BSMM_GATED_IO_BF16) != 0;
    if (io16 && (precision != BSMM_PREC_BF16 || m < 32 || nnz == 0)) return BSMM_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // the weight gradient before the input gradient: in data-parallel training its all-reduce can overlap the latter
    if (f32_plan != nullptr && !io16 && m > 0 && from_planes(nnz, precision)) {
        if (hidden <= 0 || k <= 0 || (hidden % 32) != 0 || (k % 32) != 0 || x == nullptr || pre == nullptr || dh == nullptr || workspace == nullptr ||
            (dx != nullptr && (csc_ptr == nullptr || data == nullptr)) || !aligned(x, 16) || !aligned(pre, 16) || !aligned(dh, 16) ||
            !aligned(csc_ptr, 4) || !aligned(data, 16) || !aligned(dx, 16) || !aligned(dw, 16) || !aligned(dbias, 4) || !aligned(f32_plan, 16) ||
            !aligned(workspace, 256))
            return BSMM_ERR_INVALID_ARGUMENT;
        if (gated_types(pass) != BSMM_OK || (pass & BSMM_GATED_X_BF16) != 0) return BSMM_ERR_UNSUPPORTED;
        if (nnz > 0x7fffffff || k > BSMM_GATED_MAX_K || too_large(m, k) || too_large(m, 2 * hidden)) return BSMM_ERR_TOO_LARGE;
        uint8_t* x_planes = static_cast<uint8_t*>(workspace);
        uint8_t* d_planes = x_planes + padded(6 * bsmm::plane_pitch(m) * k);
        uint8_t* rest = d_planes + padded(12 * bsmm::plane_pitch(m) * hidden);  // of each step in turn
        cudaError_t err = bsmm::launch_gated_act_backward(pre, dh, m, hidden, nullptr, dbias, reinterpret_cast<float*>(rest),
                                                          (pass & BSMM_GATED_GELU) != 0, false, false, d_planes, s);
        if (err == cudaSuccess && dw != nullptr) err = bsmm::launch_split_planes(static_cast<const float*>(x), m, k, x_planes, s);
        if (err == cudaSuccess && dw != nullptr)
            err = bsmm::launch_gated_wgrad(x_planes, d_planes, m, k, hidden, nnz, f32_plan, dw, block_sumsq, rest, s);
        if (err == cudaSuccess && dx != nullptr)
            err = bsmm::launch_gated_dgrad(d_planes, m, k, hidden, nnz, data, csc_ptr,
                                           static_cast<const uint8_t*>(f32_plan) + padded(bsmm::gated_wgrad_plan_bytes(hidden, nnz)),
                                           static_cast<float*>(dx), rest, s);
        return bsmm::report_cuda(err);
    }
    int status = bsmm_gated_act_backward(pre, dh, m, hidden, dpre, dbias, workspace, pass, stream);
    if (status == BSMM_OK && dw != nullptr)
        status = bsmm_sddmm(dpre, x, 2 * hidden, k, m, dw, blocks, nnz, idx, sddmm_plan, block_sumsq, workspace,
                            precision | (io16 ? BSMM_SDDMM_IO_BF16 : 0u), stream);
    if (status == BSMM_OK && dx != nullptr)
        status = bsmm_dsd(dpre, m, 2 * hidden, csc_ptr, csc_idx, nnz, data, packed, csc_plan, k, dx, nullptr,
                          (flags & (BSMM_PREC_MASK | BSMM_DSD_GROUP(0xFF))) | BSMM_DSD_DGRAD | (io16 ? BSMM_DSD_IO_BF16 : 0u), stream);
    return status;
}

int64_t bsmm_gated_plan_bytes(int64_t hidden, int64_t k, int64_t nnz) {
    if (hidden < 0 || k < 0 || nnz < 0 || (hidden % 32) != 0 || (k % 32) != 0 || nnz > 0x7fffffff || too_large(hidden, k)) return -1;
    return bsmm::gated_plan_bytes(hidden, k, nnz);
}

int64_t bsmm_gated_images_bytes(int64_t nnz) { return nnz < 0 || nnz > 0x7fffffff ? -1 : bsmm::gated_images_bytes(nnz); }

int bsmm_build_gated_plan(const int32_t* ptr, const int32_t* idx, int64_t hidden, int64_t k, int64_t nnz, void* plan,
                          bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (bsmm_gated_plan_bytes(hidden, k, nnz) < 0 || ptr == nullptr || plan == nullptr || (nnz > 0 && idx == nullptr) ||
        !aligned(ptr, 4) || !aligned(idx, 8) || !aligned(plan, 16))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (k > BSMM_GATED_MAX_K) return BSMM_ERR_TOO_LARGE;
    return bsmm::report_cuda(bsmm::launch_build_gated_plan(ptr, idx, hidden, k, plan, static_cast<cudaStream_t>(stream)));
}

int bsmm_gated_pack(const float* data, const void* plan, int64_t hidden, int64_t k, int64_t nnz, void* images,
                    bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (bsmm_gated_plan_bytes(hidden, k, nnz) < 0 || plan == nullptr || (nnz > 0 && (data == nullptr || images == nullptr)) ||
        !aligned(data, 16) || !aligned(plan, 16) || !aligned(images, 256))
        return BSMM_ERR_INVALID_ARGUMENT;
    return bsmm::report_cuda(bsmm::launch_pack_pairs(data, plan, hidden, k, nnz, images, static_cast<cudaStream_t>(stream)));
}

int bsmm_gated_forward(const void* x, int64_t m, int64_t k, const void* plan, const void* images, int64_t nnz, int64_t hidden,
                       const float* bias, void* h, void* pre, uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (m < 0 || k <= 0 || nnz < 0 || hidden < 0 || (hidden % 32) != 0 || (k % 32) != 0) return BSMM_ERR_INVALID_ARGUMENT;
    if ((flags & ~BSMM_GATED_GELU) != (BSMM_GATED_IO_BF16 | BSMM_GATED_PRE_BF16)) return BSMM_ERR_UNSUPPORTED;
    if (m == 0 || hidden == 0) return BSMM_OK;
    if (x == nullptr || plan == nullptr || h == nullptr || (nnz > 0 && images == nullptr)) return BSMM_ERR_INVALID_ARGUMENT;
    if (!aligned(x, 16) || !aligned(plan, 16) || !aligned(images, 256) || !aligned(bias, 16) || !aligned(h, 16) || !aligned(pre, 16))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (nnz > 0x7fffffff || k > BSMM_GATED_MAX_K || too_large(m, k) || too_large(m, 2 * hidden)) return BSMM_ERR_TOO_LARGE;
    return bsmm::report_cuda(bsmm::launch_gated_umma(x, m, k, plan, images, hidden, bias, h, pre, (flags & BSMM_GATED_GELU) != 0,
                                                     static_cast<cudaStream_t>(stream)));
}

int bsmm_dropout(const void* x, const void* residual, void* out, int64_t n, uint32_t cut, const int64_t* rng,
                 uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (n < 0 || cut >= 65536u) return BSMM_ERR_INVALID_ARGUMENT;
    if ((flags & ~BSMM_DROPOUT_BF16) != 0) return BSMM_ERR_UNSUPPORTED;
    if (n == 0) return BSMM_OK;
    if (x == nullptr || out == nullptr || rng == nullptr) return BSMM_ERR_INVALID_ARGUMENT;
    if (!aligned(x, 16) || !aligned(residual, 16) || !aligned(out, 16) || !aligned(rng, 8)) return BSMM_ERR_INVALID_ARGUMENT;
    return bsmm::report_cuda(bsmm::launch_dropout(x, residual, out, n, cut, rng, (flags & BSMM_DROPOUT_BF16) != 0,
                                                  static_cast<cudaStream_t>(stream)));
}

int bsmm_rng_next(int64_t* state, int64_t* used, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (state == nullptr || used == nullptr || !aligned(state, 8) || !aligned(used, 8)) return BSMM_ERR_INVALID_ARGUMENT;
    return bsmm::report_cuda(bsmm::launch_rng_next(state, used, static_cast<cudaStream_t>(stream)));
}

int64_t bsmm_adapters_workspace_bytes(int64_t tokens, int64_t inner, int64_t rank) {
    if (tokens < 0 || inner < 0 || (inner % 32) != 0 || rank < 0 || rank > 256 || too_large(tokens, inner)) return -1;
    return inner == 0 ? 0 : bsmm::adapters_workspace_bytes(tokens, inner, rank);
}

int bsmm_adapters(const void* x, int64_t tokens, int64_t inner, int64_t outer, const int32_t* offsets, const int32_t* ids,
                  int64_t requests, int64_t count, int64_t rank, const void* down, const void* up, const float* scaling,
                  const void* base, void* out, void* workspace, uint32_t flags, bsmm_stream_t stream) {
    (void)cudaGetLastError();
    if (tokens < 0 || inner <= 0 || outer < 0 || requests < 0 || count < 0 || (inner % 32) != 0 || (outer % 32) != 0)
        return BSMM_ERR_INVALID_ARGUMENT;
    if (rank != 16 && rank != 32 && (rank <= 0 || rank > 256 || (rank % 64) != 0)) return BSMM_ERR_INVALID_ARGUMENT;
    if ((flags & ~(BSMM_ADAPTERS_IN_BF16 | BSMM_ADAPTERS_OUT_BF16)) != 0 || flags == BSMM_ADAPTERS_OUT_BF16) return BSMM_ERR_UNSUPPORTED;
    if (tokens == 0 || outer == 0) return BSMM_OK;
    if (x == nullptr || offsets == nullptr || out == nullptr || workspace == nullptr || (requests > 0 && ids == nullptr) ||
        (count > 0 && (down == nullptr || up == nullptr || scaling == nullptr)))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (!aligned(x, 16) || !aligned(offsets, 4) || !aligned(ids, 4) || !aligned(down, 16) || !aligned(up, 16) ||
        !aligned(scaling, 4) || !aligned(base, 16) || !aligned(out, 16) || !aligned(workspace, 16))
        return BSMM_ERR_INVALID_ARGUMENT;
    if (too_large(tokens, inner) || too_large(tokens, outer) || requests > 0x7ffffffell || count > 0x7fffffffll) return BSMM_ERR_TOO_LARGE;
    bsmm::AdapterCall call = {x, down, up, scaling, offsets, ids, base, out, static_cast<float*>(workspace),
                              tokens, inner, outer, requests, count, rank};
    return bsmm::report_cuda(bsmm::launch_adapters(call, (flags & BSMM_ADAPTERS_IN_BF16) != 0,
                                                   (flags & BSMM_ADAPTERS_OUT_BF16) != 0, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"

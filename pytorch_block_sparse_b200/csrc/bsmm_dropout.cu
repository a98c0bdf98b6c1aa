// Dropout whose mask is a function of (seed, counter, element index) and is never stored, with the residual add in
// the same pass:  out[i] = (keep(i) ? x[i] / (1 - p) : 0) + residual[i].  The backward pass is the same kernel on the
// output's gradient, without a residual.
//
// Random numbers: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with
// the 64-bit seed as key and (element group, counter) as its 128-bit counter.  One call gives eight 16-bit numbers,
// word by word, low half first, for the eight elements of its group; element i is kept when its number is at least
// cut = round(p * 65536), and kept values are scaled by 65536 / (65536 - cut), so the expectation is exact for the
// quantised rate.  Sixteen bits instead of thirty-two halve the integer work per element.
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"

namespace bsmm {
namespace {

struct Philox {
    uint32_t v[4];
};

__device__ __forceinline__ Philox philox4x32(uint64_t index, uint64_t counter, uint64_t seed) {
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32), c2 = (uint32_t)counter, c3 = (uint32_t)(counter >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ float dropped(float x, uint32_t number, uint32_t cut, float scale) {
    return number >= cut ? x * scale : 0.f;  // a selection: a dropped infinity or NaN leaves nothing behind
}

// A thread takes kGroups groups, 256 apart, and asks for all of them before it draws: with one group per thread too little
// is in flight, and the ~110 integer instructions of a group come on top of the memory's latency instead of under it
// (16384 x 4096 bf16 values, one call with and one without residual, 671 MB: 122 us with one group per thread, 110 with four, 6.1 TB/s).
// Whole groups move with 16-byte accesses (the caller aligns the pointers), the ragged last one value by value.
template <typename T, bool kResidual, int kGroups>
__global__ void __launch_bounds__(256)
dropout_kernel(const T* __restrict__ x, const T* residual, T* out, int64_t n, uint32_t cut, float scale,
               const int64_t* __restrict__ rng) {
    const int64_t whole = n / 8, g0 = (int64_t)blockIdx.x * (256 * kGroups) + threadIdx.x;
    Raw8<T> v[kGroups], r[kResidual ? kGroups : 1];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
        const int64_t g = g0 + j * 256;
        if (g < whole) {
            v[j].load(x + g * 8);
            if (kResidual) r[j].load(residual + g * 8);
        }
    }
    const uint64_t seed = (uint64_t)rng[0], counter = (uint64_t)rng[1];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
        const int64_t g = g0 + j * 256, i0 = g * 8;
        if (i0 >= n) break;
        const Philox w = philox4x32((uint64_t)g, counter, seed);
        float f[8], add[8];
        if (g < whole) {
            v[j].unpack(f);
            if (kResidual) r[j].unpack(add);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = i0 + e < n ? to_float(x[i0 + e]) : 0.f;
                if (kResidual) add[e] = i0 + e < n ? to_float(residual[i0 + e]) : 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f[e] = dropped(f[e], (e & 1) ? w.v[e >> 1] >> 16 : w.v[e >> 1] & 0xFFFFu, cut, scale);
            if (kResidual) f[e] += add[e];
        }
        if (g < whole) {
            store8(out + i0, f);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i0 + e < n) out[i0 + e] = from_float<T>(f[e]);
        }
    }
}

// One draw of a state kept on the device: its (seed, counter) goes to `used`, the counter moves on.
__global__ void rng_next_kernel(int64_t* state, int64_t* used) {
    used[0] = state[0];
    used[1] = state[1];
    state[1] = (int64_t)((uint64_t)state[1] + 1u);
}

template <typename T>
cudaError_t launch(const void* x, const void* residual, void* out, int64_t n, uint32_t cut, const int64_t* rng,
                   cudaStream_t stream) {
    const float scale = 65536.f / (float)(65536u - cut);
    const int64_t groups = (n + 7) / 8;
    // several groups per thread once every thread that the GPU holds at once has eight of them to do.  One group -> several, us:
    // bf16 without residual 2^22 values 5.5 -> 6.9, 2^24 15.3 -> 15.4, 3 * 2^23 21.9 -> 21.1, 2^26 55.1 -> 49.5; with it 2^26
    // 66.8 -> 61.2; fp32 2^24 21.8 -> 22.2, 3 * 2^23 33.6 -> 32.1, 2^26 86.0 -> 80.8
    constexpr int kMany = sizeof(T) == 2 ? 4 : 2;
    const bool many = groups >= 148ll * 2048 * 8;
    const int64_t per_cta = 256 * (many ? kMany : 1), ctas = (groups + per_cta - 1) / per_cta;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    const T* in = static_cast<const T*>(x);
    const T* res = static_cast<const T*>(residual);
    T* to = static_cast<T*>(out);
    if (residual != nullptr) {
        if (many) dropout_kernel<T, true, kMany><<<(unsigned)ctas, 256, 0, stream>>>(in, res, to, n, cut, scale, rng);
        else dropout_kernel<T, true, 1><<<(unsigned)ctas, 256, 0, stream>>>(in, res, to, n, cut, scale, rng);
    } else {
        if (many) dropout_kernel<T, false, kMany><<<(unsigned)ctas, 256, 0, stream>>>(in, res, to, n, cut, scale, rng);
        else dropout_kernel<T, false, 1><<<(unsigned)ctas, 256, 0, stream>>>(in, res, to, n, cut, scale, rng);
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_dropout(const void* x, const void* residual, void* out, int64_t n, uint32_t cut, const int64_t* rng,
                           bool bf16, cudaStream_t stream) {
    if (n == 0) return cudaSuccess;
    return bf16 ? launch<__nv_bfloat16>(x, residual, out, n, cut, rng, stream)
                : launch<float>(x, residual, out, n, cut, rng, stream);
}

cudaError_t launch_rng_next(int64_t* state, int64_t* used, cudaStream_t stream) {
    rng_next_kernel<<<1, 1, 0, stream>>>(state, used);
    return cudaGetLastError();
}

}  // namespace bsmm

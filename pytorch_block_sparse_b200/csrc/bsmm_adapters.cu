// Low-rank adapters of many requests beside a shared projection: out[t] = base[t] + s_a (x[t] D_a^T) U_a^T, where a is the
// adapter of the request that token t belongs to; tokens of no request, and of requests without an adapter, keep base[t].
//
// Memory bound: work goes through mma.sync on fragments of 16 bytes per lane.  The contraction index of such a product may be
// permuted as long as both operands agree, so a lane takes eight CONSECUTIVE k of its row -- what two (bf16) or four (tf32)
// instructions want from it -- and the output columns of four instructions are permuted the same way, so that a lane ends
// with eight consecutive columns of each of its two rows.
//
// Two forms, chosen by the average number of tokens per request:
//   clusters  (few tokens per request) one launch: a cluster of eight CTAs owns 4 or 16 tokens.  Each CTA takes an eighth of the
//             input features for v[t] = x[t] D_a^T, the partial v are exchanged through distributed shared memory, and
//             each CTA writes an eighth of the outputs.  Inside a CTA the warps share the tile's distinct adapters and the
//             features; fragments come straight from global memory
//   tiles     (prompts) two launches: the shrink kernel writes v, the expand kernel multiplies by U_a.  A CTA owns 128 tokens
//             of one request; the adapter's matrix passes through shared memory once for its eight warps.  (bf16 tensors,
//             rank up to 128: the shrink kernel of bsmm_adapters_umma.cu)
//
// Arithmetic.  fp32 tensors: both operands are split into tf32 hi + lo parts and three products are added (about 2^-21
// relative per term); bf16 tensors: x D is one exact product, v is split into bf16 hi + lo (its rounding to one bf16 would
// cost as much as the output's own).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "bsmm_adapters.cuh"
#include "bsmm_ptx.cuh"

namespace bsmm {
namespace {

using namespace adapters;

namespace cg = cooperative_groups;

constexpr int kStep = 32;         // input features of one step

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma1688(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// kLen (4 or 8) consecutive values of a row as an operand: bf16 pairs, or tf32 hi and lo parts
template <typename T, int kLen>
struct Fragment;
template <int kLen>
struct Fragment<__nv_bfloat16, kLen> {
    uint32_t hi[kLen / 2];
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        if constexpr (kLen == 8) {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            hi[0] = w.x; hi[1] = w.y; hi[2] = w.z; hi[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
            hi[0] = w.x; hi[1] = w.y;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kLen / 2; ++i) hi[i] = 0;
    }
};
template <int kLen>
struct Fragment<float, kLen> {
    uint32_t hi[kLen], lo[kLen];
    __device__ __forceinline__ void set(int i, float v) {
        hi[i] = ptx::tf32_rna_bits(v);
        lo[i] = ptx::tf32_rna_bits(v - __uint_as_float(hi[i]));
    }
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < kLen / 4; ++i) {
            const float4 v = reinterpret_cast<const float4*>(p)[i];
            set(4 * i, v.x); set(4 * i + 1, v.y); set(4 * i + 2, v.z); set(4 * i + 3, v.w);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kLen; ++i) hi[i] = lo[i] = 0;
    }
};
// v as the operand that meets T's: split in the parts that T's products want
template <typename T, int kLen>
struct SplitFragment;
template <int kLen>
struct SplitFragment<__nv_bfloat16, kLen> {
    uint32_t hi[kLen / 2], lo[kLen / 2];
    __device__ __forceinline__ void set(const float (&v)[kLen]) {
#pragma unroll
        for (int i = 0; i < kLen / 2; ++i) ptx::split_bf16x2(v[2 * i], v[2 * i + 1], hi[i], lo[i]);
    }
};
template <int kLen>
struct SplitFragment<float, kLen> : Fragment<float, kLen> {
    __device__ __forceinline__ void set(const float (&v)[kLen]) {
#pragma unroll
        for (int i = 0; i < kLen; ++i) Fragment<float, kLen>::set(i, v[i]);
    }
};

// c[n] += a b[n] over kLen consecutive contraction indices per lane, n = 0 ... kN - 1; rows g and g + 8 of the left operand.
// Neighbouring instructions add into different accumulators: one that waits for its predecessor's takes four times as long.
template <int kLen, int kN>
__device__ __forceinline__ void multiply(float (*c)[4], const Fragment<__nv_bfloat16, kLen>& a0,
                                         const Fragment<__nv_bfloat16, kLen>& a1, const Fragment<__nv_bfloat16, kLen> (&b)[kN]) {
#pragma unroll
    for (int s = 0; s < kLen / 2; s += 2)
#pragma unroll
        for (int n = 0; n < kN; ++n) mma16816(c[n], a0.hi[s], a1.hi[s], a0.hi[s + 1], a1.hi[s + 1], b[n].hi[s], b[n].hi[s + 1]);
}
template <int kLen, int kN>
__device__ __forceinline__ void multiply(float (*c)[4], const SplitFragment<__nv_bfloat16, kLen>& a0,
                                         const SplitFragment<__nv_bfloat16, kLen>& a1, const Fragment<__nv_bfloat16, kLen> (&b)[kN]) {
#pragma unroll
    for (int s = 0; s < kLen / 2; s += 2) {
#pragma unroll
        for (int n = 0; n < kN; ++n) mma16816(c[n], a0.lo[s], a1.lo[s], a0.lo[s + 1], a1.lo[s + 1], b[n].hi[s], b[n].hi[s + 1]);
#pragma unroll
        for (int n = 0; n < kN; ++n) mma16816(c[n], a0.hi[s], a1.hi[s], a0.hi[s + 1], a1.hi[s + 1], b[n].hi[s], b[n].hi[s + 1]);
    }
}
// fp32: the tensor core truncates its running sums (about 2e-8 per addition), so they only run over this call's inputs.
template <int kLen, int kN>
__device__ __forceinline__ void multiply(float (*c)[4], const Fragment<float, kLen>& a0, const Fragment<float, kLen>& a1,
                                         const Fragment<float, kLen> (&b)[kN]) {
    float sum[kN][4];
#pragma unroll
    for (int n = 0; n < kN; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
#pragma unroll
    for (int s = 0; s < kLen; s += 2) {
#pragma unroll
        for (int n = 0; n < kN; ++n) mma1688(sum[n], a0.lo[s], a1.lo[s], a0.lo[s + 1], a1.lo[s + 1], b[n].hi[s], b[n].hi[s + 1]);
#pragma unroll
        for (int n = 0; n < kN; ++n) mma1688(sum[n], a0.hi[s], a1.hi[s], a0.hi[s + 1], a1.hi[s + 1], b[n].lo[s], b[n].lo[s + 1]);
#pragma unroll
        for (int n = 0; n < kN; ++n) mma1688(sum[n], a0.hi[s], a1.hi[s], a0.hi[s + 1], a1.hi[s + 1], b[n].hi[s], b[n].hi[s + 1]);
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[n][e] += sum[n][e];
}
template <typename T>
constexpr int kGroup = sizeof(T) == 2 ? 4 : 2;  // fragments of the right operand held at a time

// a fragment from shared memory, its 16-byte pieces `pitch` bytes apart
__device__ __forceinline__ void load_pieces(Fragment<__nv_bfloat16, 8>& f, const uint8_t* p, int) {
    f.load(reinterpret_cast<const __nv_bfloat16*>(p));
}
__device__ __forceinline__ void load_pieces(Fragment<__nv_bfloat16, 4>& f, const uint8_t* p, int) {
    f.load(reinterpret_cast<const __nv_bfloat16*>(p));
}
template <int kLen>
__device__ __forceinline__ void load_pieces(Fragment<float, kLen>& f, const uint8_t* p, int pitch) {
#pragma unroll
    for (int i = 0; i < kLen / 4; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(p + i * pitch);
        f.set(4 * i, v.x); f.set(4 * i + 1, v.y); f.set(4 * i + 2, v.z); f.set(4 * i + 3, v.w);
    }
}

// ids[i] = adapter of token t0 + i, or kNone, for i < count <= 16; by one warp.  Offsets and ids come from the device
// unchecked: whatever they hold, the search stays inside the arrays and ends, and an id outside [0, count) counts as none.
// 32 requests are looked at per step, so that the usual batch costs two dependent loads where a binary search costs seven.
__device__ __forceinline__ void find_adapters(const AdapterCall& p, int64_t t0, int count, int* ids) {
    const int lane = threadIdx.x & 31, n = (int)p.requests;
    if (lane < count) ids[lane] = kNone;
    int lo = 0, hi = n;  // the first request that ends behind t0 lies in [lo, hi]
    while (hi - lo > 32) {
        const int step = (hi - lo + 31) / 32, probe = lo + (lane + 1) * step - 1;
        const bool before = probe < hi && __ldg(p.offsets + probe + 1) <= t0;
        const int c = __popc(__ballot_sync(0xffffffffu, before));
        const int from = min(hi, lo + c * step);
        hi = min(hi, from + step);
        lo = from;
    }
    __syncwarp();
    const int64_t t1 = min(t0 + count, p.tokens);
    for (bool more = true; more && lo < n; lo += 32) {
        const int r = lo + lane;
        int64_t start = 0, end = 0;
        int id = kNone;
        if (r < n) {
            start = __ldg(p.offsets + r);
            end = __ldg(p.offsets + r + 1);
            id = __ldg(p.ids + r);
            if (id < 0 || id >= p.count) id = kNone;
        }
        for (int64_t t = max(start, t0); t < min(end, t1); ++t) ids[t - t0] = id;
        more = !__any_sync(0xffffffffu, r < n && end >= t1);
    }
    __syncwarp();
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <typename O>
__device__ __forceinline__ void add_base_and_store(const AdapterCall& p, int64_t t, int64_t n, float (&v)[8]) {
    const O* base = static_cast<const O*>(p.base);
    if (base != nullptr) {
        float b[8];
        load8(base + t * p.outer + n, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += b[j];
    }
    store8(static_cast<O*>(p.out) + t * p.outer + n, v);
}

// ------------------------------------------------------------------------------------------ a cluster on 4 or 16 tokens
constexpr int kClusterCtas = 8, kClusterWarps = 8, kClusterRows = 16;

// dynamic shared memory: [8 warps][16][kRank] partial sums of a round, [16][rank + 4] this CTA's v, the same of the cluster's
template <int kRank>
constexpr int cluster_smem(int64_t rank) {
    return (kClusterWarps * kClusterRows * kRank + 2 * kClusterRows * ((int)rank + 4)) * 4;
}

template <typename T, typename O, int kRank>  // kRank rows of D at a time: 16, 32 or 64
__global__ void __launch_bounds__(32 * kClusterWarps)
cluster_kernel(AdapterCall p, int tile_tokens, int64_t in_part, int64_t out_part) {
    constexpr int kLen = kRank == 16 ? 4 : 8;            // a lane's values of one load: 16 or 32 of the rank per warp load
    constexpr int kLoads = kRank / (4 * kLen);
    extern __shared__ __align__(16) float csmem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int cta = (int)(blockIdx.x % kClusterCtas);
    const int64_t t0 = (int64_t)(blockIdx.x / kClusterCtas) * tile_tokens;
    const int pitch = (int)p.rank + 4;
    float* parts = csmem;
    float* own = parts + kClusterWarps * kClusterRows * kRank;
    float* total = own + kClusterRows * pitch;

    // every warp knows the adapter of each of the tile's tokens: lane i holds token i's
    __shared__ int ids[kClusterRows];
    if (warp == 0) find_adapters(p, t0, tile_tokens, ids);
    __syncthreads();
    const int mine = lane < tile_tokens ? ids[lane] : kNone;
    const uint32_t all = __ballot_sync(0xffffffffu, mine != kNone);
    // distinct adapters: those at their first token
    const uint32_t alike = __match_any_sync(0xffffffffu, mine);
    const uint32_t leaders = __ballot_sync(0xffffffffu, mine != kNone && (int)(__ffs(alike) - 1) == lane);
    const int distinct = __popc(leaders);
    // the warps share the adapters, then each adapter's features
    const int subs = distinct >= 4 ? 4 : distinct >= 2 ? 2 : 1, shares = kClusterWarps / subs;
    const int sub = warp % subs, share = warp / subs;

    const T* x = static_cast<const T*>(p.x);
    const int64_t row0 = t0 + g, row1 = t0 + g + 8;
    const bool live0 = g < tile_tokens && row0 < p.tokens, live1 = g + 8 < tile_tokens && row1 < p.tokens;
    const int64_t begin = min(p.outer, cta * out_part), end = min(p.outer, begin + out_part);
    const int64_t each = (end - begin + 32 * shares - 1) / (32 * shares) * 32;
    const int64_t n0 = min(end, begin + share * each), n1 = min(end, n0 + each);
    {   // what the second half will read of U is asked for now
        uint32_t todo = leaders;
        for (int turn = 0; todo != 0; ++turn, todo &= todo - 1) {
            if (turn % subs != sub) continue;
            const int id = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
            const char* up = reinterpret_cast<const char*>(static_cast<const T*>(p.up) + ((int64_t)id * p.outer + n0) * p.rank);
            const int64_t bytes = (n1 - n0) * p.rank * (int64_t)sizeof(T);
            for (int64_t at = lane * 128; at < bytes; at += 32 * 128) prefetch_l2(up + at);
        }
    }
    {
        const int64_t begin = min(p.inner, cta * in_part), end = min(p.inner, begin + in_part);
        const int64_t each = (end - begin + kStep * shares - 1) / (kStep * shares) * kStep;
        const int64_t k0 = min(end, begin + share * each), k1 = min(end, k0 + each);
        for (int64_t r0 = 0; r0 < p.rank; r0 += kRank) {
            uint32_t todo = leaders;
            for (int turn = 0; todo != 0; ++turn, todo &= todo - 1) {
                if (turn % subs != sub) continue;
                const int id = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
                const uint32_t rows = __shfl_sync(0xffffffffu, alike, __ffs(todo) - 1);
                const T* down = static_cast<const T*>(p.down) + ((int64_t)id * p.rank + r0) * p.inner;
                float acc[kRank / 8][4];
#pragma unroll
                for (int n = 0; n < kRank / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll 4
                for (int64_t k = k0 + q * 8; k < k1; k += kStep) {
                    Fragment<T, 8> a0, a1;
                    if (live0) a0.load(x + row0 * p.inner + k); else a0.clear();
                    if (live1) a1.load(x + row1 * p.inner + k); else a1.clear();
#pragma unroll
                    for (int n0 = 0; n0 < kRank / 8; n0 += 2) {
                        Fragment<T, 8> b[2];
#pragma unroll
                        for (int n = 0; n < 2; ++n) b[n].load(down + (int64_t)((n0 + n) * 8 + g) * p.inner + k);
                        multiply<8, 2>(acc + n0, a0, a1, b);
                    }
                }
                float* to = parts + share * kClusterRows * kRank + 2 * q;
#pragma unroll
                for (int n = 0; n < kRank / 8; ++n) {
                    if ((rows >> g) & 1u) *reinterpret_cast<float2*>(to + g * kRank + n * 8) = make_float2(acc[n][0], acc[n][1]);
                    if ((rows >> (g + 8)) & 1u)
                        *reinterpret_cast<float2*>(to + (g + 8) * kRank + n * 8) = make_float2(acc[n][2], acc[n][3]);
                }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < tile_tokens * kRank; i += 32 * kClusterWarps) {
                const int row = i / kRank, r = i % kRank;
                if (!((all >> row) & 1u)) continue;
                float sum = 0.f;
                for (int s = 0; s < shares; ++s) sum += parts[(s * kClusterRows + row) * kRank + r];
                own[row * pitch + r0 + r] = sum;
            }
            __syncthreads();
        }
    }
    cluster.sync();
    {
        // the cluster's sums, in the CTAs' order, scaled by the token's adapter
        const int rank = (int)p.rank;
        for (int i = threadIdx.x; i < tile_tokens * rank / 4; i += 32 * kClusterWarps) {
            const int row = i * 4 / rank, r = i * 4 % rank;
            if (!((all >> row) & 1u)) continue;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kClusterCtas; ++c) {
                const float4 w = *reinterpret_cast<const float4*>(cluster.map_shared_rank(own, c) + row * pitch + r);
                sum.x += w.x; sum.y += w.y; sum.z += w.z; sum.w += w.w;
            }
            const float scale = __ldg(p.scaling + ids[row]);
            *reinterpret_cast<float4*>(total + row * pitch + r) = make_float4(sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale);
        }
    }
    cluster.barrier_arrive();  // this CTA has read the others' sums
    __syncthreads();
    if (p.base != p.out) {  // tokens without an adapter keep their base
        for (int row = warp; row < tile_tokens; row += kClusterWarps) {
            if (((all >> row) & 1u) || t0 + row >= p.tokens) continue;
#pragma unroll 2
            for (int64_t n = begin + lane * 8; n < end; n += 256) {
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                add_base_and_store<O>(p, t0 + row, n, v);
            }
        }
    }
    uint32_t todo = leaders;
    for (int turn = 0; todo != 0; ++turn, todo &= todo - 1) {
        if (turn % subs != sub) continue;
        const int id = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
        const uint32_t rows = __shfl_sync(0xffffffffu, alike, __ffs(todo) - 1);
        const bool use0 = ((rows >> g) & 1u) != 0, use1 = ((rows >> (g + 8)) & 1u) != 0;
        const T* up = static_cast<const T*>(p.up) + (int64_t)id * p.outer * p.rank;
        SplitFragment<T, kLen> v0[kLoads], v1[kLoads];
        auto load_rank = [&](int64_t r0) {  // (rows of other adapters are computed along and not stored)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                float a[kLen], b[kLen];
                const float* from = total + g * pitch + r0 + (i * 4 + q) * kLen;
#pragma unroll
                for (int e = 0; e < kLen; e += 4) {
                    *reinterpret_cast<float4*>(a + e) = *reinterpret_cast<const float4*>(from + e);
                    *reinterpret_cast<float4*>(b + e) = *reinterpret_cast<const float4*>(from + 8 * pitch + e);
                }
                v0[i].set(a);
                v1[i].set(b);
            }
        };
        if (p.rank == kRank) load_rank(0);
#pragma unroll 4
        for (int64_t n = n0; n < n1; n += 32) {
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            for (int64_t r0 = 0; r0 < p.rank; r0 += kRank) {
                if (p.rank != kRank) load_rank(r0);
#pragma unroll
                for (int j0 = 0; j0 < 4; j0 += kGroup<T>)
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        Fragment<T, kLen> b[kGroup<T>];
#pragma unroll
                        for (int j = 0; j < kGroup<T>; ++j) {
                            const int64_t col = n + (g >> 1) * 8 + (j0 + j) * 2 + (g & 1);
                            b[j].load(up + col * p.rank + r0 + (i * 4 + q) * kLen);
                        }
                        multiply<kLen, kGroup<T>>(acc + j0, v0[i], v1[i], b);
                    }
            }
            if (use0) {
                float v[8] = {acc[0][0], acc[0][1], acc[1][0], acc[1][1], acc[2][0], acc[2][1], acc[3][0], acc[3][1]};
                add_base_and_store<O>(p, row0, n + q * 8, v);
            }
            if (use1) {
                float v[8] = {acc[0][2], acc[0][3], acc[1][2], acc[1][3], acc[2][2], acc[2][3], acc[3][2], acc[3][3]};
                add_base_and_store<O>(p, row1, n + q * 8, v);
            }
        }
    }
    cluster.barrier_wait();  // nobody leaves while its sums are read
}

// ---------------------------------------------------------------------------------------------- a CTA on 128 tokens
constexpr int kTileWarps = 8, kTileThreads = 32 * kTileWarps;

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// Shrink: a stage of the ring holds 128 bytes of k of the tile's tokens -- every lane copies the pieces that it will read
// itself -- and of kRank rows of D, shared by the warps (16-byte piece c of row r at c ^ 4 (r mod 2): the two rows of a
// quarter-warp's load use different banks).  The CTAs of a cluster take a part of the input features each and add their sums
// up through distributed shared memory, every one a share of the tokens, in the order of the parts.
template <typename T, int kRank>
struct ShrinkTile {
    static constexpr int kStepK = 128 / (int)sizeof(T);             // input features of a stage
    static constexpr int kXBytes = kTileTokens * 128, kDBytes = kRank * 128;
    static constexpr int kStage = kXBytes + kDBytes;
    static constexpr int kStages = 4;
    static constexpr int kTotal = kStages * kStage;
    static_assert(kTotal >= kTileTokens * kRank * 4, "the sums reuse the ring");
};

template <typename T, int kRank>
__global__ void __launch_bounds__(kTileThreads, 2)
shrink_tile_kernel(AdapterCall p, Units units) {
    using S = ShrinkTile<T, kRank>;
    constexpr int kPieceLen = 16 / (int)sizeof(T);    // values of a 16-byte piece
    constexpr int kPieces = 8 / kPieceLen;            // pieces of a fragment
    constexpr int kSteps = S::kStepK / kStep;         // 32-feature steps of a stage
    constexpr int kN = kRank / 8 < kGroup<T> ? kRank / 8 : kGroup<T>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int parts = (int)units.parts, part = (int)blockIdx.x % parts;
    const int64_t k0 = min(p.inner, part * units.per_part), k1 = min(p.inner, k0 + units.per_part);
    const int range = (int)(k1 - k0), stages = (range + S::kStepK - 1) / S::kStepK;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
    let_expand_start();
    Tile tile;
    if (!tile.find(p, (int)blockIdx.x / parts) || tile.id == kNone) return;  // (the whole cluster alike)

    cg::cluster_group cluster = cg::this_cluster();
    const int last = tile.first + tile.rows - 1, t0 = tile.first + warp * 16 + g;
    const bool busy = warp * 16 < tile.rows;
    const T* x0 = static_cast<const T*>(p.x) + (int64_t)min(t0, last) * p.inner + k0 + q * 8;
    const T* x1 = static_cast<const T*>(p.x) + (int64_t)min(t0 + 8, last) * p.inner + k0 + q * 8;
    for (int64_t r0 = 0; r0 < p.rank; r0 += kRank) {
        const int dr = threadIdx.x >> 3, dc = threadIdx.x & 7;
        const T* d0 = static_cast<const T*>(p.down) + ((int64_t)tile.id * p.rank + r0 + dr) * p.inner + k0 + dc * kPieceLen;
        const uint32_t d_to = S::kXBytes + dr * 128 + ((dc ^ ((dr & 1) << 2)) << 4);
        auto issue = [&](int s) {
            if (s < stages) {
                const uint32_t stage = base + (s % S::kStages) * S::kStage;
                const int k = s * S::kStepK, left = range - k;  // features behind the stage's first
                if (busy) {
                    const uint32_t to = stage + threadIdx.x * 16;
#pragma unroll
                    for (int i = 0; i < kSteps; ++i)
                        if (i * kStep < left) {
#pragma unroll
                            for (int c = 0; c < kPieces; ++c) {
                                copy16(to + (i * kPieces + c) * 2 * kTileThreads * 16, x0 + k + i * kStep + c * kPieceLen);
                                copy16(to + ((i * kPieces + c) * 2 + 1) * kTileThreads * 16, x1 + k + i * kStep + c * kPieceLen);
                            }
                        }
                }
                if (dc * kPieceLen < left) {
#pragma unroll
                    for (int j = 0; j < (kRank * 8 + kTileThreads - 1) / kTileThreads; ++j)
                        if (j * 32 + dr < kRank) copy16(stage + d_to + j * 32 * 128, d0 + (int64_t)j * 32 * p.inner + k);
                }
            }
            commit_copies();
        };
        float acc[kRank / 8][4];
#pragma unroll
        for (int n = 0; n < kRank / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
        for (int s = 0; s < S::kStages - 1; ++s) issue(s);
        for (int s = 0; s < stages; ++s) {
            wait_copies<S::kStages - 2>();
            __syncthreads();  // the stage has arrived for everybody, and the one before has been read by everybody
            issue(s + S::kStages - 1);
            if (!busy) continue;
            const uint8_t* stage = smem + (s % S::kStages) * S::kStage;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (s * S::kStepK + i * kStep >= range) break;
                Fragment<T, 8> a0, a1;
                load_pieces(a0, stage + (i * kPieces * 2 * kTileThreads + threadIdx.x) * 16, 2 * kTileThreads * 16);
                load_pieces(a1, stage + ((i * kPieces * 2 + 1) * kTileThreads + threadIdx.x) * 16, 2 * kTileThreads * 16);
#pragma unroll
                for (int n0 = 0; n0 < kRank / 8; n0 += kN) {
                    Fragment<T, 8> b[kN];
#pragma unroll
                    for (int n = 0; n < kN; ++n)
                        load_pieces(b[n], stage + S::kXBytes + ((n0 + n) * 8 + g) * 128 + ((((i * 4 + q) * kPieces) ^ ((g & 1) << 2)) << 4), 16);
                    multiply<8, kN>(acc + n0, a0, a1, b);
                }
            }
        }
        wait_copies<0>();
        __syncthreads();  // the ring has been read: its memory takes the sums, [128][kRank]
        float* sums = reinterpret_cast<float*>(smem);
        float* mine = sums + (warp * 16 + g) * kRank + 2 * q;
#pragma unroll
        for (int n = 0; n < kRank / 8; ++n) {
            *reinterpret_cast<float2*>(mine + n * 8) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2*>(mine + 8 * kRank + n * 8) = make_float2(acc[n][2], acc[n][3]);
        }
        if (parts > 1) cluster.sync(); else __syncthreads();
        for (int i = part * kTileThreads + threadIdx.x; i < tile.rows * (kRank / 4); i += parts * kTileThreads) {
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < parts; ++c) {
                const float4 w = reinterpret_cast<const float4*>(parts > 1 ? cluster.map_shared_rank(sums, c) : sums)[i];
                sum.x += w.x; sum.y += w.y; sum.z += w.z; sum.w += w.w;
            }
            *reinterpret_cast<float4*>(p.workspace + (int64_t)(tile.first + i / (kRank / 4)) * p.rank + r0 + i % (kRank / 4) * 4) = sum;
        }
        if (parts > 1) cluster.sync(); else __syncthreads();  // the sums have been read
    }
}

// Expand: the ring passes kExpandCols columns of U_a (rows of the stored matrix) at a time to the CTA's warps, and to every
// lane the pieces of the base that it will add to.  v, scaled, is held in registers, of ranks that pass in pieces in
// shared memory (in shared memory throughout, with one stage less: 4096 fp32 tokens of 8 requests, 4096 -> 4096, rank 64: 178 us instead of
// 148, bf16 with an fp32 base 64 instead of 56, bf16 throughout the same).
constexpr int kExpandCols = 64;
template <typename T, typename O, int kRank>
struct ExpandTile {
    static constexpr int kUBytes = kExpandCols * kRank * (int)sizeof(T);
    static constexpr int kBaseBytes = kTileTokens * kExpandCols * (int)sizeof(O);
    static constexpr int kStage = kUBytes + kBaseBytes;
    static constexpr int kStages = sizeof(O) == 4 && kRank == 64 ? 2 : 4;  // (v of rank 256 has to fit beside them)
    static constexpr int total(int64_t rank) { return kStages * kStage + (rank > kRank ? kTileTokens * ((int)rank + 4) * 4 : 0); }
    static_assert(kStages * kStage + kTileTokens * (256 + 4) * 4 <= 232448 || kRank < 64, "rank 256");
};

template <typename T, typename O, int kRank>
__global__ void __launch_bounds__(kTileThreads, 2)
expand_tile_kernel(AdapterCall p, Units units) {
    constexpr int kLen = kRank == 16 ? 4 : 8;
    constexpr int kLoads = kRank / (4 * kLen);
    constexpr int kRowBytes = kRank * (int)sizeof(T);
    constexpr int kRowPieces = kRowBytes / 16;
    constexpr int kSwizzle = kRowPieces >= 8 ? 4 : 0;  // shorter rows: two neighbours share a 128-byte line as they lie
    using S = ExpandTile<T, O, kRank>;
    constexpr int kStages = S::kStages;
    constexpr int kBaseLen = 16 / (int)sizeof(O), kBasePieces = 8 / kBaseLen;  // of eight consecutive outputs
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int64_t part = blockIdx.x / units.tiles;
    const int64_t n0 = part * units.per_part, n1 = min(p.outer, n0 + units.per_part);
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem);
    Tile tile;
    const bool found = tile.find(p, (int)(blockIdx.x % units.tiles));
    if (!found || tile.id == kNone) {
        if (found) keep_base<O, kTileThreads>(p, tile, n0, n1);
        wait_for_shrink();
        return;
    }
    const int last = tile.first + tile.rows - 1, t0 = tile.first + warp * 16 + g;
    const bool row0 = t0 <= last, row1 = t0 + 8 <= last, busy = warp * 16 < tile.rows;
    const int chunks = (int)((n1 - n0 + kExpandCols - 1) / kExpandCols);
    const int rounds = (int)(p.rank / kRank);  // a chunk's columns pass in `rounds` pieces of the rank

    // what this thread copies into every stage: kUCopies pieces of U, and of the base what it adds to
    constexpr int kUCopies = (kExpandCols * kRowPieces + kTileThreads - 1) / kTileThreads, kUStep = kTileThreads / kRowPieces;
    static_assert(kUStep % 2 == 0, "a thread's columns have one parity");
    const int ucol = threadIdx.x / kRowPieces, uc = threadIdx.x % kRowPieces;
    const T* u0 = static_cast<const T*>(p.up) + ((int64_t)tile.id * p.outer + n0 + ucol) * p.rank + uc * (16 / (int)sizeof(T));
    const uint32_t u_to = ucol * kRowBytes + ((uc ^ ((ucol & 1) * kSwizzle)) << 4);
    const O* base0 = static_cast<const O*>(p.base) + (int64_t)t0 * p.outer + n0 + q * 8;
    const bool copy0 = row0 && p.base != nullptr, copy1 = row1 && p.base != nullptr;
    auto issue = [&](int s) {
        if (s < chunks * rounds) {
            const uint32_t stage = ring + (s % kStages) * S::kStage;
            const int chunk = rounds == 1 ? s : s / rounds, round = rounds == 1 ? 0 : s % rounds;
            const int n = chunk * kExpandCols, left = (int)(n1 - n0) - n;
            const T* u = u0 + (int64_t)n * p.rank + round * kRank;
#pragma unroll
            for (int j = 0; j < kUCopies; ++j)
                if (j * kUStep + ucol < kExpandCols && j * kUStep + ucol < left)
                    copy16(stage + u_to + j * kUStep * kRowBytes, u + (int64_t)j * kUStep * p.rank);
            if (round == rounds - 1) {
                const uint32_t to = stage + S::kUBytes + threadIdx.x * 16;
#pragma unroll
                for (int h = 0; h < kExpandCols / 32; ++h)
                    if (h * 32 < left) {
#pragma unroll
                        for (int e = 0; e < kBasePieces; ++e) {
                            if (copy0) copy16(to + (h * 2 * kBasePieces + e) * kTileThreads * 16, base0 + n + h * 32 + e * kBaseLen);
                            if (copy1)
                                copy16(to + ((h * 2 + 1) * kBasePieces + e) * kTileThreads * 16, base0 + 8 * p.outer + n + h * 32 + e * kBaseLen);
                        }
                    }
            }
        }
        commit_copies();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    const float scale = __ldg(p.scaling + tile.id);
    wait_for_shrink();

    // v: held in registers where its rank passes in one piece, else in shared memory, rows of rank + 4 floats
    float* vs = reinterpret_cast<float*>(smem + kStages * S::kStage);
    const int pitch = (int)p.rank + 4, quads = (int)p.rank / 4;
    const float* source = p.workspace + (int64_t)tile.first * p.rank;
    SplitFragment<T, kLen> v0[kLoads], v1[kLoads];
    auto load_rank = [&](const float* v, int row_pitch, bool first, bool second, float factor) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            float a[kLen], b[kLen];
#pragma unroll
            for (int e = 0; e < kLen; e += 4) {
                const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 u = first ? *reinterpret_cast<const float4*>(v + i * 4 * kLen + e) : zero;
                const float4 w = second ? *reinterpret_cast<const float4*>(v + 8 * row_pitch + i * 4 * kLen + e) : zero;
                a[e] = u.x * factor; a[e + 1] = u.y * factor; a[e + 2] = u.z * factor; a[e + 3] = u.w * factor;
                b[e] = w.x * factor; b[e + 1] = w.y * factor; b[e + 2] = w.z * factor; b[e + 3] = w.w * factor;
            }
            v0[i].set(a);
            v1[i].set(b);
        }
    };
    if (rounds == 1) {
        load_rank(source + (warp * 16 + g) * kRank + q * kLen, kRank, row0, row1, scale);
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < tile.rows * quads; i += kTileThreads) {
            float4 sum = reinterpret_cast<const float4*>(source)[i];
            sum.x *= scale; sum.y *= scale; sum.z *= scale; sum.w *= scale;
            *reinterpret_cast<float4*>(vs + (i / quads) * pitch + (i % quads) * 4) = sum;
        }
        __syncthreads();
    }
    float acc[kExpandCols / 8][4];
    for (int s = 0; s < chunks * rounds; ++s) {
        const int chunk = rounds == 1 ? s : s / rounds, round = rounds == 1 ? 0 : s % rounds;
        wait_copies<kStages - 2>();
        __syncthreads();
        issue(s + kStages - 1);
        if (!busy) continue;
        if (rounds > 1) load_rank(vs + (warp * 16 + g) * pitch + round * kRank + q * kLen, pitch, true, true, 1.f);  // (rows behind the last: not stored)
        if (round == 0) {
#pragma unroll
            for (int j = 0; j < kExpandCols / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        }
        const uint8_t* stage = smem + (s % kStages) * S::kStage;
#pragma unroll
        for (int j0 = 0; j0 < kExpandCols / 8; j0 += kGroup<T>)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                Fragment<T, kLen> b[kGroup<T>];
#pragma unroll
                for (int j = 0; j < kGroup<T>; ++j) {
                    const int col = (j0 + j) / 4 * 32 + (g >> 1) * 8 + (j0 + j) % 4 * 2 + (g & 1);
                    const int c = (i * 4 + q) * kLen * (int)sizeof(T);  // byte in the row
                    load_pieces(b[j], stage + col * kRowBytes + (c ^ ((g & 1) * kSwizzle * 16)), 16);
                }
                multiply<kLen, kGroup<T>>(acc + j0, v0[i], v1[i], b);
            }
        if (round != rounds - 1) continue;
        const int n = chunk * kExpandCols, left = (int)(n1 - n0) - n;
        O* out0 = static_cast<O*>(p.out) + (int64_t)t0 * p.outer + n0 + n + q * 8;
#pragma unroll
        for (int h = 0; h < kExpandCols / 32; ++h) {
            if (h * 32 >= left) break;
            const uint8_t* from = stage + S::kUBytes + (h * 2 * kBasePieces * kTileThreads + threadIdx.x) * 16;
#pragma unroll
            for (int second = 0; second < 2; ++second) {
                if (second ? !row1 : !row0) continue;
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (p.base != nullptr) {
                    Raw8<O> b;
                    b.load_pieces(from + second * kBasePieces * kTileThreads * 16, kTileThreads * 16);
                    b.unpack(v);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += acc[h * 4 + (e >> 1)][2 * second + (e & 1)];
                store8(out0 + (second ? 8 * p.outer : 0) + h * 32, v);
            }
        }
    }
    wait_copies<0>();
}

// Prompts go by tiles of 128 tokens, short requests and small batches by clusters.  us at 4096 -> 4096 features, rank 64,
// clusters / tiles: 512 tokens in 2 requests 15 / 18, in 16 requests 15 / 19; 1024 tokens in 4 requests 29 / 20, in 32 29 / 28, in
// 64 30 / 37; 4096 tokens in 64 requests 117 / 47, in 128 117 / 84, in 256 117 / 109 (rank 16: 66 / 29, 66 / 50, 66 / 71).
bool by_tiles(int64_t tokens, int64_t requests) { return tokens >= 768 && tokens >= 32 * requests; }

template <typename T, typename O, int kRank>
cudaError_t launch_tiles(const AdapterCall& p, cudaStream_t stream) {
    const Units shrink = tile_units(p);
    Units expand = shrink;
    cut_outputs(expand, p.outer, kExpandCols, 2 * 148 / (ceil_div(p.tokens, kTileTokens) + p.requests / 2));
    constexpr int kShrinkBytes = ShrinkTile<T, kRank>::kTotal;
    static bool shrink_ready[64] = {false}, expand_ready[64] = {false};
    cudaError_t err = allow_smem(expand_tile_kernel<T, O, kRank>, ExpandTile<T, O, kRank>::total(kRank < 64 ? kRank : 256), expand_ready);
    if (err != cudaSuccess) return err;
    if (shrink_on_umma(p, sizeof(T) == 2)) {
        err = launch_shrink_umma(p, shrink, stream);
    } else {
        err = allow_smem(shrink_tile_kernel<T, kRank>, kShrinkBytes, shrink_ready);
        if (err == cudaSuccess)
            err = launch_with(shrink_tile_kernel<T, kRank>, shrink.tiles * shrink.parts, kTileThreads, kShrinkBytes, (int)shrink.parts,
                              false, stream, p, shrink);
    }
    if (err != cudaSuccess) return err;
    return launch_with(expand_tile_kernel<T, O, kRank>, expand.tiles * expand.parts, kTileThreads,
                       ExpandTile<T, O, kRank>::total(p.rank), 1, true, stream, p, expand);
}

template <typename T, typename O, int kRank>
cudaError_t launch(const AdapterCall& p, cudaStream_t stream) {
    if (by_tiles(p.tokens, p.requests)) return launch_tiles<T, O, kRank>(p, stream);
    static bool ready[64] = {false};
    const cudaError_t err = allow_smem(cluster_kernel<T, O, kRank>, cluster_smem<kRank>(kRank < 64 ? kRank : 256), ready);
    if (err != cudaSuccess) return err;
    // few tokens: smaller tiles, more CTAs
    const int tile_tokens = ceil_div(p.tokens, 4) * kClusterCtas <= 2 * 148 ? 4 : kClusterRows;
    const int64_t in_part = ceil_div(p.inner, kClusterCtas * 32) * 32, out_part = ceil_div(p.outer, kClusterCtas * 32) * 32;
    return launch_with(cluster_kernel<T, O, kRank>, ceil_div(p.tokens, tile_tokens) * kClusterCtas, 32 * kClusterWarps,
                       cluster_smem<kRank>(p.rank), kClusterCtas, false, stream, p, tile_tokens, in_part, out_part);
}

template <typename T, typename O>
cudaError_t by_rank(const AdapterCall& p, cudaStream_t stream) {
    if (p.rank == 16) return launch<T, O, 16>(p, stream);
    if (p.rank == 32) return launch<T, O, 32>(p, stream);
    if (p.rank % 64 == 0) return launch<T, O, 64>(p, stream);
    return cudaErrorInvalidValue;
}

}  // namespace

int64_t adapters_workspace_bytes(int64_t tokens, int64_t inner, int64_t rank) {
    if (tokens == 0) return 0;
    (void)inner;
    return tokens * rank * (int64_t)sizeof(float);  // v
}

cudaError_t launch_adapters(const AdapterCall& p, bool in_bf16, bool out_bf16, cudaStream_t stream) {
    if (p.tokens == 0 || p.outer == 0) return cudaSuccess;
    if (!in_bf16) return out_bf16 ? cudaErrorInvalidValue : by_rank<float, float>(p, stream);
    return out_bf16 ? by_rank<__nv_bfloat16, __nv_bfloat16>(p, stream) : by_rank<__nv_bfloat16, float>(p, stream);
}

}  // namespace bsmm

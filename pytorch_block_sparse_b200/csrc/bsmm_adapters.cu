// Low-rank adapters of many requests beside a shared projection: out[t] = base[t] + s_a (x[t] D_a^T) U_a^T, where a is the
// adapter of the request that token t belongs to; tokens of no request, and of requests without an adapter, keep base[t].
//
// Two launches: the shrink kernel writes v[t] = x[t] D_a^T in fp32 (partial sums over ranges of the input features when
// few tokens would leave SMs idle), the expand kernel adds the partial sums in order, scales and multiplies by U_a.
// Both are memory bound (2 rank FLOP per input byte): one warp owns 16 tokens and works with mma.m16n8k16 on fragments
// loaded straight from global memory, 16 bytes per lane.  The contraction index of such a product may be permuted as long
// as both operands agree, so a lane takes eight CONSECUTIVE k of its row -- the four pairs that two instructions want
// from it -- and nothing passes through shared memory; the output columns of four instructions are permuted the same
// way so that a lane ends with eight consecutive columns of each of its two rows.
// A warp walks the distinct adapters among its tokens.  With many short requests the walk is shared between `subs` warps.
// fp32 tensors: both operands are split into bf16 hi + lo parts and three products are added (about 2^-16 relative per
// term); bf16 tensors: x D is one product, v is split (its rounding to bf16 would cost as much as the output's own).
#include <cuda_bf16.h>

#include "bsmm_feedforward.cuh"
#include "bsmm_ptx.cuh"

namespace bsmm {
namespace {

constexpr int kTokens = 16;       // tokens of a warp
constexpr int kWarps = 4;         // warps of a CTA, each on its own
constexpr int kStep = 32;         // input features of one step
constexpr int kNone = -1;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// kPairs pairs of consecutive values as bf16 pairs: hi parts, and lo parts (what hi leaves) of fp32 values
template <typename T, int kPairs>
struct Fragment;
template <int kPairs>
struct Fragment<__nv_bfloat16, kPairs> {
    static constexpr bool kSplit = false;
    uint32_t hi[kPairs];
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        if (kPairs == 4) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
            hi[0] = w.x; hi[1] = w.y; hi[2 % kPairs] = w.z; hi[3 % kPairs] = w.w;
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
            hi[0] = w.x; hi[1] = w.y;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) hi[i] = 0;
    }
};
template <int kPairs>
struct Fragment<float, kPairs> {
    static constexpr bool kSplit = true;
    uint32_t hi[kPairs], lo[kPairs];
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < kPairs / 2; ++i) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
            ptx::split_bf16x2(v.x, v.y, hi[2 * i], lo[2 * i]);
            ptx::split_bf16x2(v.z, v.w, hi[2 * i + 1], lo[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) hi[i] = lo[i] = 0;
    }
};

// The adapter of token t, or kNone.  Offsets and ids come from the device unchecked: whatever they hold, the search stays
// inside the arrays and ends, and an id outside [0, count) counts as none.
__device__ __forceinline__ int adapter_of(int64_t t, int64_t tokens, const int32_t* __restrict__ offsets,
                                          const int32_t* __restrict__ ids, int requests, int count) {
    if (t >= tokens || requests == 0) return kNone;
    int lo = 0, hi = requests;  // first request whose end lies behind t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(offsets + mid + 1) <= t) lo = mid + 1; else hi = mid;
    }
    if (lo == requests || __ldg(offsets + lo) > t) return kNone;
    const int id = __ldg(ids + lo);
    return id >= 0 && id < count ? id : kNone;
}

struct Units {
    int64_t tiles;      // of kTokens tokens
    int64_t parts;      // ranges of input features (shrink) or of output features (expand)
    int subs;           // warps that share a tile's adapters
    int64_t per_part;   // features of a part, a multiple of 32
};

// v[split][t][0 .. rank) = sum over the split's input features of x[t] D_a^T
template <typename T, int kRank>  // kRank rows of D at a time: 16, 32 or 64
__global__ void __launch_bounds__(32 * kWarps)
shrink_kernel(AdapterCall p, Units units) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (unit >= units.tiles * units.parts * units.subs) return;
    const int64_t tile = unit % units.tiles, rest = unit / units.tiles;
    const int sub = (int)(rest % units.subs);
    const int64_t part = rest / units.subs;
    const int64_t k0 = part * units.per_part, k1 = min(p.inner, k0 + units.per_part);
    const int64_t t0 = tile * kTokens;
    const T* x = static_cast<const T*>(p.x);

    const int mine = lane < kTokens ? adapter_of(t0 + lane, p.tokens, p.offsets, p.ids, (int)p.requests, (int)p.count) : kNone;
    uint32_t todo = __ballot_sync(0xffffffffu, mine != kNone);
    const bool live0 = t0 + g < p.tokens, live1 = t0 + g + 8 < p.tokens;
    for (int turn = 0; todo != 0; ++turn) {
        const int id = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
        const uint32_t rows = __ballot_sync(0xffffffffu, mine == id);
        todo &= ~rows;
        if (turn % units.subs != sub) continue;
        for (int64_t r0 = 0; r0 < p.rank; r0 += kRank) {
            const T* down = static_cast<const T*>(p.down) + ((int64_t)id * p.rank + r0) * p.inner;
            float acc[kRank / 8][4];
#pragma unroll
            for (int n = 0; n < kRank / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll 2
            for (int64_t k = k0 + q * 8; k < k1; k += kStep) {
                Fragment<T, 4> a0, a1;
                if (live0) a0.load(x + (t0 + g) * p.inner + k); else a0.clear();
                if (live1) a1.load(x + (t0 + g + 8) * p.inner + k); else a1.clear();
#pragma unroll
                for (int n = 0; n < kRank / 8; ++n) {
                    Fragment<T, 4> b;
                    b.load(down + (int64_t)(n * 8 + g) * p.inner + k);
#pragma unroll
                    for (int s = 0; s < 4; s += 2) {
                        mma16816(acc[n], a0.hi[s], a1.hi[s], a0.hi[s + 1], a1.hi[s + 1], b.hi[s], b.hi[s + 1]);
                        if constexpr (Fragment<T, 4>::kSplit) {
                            mma16816(acc[n], a0.hi[s], a1.hi[s], a0.hi[s + 1], a1.hi[s + 1], b.lo[s], b.lo[s + 1]);
                            mma16816(acc[n], a0.lo[s], a1.lo[s], a0.lo[s + 1], a1.lo[s + 1], b.hi[s], b.hi[s + 1]);
                        }
                    }
                }
            }
            float* v = p.workspace + (part * p.tokens + t0) * p.rank + r0 + 2 * q;
#pragma unroll
            for (int n = 0; n < kRank / 8; ++n) {
                if ((rows >> g) & 1u) *reinterpret_cast<float2*>(v + g * p.rank + n * 8) = make_float2(acc[n][0], acc[n][1]);
                if ((rows >> (g + 8)) & 1u)
                    *reinterpret_cast<float2*>(v + (g + 8) * p.rank + n * 8) = make_float2(acc[n][2], acc[n][3]);
            }
        }
    }
}

// the values of v that a lane holds as an operand: kPairs pairs of a row, summed over the splits, scaled, split in two
template <int kPairs>
__device__ __forceinline__ void load_v(const AdapterCall& p, int64_t splits, int64_t t, int64_t r, float scale, bool wanted,
                                       uint32_t (&hi)[kPairs], uint32_t (&lo)[kPairs]) {
    float v[2 * kPairs];
#pragma unroll
    for (int i = 0; i < 2 * kPairs; ++i) v[i] = 0.f;
    if (wanted) {
        for (int64_t s = 0; s < splits; ++s) {
            const float4* src = reinterpret_cast<const float4*>(p.workspace + (s * p.tokens + t) * p.rank + r);
#pragma unroll
            for (int i = 0; i < kPairs / 2; ++i) {
                const float4 w = src[i];
                v[4 * i] += w.x; v[4 * i + 1] += w.y; v[4 * i + 2] += w.z; v[4 * i + 3] += w.w;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) ptx::split_bf16x2(v[2 * i] * scale, v[2 * i + 1] * scale, hi[i], lo[i]);
}

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

template <typename T, typename O, int kRank>
__global__ void __launch_bounds__(32 * kWarps)
expand_kernel(AdapterCall p, Units units, int64_t splits) {
    constexpr int kPairs = kRank == 16 ? 2 : 4;          // a lane's pairs of one load: 16 or 32 of the rank per warp load
    constexpr int kLoads = kRank / (8 * kPairs);
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (unit >= units.tiles * units.parts * units.subs) return;
    const int64_t tile = unit % units.tiles, rest = unit / units.tiles;
    const int sub = (int)(rest % units.subs);
    const int64_t part = rest / units.subs;
    const int64_t n0 = part * units.per_part, n1 = min(p.outer, n0 + units.per_part);
    const int64_t t0 = tile * kTokens;

    const int mine = lane < kTokens ? adapter_of(t0 + lane, p.tokens, p.offsets, p.ids, (int)p.requests, (int)p.count) : kNone;
    uint32_t todo = __ballot_sync(0xffffffffu, mine != kNone);
    const uint32_t idle = ~todo & 0xFFFFu;  // tokens without an adapter keep their base
    if (sub == 0 && (p.base != p.out)) {
        for (int row = g; row < kTokens; row += 8) {
            if (!((idle >> row) & 1u) || t0 + row >= p.tokens) continue;
            for (int64_t n = n0 + q * 8; n < n1; n += 32) {
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                add_base_and_store<O>(p, t0 + row, n, v);
            }
        }
    }
    for (int turn = 0; todo != 0; ++turn) {
        const int id = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
        const uint32_t rows = __ballot_sync(0xffffffffu, mine == id);
        todo &= ~rows;
        if (turn % units.subs != sub) continue;
        const bool row0 = ((rows >> g) & 1u) != 0, row1 = ((rows >> (g + 8)) & 1u) != 0;
        const float scale = __ldg(p.scaling + id);
        const T* up = static_cast<const T*>(p.up) + (int64_t)id * p.outer * p.rank;
        uint32_t hi0[kLoads][kPairs], lo0[kLoads][kPairs], hi1[kLoads][kPairs], lo1[kLoads][kPairs];
        auto load_rank = [&](int64_t r0) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int64_t r = r0 + i * 8 * kPairs + q * 2 * kPairs;
                load_v<kPairs>(p, splits, t0 + g, r, scale, row0, hi0[i], lo0[i]);
                load_v<kPairs>(p, splits, t0 + g + 8, r, scale, row1, hi1[i], lo1[i]);
            }
        };
        if (p.rank == kRank) load_rank(0);
        for (int64_t n = n0; n < n1; n += 32) {
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            for (int64_t r0 = 0; r0 < p.rank; r0 += kRank) {
                if (p.rank != kRank) load_rank(r0);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t col = n + (g >> 1) * 8 + j * 2 + (g & 1);
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        Fragment<T, kPairs> b;
                        b.load(up + col * p.rank + r0 + i * 8 * kPairs + q * 2 * kPairs);
#pragma unroll
                        for (int s = 0; s < kPairs; s += 2) {
                            mma16816(acc[j], hi0[i][s], hi1[i][s], hi0[i][s + 1], hi1[i][s + 1], b.hi[s], b.hi[s + 1]);
                            mma16816(acc[j], lo0[i][s], lo1[i][s], lo0[i][s + 1], lo1[i][s + 1], b.hi[s], b.hi[s + 1]);
                            if constexpr (Fragment<T, kPairs>::kSplit)
                                mma16816(acc[j], hi0[i][s], hi1[i][s], hi0[i][s + 1], hi1[i][s + 1], b.lo[s], b.lo[s + 1]);
                        }
                    }
                }
            }
            if (row0) {
                float v[8] = {acc[0][0], acc[0][1], acc[1][0], acc[1][1], acc[2][0], acc[2][1], acc[3][0], acc[3][1]};
                add_base_and_store<O>(p, t0 + g, n + q * 8, v);
            }
            if (row1) {
                float v[8] = {acc[0][2], acc[0][3], acc[1][2], acc[1][3], acc[2][2], acc[2][3], acc[3][2], acc[3][3]};
                add_base_and_store<O>(p, t0 + g + 8, n + q * 8, v);
            }
        }
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kWantedWarps = 148 * 8;

// How the input features are cut: enough warps to fill the GPU, at least 128 features each, at most 16 partial sums.
Units shrink_units(int64_t tokens, int64_t inner) {
    Units u;
    u.tiles = ceil_div(tokens, kTokens);
    u.subs = 1;
    int64_t parts = ceil_div(kWantedWarps, u.tiles);
    parts = parts < 16 ? parts : 16;
    const int64_t most = ceil_div(inner, 128);
    parts = parts < most ? parts : most;
    u.per_part = ceil_div(ceil_div(inner, parts), 32) * 32;
    u.parts = ceil_div(inner, u.per_part);
    return u;
}

// Distinct adapters a tile may hold: as many as the requests that meet in it, on average.
int sub_count(const AdapterCall& p) {
    const int64_t meet = ceil_div(kTokens * p.requests, p.tokens);
    int subs = 1;
    while (subs < meet && subs < kTokens) subs *= 2;
    return subs;
}

template <typename T, typename O, int kRank>
cudaError_t launch(const AdapterCall& p, cudaStream_t stream) {
    Units shrink = shrink_units(p.tokens, p.inner);
    Units expand = shrink;
    shrink.subs = expand.subs = sub_count(p);
    int64_t parts = ceil_div(kWantedWarps * 2, expand.tiles * expand.subs);
    const int64_t most = p.outer / 32;
    parts = parts < most ? parts : most;
    expand.per_part = ceil_div(most, parts) * 32;
    expand.parts = ceil_div(p.outer, expand.per_part);
    const int64_t shrink_ctas = ceil_div(shrink.tiles * shrink.parts * shrink.subs, kWarps);
    const int64_t expand_ctas = ceil_div(expand.tiles * expand.parts * expand.subs, kWarps);
    if (shrink_ctas > 0x7fffffffll || expand_ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    shrink_kernel<T, kRank><<<(unsigned)shrink_ctas, 32 * kWarps, 0, stream>>>(p, shrink);
    expand_kernel<T, O, kRank><<<(unsigned)expand_ctas, 32 * kWarps, 0, stream>>>(p, expand, shrink.parts);
    return cudaGetLastError();
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
    return shrink_units(tokens, inner).parts * tokens * rank * (int64_t)sizeof(float);
}

cudaError_t launch_adapters(const AdapterCall& p, bool in_bf16, bool out_bf16, cudaStream_t stream) {
    if (p.tokens == 0 || p.outer == 0) return cudaSuccess;
    if (!in_bf16) return out_bf16 ? cudaErrorInvalidValue : by_rank<float, float>(p, stream);
    return out_bf16 ? by_rank<__nv_bfloat16, __nv_bfloat16>(p, stream) : by_rank<__nv_bfloat16, float>(p, stream);
}

}  // namespace bsmm

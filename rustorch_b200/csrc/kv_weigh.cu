// Softmax weights of queries over a bf16 cache, summed into an accumulator:
//   weights[t] += sum over the queries i and heads g that share K of 2^(scale_log2 * q . k_t - lse_log2),  t <= len - seq_q + i.
//
// A warp owns 16 or 32 tokens: their keys are the A operand of mma.sync.m16n8k16 and stay in registers (each lane loads 16
// neighbouring values of a row, which are the k pairs of two products: the order of k is free as long as q has the same),
// while the query rows pass by as B operands, eight at a time.  Every weight has one writer and is touched once.  CTAs walk over
// the tokens that there are: 64 sequences of 1000 tokens, 8 KV heads, D = 128, one query, took 22 us in a cache of 1024 rows and
// 541 in one of 131,072 with a CTA for every 128 rows of cache, and 22 in both so.
//
// What bounds it: with one query a sequence, the keys' bytes; with a prompt's last queries, the exponentials and products.
#include <algorithm>

#include "cache_kernels.h"
#include "kernels.h"
#include "common.cuh"
#include "mma_sync.cuh"

namespace rt {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
// Query rows of a KV head from which kv_weigh_tc.cu's kernel is taken.  Its time hardly depends on their number up to 64.  Here and
// there, us, 8 heads of 16,001 tokens, 128 of 2000 and 128 of 8000:
//     D = 64    32 rows  6.3 |  8.1   10.6 | 12.7    37.0 |  50.6     48 rows   7.6 |  8.2   13.1 | 12.8    45.5 |  50.7
//     D = 128    8 rows  7.1 |  8.8   12.2 | 13.7    48.4 |  56.5     16 rows   8.3 |  8.8   14.4 | 13.8    55.0 |  56.2
//     D = 256   16 rows 16.7 | 13.4   34.5 | 35.3    96.2 | 121.3     24 rows  19.3 | 13.4   39.2 | 35.3   108.2 | 121.5
// (60 rows at D = 64: 9.0 | 8.2, 15.4 | 12.8, 54.1 | 50.6.)  Below, a warp loads its keys and then takes the rows: 28 rows at
// D = 128 waited for the loads half of the time, at 0.4 of the issue rate and 42 % of DRAM's.
__host__ __device__ constexpr int tensor_rows(int head_dim) { return head_dim == 64 ? 48 : head_dim == 128 ? 16 : 24; }

struct WeighParams {
    const __nv_bfloat16 *q, *k;
    const float* lse;
    float* weights;
    int64_t max_seq, seq_q;
    const int32_t* kv_lens;
    int kv_len, n_kv, group;
    float scale_log2;
};

template <int D>
struct WeighShape {
    static constexpr int kTiles = D == 256 ? 1 : 2;  // of 16 tokens a warp: their keys take D / 4 registers a lane each
    static constexpr int kTokens = 16 * kTiles * kWarps;
    static constexpr int kChunks = D / 32;           // 16-byte pieces of a row per lane
    static constexpr int kPitch = 2 * D + 64;        // of a query row in shared memory: two rows fill all banks
};

__device__ __forceinline__ float lse_log2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }
// A row that saw nothing adds nothing, whatever its query holds.
__device__ __forceinline__ float weight(float score, float scale_log2, float lse2) {
    return lse2 == INFINITY ? 0.f : fast_exp2(fmaf(score, scale_log2, -lse2));
}

// Scores of 16 tokens and 8 query rows, as accumulators of (row t = g or g + 8, queries 2j and 2j + 1).
template <int D>
__device__ __forceinline__ void scores(float (&c)[4], const uint4 (&k)[WeighShape<D>::kChunks][2], const uint4 (&q)[WeighShape<D>::kChunks]) {
    c[0] = c[1] = c[2] = c[3] = 0.f;
#pragma unroll
    for (int n = 0; n < WeighShape<D>::kChunks; ++n) {
        const uint32_t a[4] = {k[n][0].x, k[n][1].x, k[n][0].y, k[n][1].y}, b[4] = {k[n][0].z, k[n][1].z, k[n][0].w, k[n][1].w};
        mma_bf16(c, a, q[n].x, q[n].y);
        mma_bf16(c, b, q[n].z, q[n].w);
    }
}

// kSingle: one query a sequence, its rows in registers.
template <int D, bool kSingle>
__global__ void __launch_bounds__(kThreads) kv_weigh_kernel(const WeighParams p) {
    using S = WeighShape<D>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid % 32, g = lane / 4, j = lane % 4;
    const int64_t b = blockIdx.z, bh = b * p.n_kv + blockIdx.y;
    const int len = max(0, (int)min(p.kv_lens ? (int64_t)p.kv_lens[b] : (int64_t)p.kv_len, p.max_seq));
    const int tiles = (len + S::kTokens - 1) / S::kTokens;
    if ((int)blockIdx.x >= tiles) return;
    const int64_t row0 = bh * p.group * p.seq_q;
    // the query rows: one query's in registers, more in shared memory
    constexpr int kRows = kSingle ? 8 : tensor_rows(D);  // as many at least
    static_assert(kRows % 8 == 0, "rows pass by in eights");
    const int rows = p.group * (int)p.seq_q;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) float s_lse[kRows];
    __shared__ int s_last[kRows];  // the last token that a row sees
    uint4 q[S::kChunks];
    float2 l;
    if constexpr (kSingle) {
#pragma unroll
        for (int n = 0; n < S::kChunks; ++n) {
            q[n] = make_uint4(0, 0, 0, 0);
            if (g < rows) q[n] = *reinterpret_cast<const uint4*>(p.q + (row0 + g) * D + 32 * n + 8 * j);
        }
        l.x = 2 * j < rows ? lse_log2(p.lse[row0 + 2 * j]) : INFINITY;
        l.y = 2 * j + 1 < rows ? lse_log2(p.lse[row0 + 2 * j + 1]) : INFINITY;
    } else {
        for (int i = tid; i < kRows * (D / 8); i += kThreads) {
            const int r = i / (D / 8), c = i % (D / 8);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < rows) x = *reinterpret_cast<const uint4*>(p.q + (row0 + r) * D + 8 * c);
            *reinterpret_cast<uint4*>(smem + r * S::kPitch + 16 * c) = x;
        }
        if (tid < kRows) {
            s_lse[tid] = tid < rows ? lse_log2(p.lse[row0 + tid]) : INFINITY;
            s_last[tid] = len - (int)p.seq_q + tid % (int)p.seq_q;
        }
        __syncthreads();
    }
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int t0 = tile * S::kTokens + (tid / 32) * 16 * S::kTiles;
        uint4 k[S::kTiles][S::kChunks][2];
#pragma unroll
        for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int t = t0 + 16 * m + 8 * r + g;
                const __nv_bfloat16* row = p.k + (bh * p.max_seq + min(t, len - 1)) * D + 8 * j;
#pragma unroll
                for (int n = 0; n < S::kChunks; ++n) k[m][n][r] = ld_stream_16B(row + 32 * n);
            }
        float w[S::kTiles][2] = {};
        if constexpr (kSingle) {
#pragma unroll
            for (int m = 0; m < S::kTiles; ++m) {
                float c[4];
                scores<D>(c, k[m], q);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[m][i / 2] += weight(c[i], p.scale_log2, i & 1 ? l.y : l.x);
            }
        } else {
            // the first query's place: whether any row of this warp's tokens can be hidden
            const bool all_seen = t0 + 16 * S::kTiles - 1 <= len - p.seq_q;
            for (int n0 = 0; n0 < rows; n0 += 8) {
#pragma unroll
                for (int n = 0; n < S::kChunks; ++n)
                    q[n] = *reinterpret_cast<const uint4*>(smem + (n0 + g) * S::kPitch + 64 * n + 16 * j);
                l = *reinterpret_cast<const float2*>(&s_lse[n0 + 2 * j]);
#pragma unroll
                for (int m = 0; m < S::kTiles; ++m) {
                    float c[4];
                    scores<D>(c, k[m], q);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float e = weight(c[i], p.scale_log2, i & 1 ? l.y : l.x);
                        if (!all_seen && t0 + 16 * m + 4 * (i & 2) + g > s_last[n0 + 2 * j + (i & 1)]) e = 0.f;
                        w[m][i / 2] += e;
                    }
                }
            }
        }
#pragma unroll
        for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x = w[m][r];
                x += __shfl_xor_sync(kFullMask, x, 1);
                x += __shfl_xor_sync(kFullMask, x, 2);
                const int t = t0 + 16 * m + 8 * r + g;
                if (j == 0 && t < len) p.weights[bh * p.max_seq + t] += x;
            }
    }
}

}  // namespace

int64_t bounded_blocks(int64_t most, int64_t groups, int per_sm) {
    return std::max<int64_t>(1, std::min(most, per_sm * (int64_t)sm_count() / groups));
}

cudaError_t launch_kv_weigh(const void* q, const void* k_cache, const float* lse, float* weights, int64_t batch, int n_heads,
                            int n_kv, int64_t seq_q, int head_dim, int64_t max_seq, const int32_t* kv_lens,
                            int64_t kv_len_uniform, float scale, cudaStream_t stream) {
    WeighParams p;
    p.q = (const __nv_bfloat16*)q, p.k = (const __nv_bfloat16*)k_cache, p.lse = lse, p.weights = weights;
    p.max_seq = max_seq, p.seq_q = seq_q, p.kv_lens = kv_lens, p.kv_len = (int)kv_len_uniform;
    p.n_kv = n_kv, p.group = n_heads / n_kv, p.scale_log2 = scale * kLog2e;
    const int64_t longest = kv_lens ? max_seq : kv_len_uniform;
    if (longest == 0) return cudaSuccess;
    if (p.group * seq_q >= tensor_rows(head_dim))
        return launch_kv_weigh_tc(q, k_cache, lse, weights, batch, n_heads, n_kv, seq_q, head_dim, max_seq, longest, kv_lens, kv_len_uniform,
                                  scale, stream);
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        using S = WeighShape<D>;
        // 48 an SM (32, 64): one query on 64 sequences of 1024 to 8192 tokens, D = 128, 92.6 us (94.5, 91.4); 8 of 1000 in a cache
        // of 131,072 rows 9.6 (7.4, 11.8)
        const dim3 grid((unsigned)bounded_blocks((longest + S::kTokens - 1) / S::kTokens, batch * n_kv, 48), n_kv, (unsigned)batch);
        if (seq_q == 1) return launch_chained(kv_weigh_kernel<D, true>, grid, kThreads, 0, stream, p);
        return launch_chained(kv_weigh_kernel<D, false>, grid, kThreads, (size_t)tensor_rows(D) * S::kPitch, stream, p);
    });
}

}  // namespace rt

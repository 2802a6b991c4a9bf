// Softmax weights of queries over a bf16 cache, summed into an accumulator:
//   weights[t] += sum over the queries i and heads g that share K of exp2(scale_log2 * q . k_t - lse_log2),  t <= len - seq_q + i.
#include "cache_kernels.h"
#include "kernels.h"
#include "common.cuh"

namespace rt {
namespace {

constexpr int kThreads = 128;

struct WeighParams {
    const __nv_bfloat16 *q, *k;
    const float* lse;
    float* weights;
    int64_t max_seq, seq_q;
    const int32_t* kv_lens;
    int kv_len, n_kv, group;
    float scale_log2;
};

// A thread a token; the query rows pass through shared memory one at a time.
template <int D>
__global__ void __launch_bounds__(kThreads) kv_weigh_kernel(const WeighParams p) {
    __shared__ float q[D];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int h = blockIdx.y;
    const int64_t b = blockIdx.z, bh = b * p.n_kv + h;
    const int64_t len = max((int64_t)0, min(p.kv_lens ? (int64_t)p.kv_lens[b] : (int64_t)p.kv_len, p.max_seq));
    const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const __nv_bfloat16* k = p.k + (bh * p.max_seq + min(t, p.max_seq - 1)) * D;
    float w = 0.f;
    for (int64_t r = 0; r < p.group * p.seq_q; ++r) {
        const int64_t row = bh * p.group * p.seq_q + r;
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kThreads) q[d] = __bfloat162float(p.q[row * D + d]);
        __syncthreads();
        const float lse = p.lse[row];
        if (t < len && t <= len - p.seq_q + r % p.seq_q && lse != -INFINITY) {
            float x = 0.f;
            for (int d = 0; d < D; ++d) x = fmaf(q[d], __bfloat162float(k[d]), x);
            w += exp2f(x * p.scale_log2 - lse * kLog2e);
        }
    }
    if (t < len) p.weights[bh * p.max_seq + t] += w;
}

}  // namespace

cudaError_t launch_kv_weigh(const void* q, const void* k_cache, const float* lse, float* weights, int64_t batch, int n_heads,
                            int n_kv, int64_t seq_q, int head_dim, int64_t max_seq, const int32_t* kv_lens,
                            int64_t kv_len_uniform, float scale, cudaStream_t stream) {
    WeighParams p;
    p.q = (const __nv_bfloat16*)q, p.k = (const __nv_bfloat16*)k_cache, p.lse = lse, p.weights = weights;
    p.max_seq = max_seq, p.seq_q = seq_q, p.kv_lens = kv_lens, p.kv_len = (int)kv_len_uniform;
    p.n_kv = n_kv, p.group = n_heads / n_kv, p.scale_log2 = scale * kLog2e;
    const dim3 grid((unsigned)((max_seq + kThreads - 1) / kThreads), n_kv, (unsigned)batch);
    return for_head_dim(head_dim, [&](auto d) {
        return launch_chained(kv_weigh_kernel<decltype(d)::value>, grid, kThreads, 0, stream, p);
    });
}

}  // namespace rt

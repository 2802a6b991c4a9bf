// Launch interface between the C ABI of the 4-bit cache and of eviction (api_cache.cu) and their kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch_chained.h"

namespace rt {

struct Kv4Cache {
    const void *k_codes, *k_scales, *v_codes, *v_scales;  // written by the appends
};

template <class F>
inline cudaError_t for_head_dim(int head_dim, F&& f) {
    switch (head_dim) {
        case 64: return f(std::integral_constant<int, 64>{});
        case 128: return f(std::integral_constant<int, 128>{});
        default: return f(std::integral_constant<int, 256>{});
    }
}

// CTAs of a (sequence, KV head) whose lengths only the device knows, for a launch whose CTAs walk over what there is: one for each
// of `most` pieces of the longest, but no more than `per_sm` an SM of all heads together, since the cache may be much larger than
// what it holds and a CTA without work takes 0.5 to 1 ns of the launch.
int64_t bounded_blocks(int64_t most, int64_t groups, int per_sm);

// ---- kv4_rows.cu
cudaError_t launch_kv4_append(const Kv4Cache& c, const void* k, const void* v, const int64_t* ks, const int64_t* vs,
                              int64_t batch, int n_kv, int64_t rows, int head_dim, int64_t max_seq, int64_t pos,
                              const int32_t* positions, const int32_t* lens, cudaStream_t stream);
cudaError_t launch_rope_kv4_append(const Kv4Cache& c, void* q, const void* k, const void* v, const float* inv_freq,
                                   int64_t batch, int n_heads, int n_kv, int head_dim, int64_t max_seq, int64_t pos,
                                   const int32_t* positions, int64_t slot, const int32_t* slots, int style,
                                   cudaStream_t stream);
cudaError_t launch_kv4_read(const Kv4Cache& c, void* k, void* v, int64_t batch, int n_kv, int head_dim, int64_t max_seq,
                            int64_t rows, int64_t start, const int32_t* starts, const int32_t* kv_lens, cudaStream_t stream);

// ---- kv4_decode.cu
size_t kv4_decode_workspace_bytes(int64_t batch, int n_heads, int n_kv, int head_dim, int64_t max_seq, bool weighed);
cudaError_t launch_kv4_decode(const Kv4Cache& c, const void* q, void* out, float* lse, float* weights, int64_t batch,
                              int n_heads, int n_kv, int head_dim, int64_t max_seq, const int32_t* kv_lens,
                              int64_t kv_len_uniform, float scale, void* workspace, cudaStream_t stream);

// ---- kv_weigh.cu
cudaError_t launch_kv_weigh(const void* q, const void* k_cache, const float* lse, float* weights, int64_t batch, int n_heads,
                            int n_kv, int64_t seq_q, int head_dim, int64_t max_seq, const int32_t* kv_lens,
                            int64_t kv_len_uniform, float scale, cudaStream_t stream);

// ---- kv_weigh_tc.cu: the same on tcgen05, for the rows from which it is faster
cudaError_t launch_kv_weigh_tc(const void* q, const void* k_cache, const float* lse, float* weights, int64_t batch, int n_heads,
                               int n_kv, int64_t seq_q, int head_dim, int64_t max_seq, int64_t longest, const int32_t* kv_lens,
                               int64_t kv_len_uniform, float scale, cudaStream_t stream);

// ---- kv_evict.cu
struct EvictPlanes {
    static constexpr int kMost = 4;
    const void* src[kMost];
    void* dst[kMost];
    int row_bytes[kMost];
    int n;
};
cudaError_t launch_kv_evict(const EvictPlanes& planes, const float* weights, float* weights_out, int32_t* kept,
                            int32_t* lens_out, int64_t batch, int n_kv, int64_t max_seq, int64_t max_seq_out,
                            const int32_t* kv_lens, int64_t kv_len_uniform, int64_t keep, int64_t recent,
                            cudaStream_t stream);

}  // namespace rt

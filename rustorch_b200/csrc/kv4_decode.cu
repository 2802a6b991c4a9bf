// Single-token GQA attention over a 4-bit KV cache.
//
// out = sum_t p_t v_t, p = softmax(scale * q . k_t), with k, v = lo + scale * code per group of 32 values.  A CTA takes an
// equal part of one (sequence, KV head)'s tokens in tiles of 64 with the running maximum and sum of a softmax; the G query
// heads share every row that is read.  The parts' results are merged by their log-sum-exp.
#include "cache_kernels.h"
#include "kernels.h"
#include "kv4.cuh"

namespace rt {
namespace {

constexpr int kTile = 64, kThreads = 128, kMaxGroup = 8;

struct DecodeParams {
    const __nv_bfloat16* q;
    const uint8_t *k_codes, *v_codes;
    const uint32_t *k_scales, *v_scales;
    __nv_bfloat16* out;
    float *lse, *part_o, *part_lse, *weights;
    int64_t max_seq, rows;
    const int32_t* kv_lens;
    int kv_len, n_kv, group, parts;
    float scale_log2;
};

__device__ __forceinline__ int visible(const int32_t* kv_lens, int uniform, int64_t max_seq, int64_t b) {
    return max(0, (int)min(kv_lens ? (int64_t)kv_lens[b] : (int64_t)uniform, max_seq));
}

template <int D>
__device__ __forceinline__ float value_at(const uint8_t* codes, const uint32_t* scales, int64_t row, int d) {
    using R = Kv4Row<D>;
    const uint32_t c = codes[row * R::kCodeBytes + d / 2] >> (4 * (d & 1)) & 15u;
    return kv4_value(kv4_scale(scales[row * R::kGroups + R::group_of_octet(d / 8)]), c);
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_decode_kernel(const DecodeParams p) {
    __shared__ float q[kMaxGroup][D], s[kMaxGroup][kTile], alpha[kMaxGroup], sum[kMaxGroup], top[kMaxGroup];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, h = blockIdx.y, G = p.group;
    const int64_t b = blockIdx.z, bh = b * p.n_kv + h;
    const int len = visible(p.kv_lens, p.kv_len, p.max_seq, b);
    const int size = (len + p.parts - 1) / p.parts;
    const int lo = min(len, (int)blockIdx.x * size), hi = min(len, lo + size);
    for (int i = tid; i < G * D; i += kThreads) q[i / D][i % D] = __bfloat162float(p.q[bh * G * D + i]);
    if (tid < kMaxGroup) sum[tid] = 0.f, top[tid] = -INFINITY;
    constexpr int kPer = (D + kThreads - 1) / kThreads;
    float acc[kPer][kMaxGroup] = {};
    __syncthreads();
    for (int t0 = lo; t0 < hi; t0 += kTile) {
        const int n = min(kTile, hi - t0);
        for (int i = tid; i < G * kTile; i += kThreads) {
            const int g = i / kTile, t = i % kTile;
            float x = -INFINITY;
            if (t < n) {
                x = 0.f;
                for (int d = 0; d < D; ++d) x = fmaf(q[g][d], value_at<D>(p.k_codes, p.k_scales, bh * p.max_seq + t0 + t, d), x);
                x *= p.scale_log2;
            }
            s[g][t] = x;
        }
        __syncthreads();
        for (int g = tid / 32; g < G; g += kThreads / 32) {
            const int lane = tid % 32;
            const float a = s[g][lane], c = s[g][lane + 32], old = top[g];
            float m = fmaxf(fmaxf(a, c), old);
            for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, off));
            const float ref = m == -INFINITY ? 0.f : m;
            const float pa = exp2f(a - ref), pc = exp2f(c - ref);
            float l = pa + pc;
            for (int off = 16; off; off >>= 1) l += __shfl_xor_sync(kFullMask, l, off);
            s[g][lane] = pa, s[g][lane + 32] = pc;
            if (lane == 0) {
                const float f = old == -INFINITY ? 0.f : exp2f(old - ref);
                alpha[g] = f, sum[g] = sum[g] * f + l, top[g] = m;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int d = tid + j * kThreads;
            if (d < D) {
                for (int g = 0; g < kMaxGroup; ++g)
                    if (g < G) acc[j][g] *= alpha[g];
                for (int t = 0; t < n; ++t) {
                    const float v = value_at<D>(p.v_codes, p.v_scales, bh * p.max_seq + t0 + t, d);
                    for (int g = 0; g < kMaxGroup; ++g)
                        if (g < G) acc[j][g] = fmaf(s[g][t], v, acc[j][g]);
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int d = tid + j * kThreads;
        if (d < D)
            for (int g = 0; g < kMaxGroup; ++g)
                if (g < G) {
                    const float o = hi > lo ? acc[j][g] / sum[g] : 0.f;
                    if (p.part_o) p.part_o[((int64_t)blockIdx.x * p.rows + bh * G + g) * D + d] = o;
                    else p.out[(bh * G + g) * D + d] = __float2bfloat16(o);
                }
    }
    if (tid < G) {
        const float l = hi > lo ? top[tid] * kLn2 + logf(sum[tid]) : -INFINITY;
        if (p.part_o) p.part_lse[(int64_t)blockIdx.x * p.rows + bh * G + tid] = l;
        else if (p.lse) p.lse[bh * G + tid] = l;
    }
}

// weights[t] += sum over the group of exp(score - lse), a thread a token.
template <int D>
__global__ void __launch_bounds__(kThreads) kv4_weigh_kernel(const DecodeParams p) {
    __shared__ float q[kMaxGroup][D], lse[kMaxGroup];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, h = blockIdx.y, G = p.group;
    const int64_t b = blockIdx.z, bh = b * p.n_kv + h;
    const int len = visible(p.kv_lens, p.kv_len, p.max_seq, b);
    for (int i = tid; i < G * D; i += kThreads) q[i / D][i % D] = __bfloat162float(p.q[bh * G * D + i]);
    if (tid < G) lse[tid] = p.lse[bh * G + tid] * kLog2e;
    __syncthreads();
    const int t = blockIdx.x * kThreads + tid;
    if (t >= len) return;
    float x[kMaxGroup] = {}, w = 0.f;
    for (int d = 0; d < D; ++d) {
        const float k = value_at<D>(p.k_codes, p.k_scales, bh * p.max_seq + t, d);
        for (int g = 0; g < kMaxGroup; ++g)
            if (g < G) x[g] = fmaf(q[g][d], k, x[g]);
    }
    for (int g = 0; g < kMaxGroup; ++g)
        if (g < G) w += exp2f(x[g] * p.scale_log2 - lse[g]);
    p.weights[bh * p.max_seq + t] += w;
}

// One CTA a row: the parts' results weighed by their log-sum-exp.  A NaN part makes the row NaN.
__global__ void __launch_bounds__(kThreads) kv4_merge_kernel(const DecodeParams p, int dim) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t row = blockIdx.x;
    float top = -INFINITY;
    for (int r = 0; r < p.parts; ++r) top = fmaxf(top, p.part_lse[r * p.rows + row]);
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    for (int r = 0; r < p.parts; ++r) total += expf(p.part_lse[r * p.rows + row] - ref);
    for (int d = threadIdx.x; d < dim; d += kThreads) {
        float o = 0.f;
        for (int r = 0; r < p.parts; ++r)
            o += expf(p.part_lse[r * p.rows + row] - ref) * p.part_o[(r * p.rows + row) * dim + d];
        p.out[row * dim + d] = __float2bfloat16(total == 0.f ? 0.f : o / total);
    }
    if (threadIdx.x == 0 && p.lse) p.lse[row] = ref + logf(total);
}

int parts_of(int64_t batch, int n_kv, int64_t max_seq) {
    const int64_t groups = batch * n_kv, want = (4 * (int64_t)sm_count() + groups - 1) / groups;
    return (int)max((int64_t)1, min(want, (max_seq + kTile - 1) / kTile));
}

}  // namespace

size_t kv4_decode_workspace_bytes(int64_t batch, int n_heads, int n_kv, int head_dim, int64_t max_seq, bool weighed) {
    const int parts = parts_of(batch, n_kv, max_seq);
    const size_t rows = (size_t)batch * n_heads;
    return (parts > 1 ? (size_t)parts * rows * (head_dim + 1) * sizeof(float) : 0) + (weighed ? rows * sizeof(float) : 0);
}

cudaError_t launch_kv4_decode(const Kv4Cache& c, const void* q, void* out, float* lse, float* weights, int64_t batch,
                              int n_heads, int n_kv, int head_dim, int64_t max_seq, const int32_t* kv_lens,
                              int64_t kv_len_uniform, float scale, void* workspace, cudaStream_t stream) {
    DecodeParams p = {};
    p.q = (const __nv_bfloat16*)q;
    p.k_codes = (const uint8_t*)c.k_codes, p.v_codes = (const uint8_t*)c.v_codes;
    p.k_scales = (const uint32_t*)c.k_scales, p.v_scales = (const uint32_t*)c.v_scales;
    p.out = (__nv_bfloat16*)out, p.weights = weights;
    p.max_seq = max_seq, p.rows = batch * n_heads, p.kv_lens = kv_lens, p.kv_len = (int)kv_len_uniform;
    p.n_kv = n_kv, p.group = n_heads / n_kv, p.parts = parts_of(batch, n_kv, max_seq);
    p.scale_log2 = scale * kLog2e;
    float* ws = static_cast<float*>(workspace);
    if (p.parts > 1) {
        p.part_o = ws, p.part_lse = ws + (size_t)p.parts * p.rows * head_dim;
        ws = p.part_lse + (size_t)p.parts * p.rows;
    }
    if (!lse && weights) lse = ws;
    p.lse = lse;
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        cudaError_t e = launch_chained(kv4_decode_kernel<D>, dim3(p.parts, n_kv, (unsigned)batch), kThreads, 0, stream, p);
        if (e == cudaSuccess && p.parts > 1)
            e = launch_chained(kv4_merge_kernel, dim3((unsigned)p.rows), kThreads, 0, stream, p, D);
        if (e == cudaSuccess && weights)
            e = launch_chained(kv4_weigh_kernel<D>, dim3((unsigned)((max_seq + kThreads - 1) / kThreads), n_kv, (unsigned)batch),
                               kThreads, 0, stream, p);
        return e;
    });
}

}  // namespace rt

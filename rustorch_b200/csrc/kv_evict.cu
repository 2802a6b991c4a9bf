// Eviction from a KV cache: which rows stay (the heaviest and the latest), then their move to another cache.
#include <algorithm>

#include "cache_kernels.h"
#include "kernels.h"
#include "common.cuh"

namespace rt {
namespace {

constexpr int kThreads = 1024, kBins = 2048;

struct SelectParams {
    const float* weights;
    float* weights_out;
    int32_t *kept, *lens_out;
    int64_t max_seq, max_seq_out;
    const int32_t* kv_lens;
    int kv_len, n_kv, keep, recent;
};

// A key that orders floats as unsigned integers, -0 as 0 and every NaN above infinity.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive sum over the CTA; `total` the sum of all.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* warps, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(kFullMask, x, off);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int i = 0; i < kThreads / 32; ++i) {
        const uint32_t y = warps[i];
        before += i < warp ? y : 0;
        all += y;
    }
    total = all;
    return x + before;
}

// One CTA a (sequence, KV head): the want-th largest key by its digits of 11, 11 and 10 bits, then one pass in order.
__global__ void __launch_bounds__(kThreads) kv_select_kernel(const SelectParams p) {
    __shared__ uint32_t bins[kBins], warps[kThreads / 32], s_digit, s_above;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x;
    const int64_t b = blockIdx.y, bh = b * p.n_kv + blockIdx.x;
    const int len = (int)max((int64_t)0, min(p.kv_lens ? (int64_t)p.kv_lens[b] : (int64_t)p.kv_len, p.max_seq));
    const int m = min(len, p.keep);
    const float* w = p.weights + bh * p.max_seq;
    float* w_out = p.weights_out + bh * p.max_seq_out;
    int32_t* kept = p.kept + bh * p.keep;
    if (blockIdx.x == 0 && tid == 0) p.lens_out[b] = m;
    for (int i = m + tid; i < p.keep; i += kThreads) kept[i] = -1;
    for (int64_t i = m + tid; i < p.max_seq_out; i += kThreads) w_out[i] = 0.f;
    if (len <= p.keep) {
        for (int i = tid; i < len; i += kThreads) kept[i] = i, w_out[i] = w[i];
        return;
    }
    const int n = len - p.recent;        // candidates
    const int want = p.keep - p.recent;  // of which so many stay
    uint32_t prefix = 0, mask = 0;
    int left = want;  // of the candidates with the prefix
    if (want > 0) {
        const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = shifts[pass];
            const uint32_t digit = (1u << widths[pass]) - 1;
            for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t k = order_key(w[i]);
                if ((k & mask) == prefix) atomicAdd(&bins[k >> shift & digit], 1u);
            }
            __syncthreads();
            // the digit where the count from above reaches `left`: thread i holds bins 2i and 2i+1 from the top
            const uint32_t hi_bin = kBins - 1 - 2 * tid, a = bins[hi_bin], c = bins[hi_bin - 1];
            uint32_t total;
            const uint32_t upto = block_scan(a + c, warps, total), before = upto - a - c;
            if (before < (uint32_t)left && upto >= (uint32_t)left) {
                const bool first = before + a >= (uint32_t)left;
                s_digit = first ? hi_bin : hi_bin - 1;
                s_above = first ? before : before + a;
            }
            __syncthreads();
            prefix |= s_digit << shift;
            mask |= digit << shift;
            left -= (int)s_above;
            __syncthreads();
        }
        // in order: larger keys, and the first `left` equal ones
        uint32_t larger = 0, equal = 0;
        for (int i0 = 0; i0 < n; i0 += kThreads) {
            const int i = i0 + tid;
            const float x = i < n ? w[i] : 0.f;
            const uint32_t k = order_key(x);
            const bool gt = i < n && k > prefix, eq = i < n && k == prefix;
            uint32_t total;
            const uint32_t at = block_scan((uint32_t)gt | (uint32_t)eq << 16, warps, total);
            const uint32_t gt_before = larger + (at & 0xffffu) - gt, eq_before = equal + (at >> 16) - eq;
            if (gt || (eq && eq_before < (uint32_t)left)) {
                const uint32_t to = gt_before + min(eq_before, (uint32_t)left);
                kept[to] = i, w_out[to] = x;
            }
            larger += total & 0xffffu, equal += total >> 16;
        }
    }
    for (int i = tid; i < p.recent; i += kThreads) kept[want + i] = n + i, w_out[want + i] = w[n + i];
}

struct MoveParams {
    EvictPlanes planes;
    const int32_t* kept;
    int64_t max_seq, max_seq_out;
    int keep;
};

// 8 bytes a thread and step; grid: (rows, plane, sequence and head).
__global__ void __launch_bounds__(256) kv_move_kernel(const MoveParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t bh = blockIdx.z;
    const int plane = blockIdx.y, units = p.planes.row_bytes[plane] / 8;
    const uint2* src = static_cast<const uint2*>(p.planes.src[plane]) + bh * p.max_seq * units;
    uint2* dst = static_cast<uint2*>(p.planes.dst[plane]) + bh * p.max_seq_out * units;
    const int32_t* kept = p.kept + bh * p.keep;
    const int64_t all = (int64_t)p.keep * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / units, from = kept[row];
        if (from >= 0) dst[i] = src[from * units + i % units];
    }
}

}  // namespace

cudaError_t launch_kv_evict(const EvictPlanes& planes, const float* weights, float* weights_out, int32_t* kept,
                            int32_t* lens_out, int64_t batch, int n_kv, int64_t max_seq, int64_t max_seq_out,
                            const int32_t* kv_lens, int64_t kv_len_uniform, int64_t keep, int64_t recent,
                            cudaStream_t stream) {
    SelectParams s;
    s.weights = weights, s.weights_out = weights_out, s.kept = kept, s.lens_out = lens_out;
    s.max_seq = max_seq, s.max_seq_out = max_seq_out, s.kv_lens = kv_lens, s.kv_len = (int)kv_len_uniform;
    s.n_kv = n_kv, s.keep = (int)keep, s.recent = (int)recent;
    cudaError_t e = launch_chained(kv_select_kernel, dim3(n_kv, (unsigned)batch), kThreads, 0, stream, s);
    if (e != cudaSuccess) return e;
    MoveParams m;
    m.planes = planes, m.kept = kept, m.max_seq = max_seq, m.max_seq_out = max_seq_out, m.keep = (int)keep;
    int units = 1;
    for (int i = 0; i < planes.n; ++i) units = max(units, planes.row_bytes[i] / 8);
    const unsigned x = (unsigned)min((int64_t)256, (keep * units + 1023) / 1024);
    return launch_chained(kv_move_kernel, dim3(x, planes.n, (unsigned)(batch * n_kv)), 256, 0, stream, m);
}

}  // namespace rt

// Eviction from a KV cache: which rows stay (the heaviest and the latest), then their move to another cache.
//
// Selection: the weight of the last row that stays is found digit by digit (11, 11 and 10 bits of an order-preserving
// integer), by histograms in shared memory; a scan in order then gives every kept row its place.  A cluster of 1 to 8 CTAs
// shares the candidates of a (sequence, KV head): each has an equal run of them in its shared memory, reads the others'
// histograms and counts there, and touches global memory once.  No order of atomics reaches the result: the histograms
// are sums.
#include <algorithm>

#include "cache_kernels.h"
#include "cluster.cuh"
#include "kernels.h"
#include "common.cuh"

namespace rt {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2048, kPasses = 3;
constexpr int kMostCluster = 8;
constexpr int kHeld = 32 * 1024;  // candidates of a CTA that its shared memory holds; longer runs are read again instead

struct SelectParams {
    const float* weights;
    float* weights_out;
    int32_t *kept, *lens_out;
    int64_t max_seq, max_seq_out;
    const int32_t* kv_lens;
    int kv_len, n_kv, keep, recent, cluster, held;  // held: candidates that the launch has shared memory for
};

struct SelectShared {
    uint32_t bins[kPasses][kBins];
    uint32_t larger, equal;  // of this CTA's candidates
    uint64_t warps[kWarps];
    uint32_t digit, above;
};

// A key that orders floats as unsigned integers, -0 as 0 and every NaN above infinity.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive sum over the CTA.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint64_t y = __shfl_up_sync(kFullMask, x, off);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += w < warp ? warps[w] : 0;
    return x;
}

// Of this CTA's candidates (load(0) to load(count - 1), the first of them the row's candidate `first`), those that belong
// to the cluster's `want` heaviest go to their places.
template <class Load>
__device__ __forceinline__ void choose(SelectShared& sh, int C, int rank, int count, int first, int want, int32_t* kept, float* w_out,
                                       Load&& load) {
    const int tid = threadIdx.x;
    constexpr int kBatch = 4;  // loads of a thread in flight
    uint32_t prefix = 0, mask = 0;
    int left = want;  // of the candidates with the prefix
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
        constexpr int shifts[kPasses] = {21, 10, 0}, widths[kPasses] = {11, 11, 10};
        const int shift = shifts[pass];
        const uint32_t digit = (1u << widths[pass]) - 1;
        uint32_t* bins = sh.bins[pass];
        for (int i0 = tid; i0 < count; i0 += kBatch * kThreads) {
            uint32_t k[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) k[u] = order_key(load(min(i0 + u * kThreads, count - 1)));
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (i0 + u * kThreads < count && (k[u] & mask) == prefix) atomicAdd(&bins[k[u] >> shift & digit], 1u);
        }
        if (C > 1) cluster_barrier();
        else __syncthreads();
        // the digit where the count from above reaches `left`: a thread has four bins, from the top
        static_assert(kBins == 4 * kThreads, "four bins a thread");
        const int low = kBins - 4 - 4 * tid;
        uint4 u = *reinterpret_cast<const uint4*>(&bins[low]);
        for (int r = 1; r < C; ++r) {
            const uint4 x = load_remote(reinterpret_cast<const uint4*>(&bins[low]), rank + r < C ? rank + r : rank + r - C);
            u.x += x.x, u.y += x.y, u.z += x.z, u.w += x.w;
        }
        const uint32_t all = u.x + u.y + u.z + u.w;
        const uint32_t upto = (uint32_t)block_scan(all, sh.warps), before = upto - all;
        if (before < (uint32_t)left && upto >= (uint32_t)left) {
            uint32_t above = before;
            int at = 3;
            if (above + u.w < (uint32_t)left) above += u.w, at = 2;
            if (at == 2 && above + u.z < (uint32_t)left) above += u.z, at = 1;
            if (at == 1 && above + u.y < (uint32_t)left) above += u.y, at = 0;
            sh.digit = low + at;
            sh.above = above;
        }
        __syncthreads();
        prefix |= sh.digit << shift;
        mask |= digit << shift;
        left -= (int)sh.above;
    }
    // In order: larger keys, and the first `left` equal ones.  A thread has an odd number of neighbours, so that a warp's
    // reads lie in different banks.
    const int each = ((count + kThreads - 1) / kThreads) | 1;
    const int begin = min(count, tid * each), end = min(count, begin + each);
    uint32_t gt = 0, eq = 0;
#pragma unroll 4
    for (int i = begin; i < end; ++i) {
        const uint32_t k = order_key(load(i));
        gt += k > prefix, eq += k == prefix;
    }
    const uint64_t upto = block_scan((uint64_t)gt << 32 | eq, sh.warps);
    gt = (uint32_t)(upto >> 32) - gt, eq = (uint32_t)upto - eq;  // of the threads before
    if (C > 1) {
        if (tid == kThreads - 1) sh.larger = (uint32_t)(upto >> 32), sh.equal = (uint32_t)upto;
        cluster_barrier();
        for (int r = 0; r < rank; ++r) gt += load_remote(&sh.larger, r), eq += load_remote(&sh.equal, r);
    }
#pragma unroll 4
    for (int i = begin; i < end; ++i) {
        const float v = load(i);
        const uint32_t k = order_key(v);
        if (k > prefix || (k == prefix && eq < (uint32_t)left)) {
            const uint32_t to = gt + min(eq, (uint32_t)left);
            kept[to] = first + i, w_out[to] = v;
        }
        gt += k > prefix, eq += k == prefix;
    }
}

__global__ void __launch_bounds__(kThreads) kv_select_kernel(const SelectParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    SelectShared& sh = *reinterpret_cast<SelectShared*>(smem);
    float* held = reinterpret_cast<float*>(smem + sizeof(SelectShared));
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, C = p.cluster, rank = blockIdx.x % C, h = blockIdx.x / C;
    const int64_t b = blockIdx.y, bh = b * p.n_kv + h;
    const int len = (int)max((int64_t)0, min(p.kv_lens ? (int64_t)p.kv_lens[b] : (int64_t)p.kv_len, p.max_seq));
    const int m = min(len, p.keep);
    const float* w = p.weights + bh * p.max_seq;
    float* w_out = p.weights_out + bh * p.max_seq_out;
    int32_t* kept = p.kept + bh * p.keep;
    const int every = C * kThreads, mine = rank * kThreads + tid;
    if (blockIdx.x == 0 && tid == 0) p.lens_out[b] = m;
    for (int i = m + mine; i < p.keep; i += every) kept[i] = -1;
    for (int64_t i = m + mine; i < p.max_seq_out; i += every) w_out[i] = 0.f;
    if (len <= p.keep) {
        for (int i = mine; i < len; i += every) kept[i] = i, w_out[i] = w[i];
        return;  // the whole cluster does
    }
    const int n = len - p.recent;        // candidates
    const int want = p.keep - p.recent;  // of which so many stay
    for (int i = mine; i < p.recent; i += every) kept[want + i] = n + i, w_out[want + i] = w[n + i];
    if (want == 0) return;
    // this CTA's run of them
    const int run = (n + C - 1) / C, first = min(n, rank * run), count = min(n, first + run) - first;
    const float* x = w + first;
    for (int i = tid; i < kPasses * kBins; i += kThreads) sh.bins[0][i] = 0;
    if (run <= p.held)
        for (int i = tid; i < count; i += kThreads) held[i] = x[i];
    __syncthreads();
    if (run <= p.held) choose(sh, C, rank, count, first, want, kept, w_out, [&](int i) { return held[i]; });
    else choose(sh, C, rank, count, first, want, kept, w_out, [&](int i) { return x[i]; });
    if (C > 1) cluster_barrier();  // nobody leaves while its shared memory is read
}

constexpr int kMoveThreads = 256, kMoveBatch = 4;  // a thread's loads in flight

struct MoveParams {
    EvictPlanes planes;
    const int32_t* kept;
    int64_t max_seq, max_seq_out;
    int keep;
};

// A run of a plane's kept rows of a (sequence, KV head), 16 (or 8) bytes a load.
template <class Unit>
__device__ __forceinline__ void move_rows(const MoveParams& p, int plane, int64_t bh) {
    const unsigned row_bytes = p.planes.row_bytes[plane], units = row_bytes / sizeof(Unit);
    const uint8_t* src = static_cast<const uint8_t*>(p.planes.src[plane]) + bh * p.max_seq * row_bytes;
    uint8_t* dst = static_cast<uint8_t*>(p.planes.dst[plane]) + bh * p.max_seq_out * row_bytes;
    const int32_t* kept = p.kept + bh * p.keep;
    const int64_t all = (int64_t)p.keep * units, first = (int64_t)blockIdx.x * kMoveThreads * kMoveBatch + threadIdx.x;
    int32_t from[kMoveBatch];
    unsigned at[kMoveBatch];
#pragma unroll
    for (int k = 0; k < kMoveBatch; ++k) {
        const int64_t i = first + k * kMoveThreads;
        const int64_t r = i >> 32 ? i / units : (unsigned)i / units;
        at[k] = (unsigned)(i - r * units);
        from[k] = i < all ? kept[r] : -1;
    }
    Unit x[kMoveBatch];
#pragma unroll
    for (int k = 0; k < kMoveBatch; ++k)
        if (from[k] >= 0) x[k] = *reinterpret_cast<const Unit*>(src + (int64_t)from[k] * row_bytes + at[k] * sizeof(Unit));
#pragma unroll
    for (int k = 0; k < kMoveBatch; ++k)
        if (from[k] >= 0) *reinterpret_cast<Unit*>(dst + (first + k * kMoveThreads) * sizeof(Unit)) = x[k];
}

// Grid: (runs of rows, plane, sequence and KV head).
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const MoveParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (p.planes.row_bytes[blockIdx.y] % 16 == 0) move_rows<uint4>(p, blockIdx.y, blockIdx.z);
    else move_rows<uint2>(p, blockIdx.y, blockIdx.z);
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
    // More CTAs a head while each keeps 2048 candidates and all find an SM.  Replayed from a graph, rows of 16 bytes: 8 heads of
    // 131,072 tokens 158 us with one CTA a head, 87.5 with two, 32.8 with four, 26.4 with eight; 30,001: 26.6, 20.3, 17.4 and 18.4;
    // 9000: 13.8, 13.5 and 13.8.
    const int64_t longest = kv_lens ? max_seq : kv_len_uniform;
    int cluster = 1;
    while (cluster < kMostCluster && longest >= 2 * cluster * 2048 && 2 * cluster * batch * n_kv <= sm_count()) cluster *= 2;
    s.cluster = cluster;
    const int64_t run = (longest + cluster - 1) / cluster;
    s.held = run <= kHeld ? (int)run : 0;
    const size_t smem = sizeof(SelectShared) + s.held * sizeof(float);
    cudaError_t e = set_max_dynamic_smem_once<kv_select_kernel>((int)sizeof(SelectShared) + kHeld * (int)sizeof(float));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_kv * cluster), (unsigned)batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    // Not chained to the kernel ahead (8 heads of 30,001 tokens, calls back to back: 37 us a call chained, 29 not).
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kv_select_kernel, s);
    if (e != cudaSuccess) return e;
    MoveParams m;
    m.planes = planes, m.kept = kept, m.max_seq = max_seq, m.max_seq_out = max_seq_out, m.keep = (int)keep;
    int64_t units = 1;
    for (int i = 0; i < planes.n; ++i) units = std::max(units, keep * (planes.row_bytes[i] / (planes.row_bytes[i] % 16 ? 8 : 16)));
    const int64_t per = kMoveThreads * kMoveBatch;
    return launch_chained(kv_move_kernel, dim3((unsigned)((units + per - 1) / per), planes.n, (unsigned)(batch * n_kv)), kMoveThreads, 0,
                          stream, m);
}

}  // namespace rt

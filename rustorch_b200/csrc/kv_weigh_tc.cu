// Softmax weights of many queries over a bf16 cache (a prompt's last ones), on tcgen05:
//   weights[t] += sum over the query rows r that share K of 2^(scale_log2 * q_r . k_t - lse_log2_r),  t <= last(r).
//
// A CTA takes every so many-th tile of 128 tokens of a (sequence, KV head).  A tile's keys are the A operand, blocks of 64
// query rows pass by as B through a ring of four, and the 128 x 64 scores through four TMEM buffers: what is queued there
// covers the load of the next tile's keys and the latency of the rows' loads (worth little by itself: 64 queries on 16,001
// tokens, 32 heads on 8, D = 128, took 24.3 us with rings of two and 24.1 with these; the mask's test compiled apart from
// the blocks without one brought 21.7).  A token is a TMEM lane, so a thread of the four epilogue warps has a token's scores
// to itself: it adds up their exponentials in a register, with the rows' log-sum-exps broadcast from shared memory,
// and writes the token's weight once.  One thread issues all loads and products.  Two CTAs an SM, at D = 256
// one.
//
// What bounds it: no pipe is full.  The exponentials come nearest, 16 a clock and SM (512 clocks a block): that pipe is busy
// for 40 % of the active clocks, and stalls are fixed latency, TMEM reads, shared memory and barriers, in this order.  They are
// ex2's, not a short polynomial's, since the weights are f32 sums.
#include <algorithm>
#include <climits>

#include "cache_kernels.h"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace rt {

// prefill_tc.cu
bool make_tensor_map_bf16_4d(CUtensorMap* map, const void* base, int64_t batch, int64_t heads, int64_t seq, int dim,
                             int64_t stride_b, int64_t stride_h, int64_t stride_row, int box_rows);

namespace {

using namespace ptx;

constexpr int kTile = 128, kRows = 64, kRing = 4;  // tokens of a tile, query rows of a block, blocks in flight
constexpr int kEpilogue = 128, kThreads = kEpilogue + 32;
enum { kToKeys = 501, kToQueries = 502, kToScores = 503, kToBuffer = 504 };  // which bounded wait gave up

struct WeighTcParams {
    const float* lse;
    float* weights;
    int64_t max_seq, seq_q;
    const int32_t* kv_lens;
    int kv_len, n_kv, group;
    float scale_log2;
    int* status;
};

template <int D>
struct WeighTc {
    // 64 columns are a swizzled piece
    static constexpr int kKeys = kTile * D * 2, kKeySub = kTile * 128, kQueries = kRows * D * 2, kQuerySub = kRows * 128, kSubs = D / 64;
    static constexpr int kSmem = kKeys + kRing * kQueries + 1024;  // and their alignment
    static constexpr int kPerSm = 2 * kSmem <= 224 * 1024 ? 2 : 1;  // CTAs that an SM's shared memory holds
};

// Barrier of the epilogue's warps, and whether `x` holds in any of their threads.
__device__ __forceinline__ bool barrier_or(bool x) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, 1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)x), "n"(kEpilogue)
        : "memory");
    return any;
}

// A token's scores of a block of rows: their exponentials into `sum`.  The buffer is handed back once it is in registers.
template <bool kHidden>
__device__ __forceinline__ void add_block(float2 (&sum)[2], uint32_t tmem, const float (&lse)[kRows], const int (&last)[kRows], int t,
                                          float2 scale, uint64_t* buffer_free) {
#pragma unroll
    for (int c0 = 0; c0 < kRows; c0 += 32) {
        uint32_t s[32];
        tmem_ld32(tmem + c0, s);
        tc_wait_ld();
        if (c0 + 32 == kRows) {
            tc_fence_before();
            mbar_arrive(buffer_free);
        }
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            const float4 l = *reinterpret_cast<const float4*>(&lse[c0 + c]);
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale, make_float2(l.x, l.y)),
                         y = __ffma2_rn(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), scale, make_float2(l.z, l.w));
            float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y)), f = make_float2(fast_exp2(y.x), fast_exp2(y.y));
            if (kHidden) {
                const int4 m = *reinterpret_cast<const int4*>(&last[c0 + c]);
                e.x = t > m.x ? 0.f : e.x, e.y = t > m.y ? 0.f : e.y, f.x = t > m.z ? 0.f : f.x, f.y = t > m.w ? 0.f : f.y;
            }
            sum[0] = __fadd2_rn(sum[0], e);
            sum[1] = __fadd2_rn(sum[1], f);
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv_weigh_tc_kernel(const __grid_constant__ CUtensorMap map_k,
                                                               const __grid_constant__ CUtensorMap map_q, const WeighTcParams p) {
    using S = WeighTc<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *s_keys = smem, *s_queries = smem + S::kKeys;
    __shared__ __align__(16) float s_lse[2][kRows];  // negated
    __shared__ __align__(16) int s_last[2][kRows];   // the last token that a row sees
    __shared__ uint64_t keys_full, queries_full[kRing], scores_full[kRing], buffer_free[kRing];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = tid / 32;

    if (tid == 0) {
        mbar_init(&keys_full, 1);
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&queries_full[i], 1);
            mbar_init(&scores_full[i], 1);
            mbar_init(&buffer_free[i], kEpilogue);
        }
        fence_barrier_init();
        fence_proxy_async();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t b = blockIdx.z, bh = b * p.n_kv + blockIdx.y;
    const int len = max(0, (int)min(p.kv_lens ? (int64_t)p.kv_lens[b] : (int64_t)p.kv_len, p.max_seq));
    const int all_tiles = (len + kTile - 1) / kTile;
    if ((int)blockIdx.x >= all_tiles) return;  // the whole CTA
    const int tiles = (all_tiles - blockIdx.x + gridDim.x - 1) / gridDim.x;  // of this CTA
    const int64_t rows = p.group * p.seq_q;
    const int blocks = (int)((rows + kRows - 1) / kRows);
    const int64_t units = (int64_t)tiles * blocks;  // a tile against a block of rows
    if (warp == 4) {
        tmem_alloc(&tmem_slot, kRing * kRows);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // Not before: a CTA of the next kernel that has TMEM and waits for this one must not keep this one's from theirs.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 4) {
        if (elect_one()) {
            int keys_loaded = 0, block_loaded = 0;  // tiles; the next block of rows
            int64_t loaded = 0;                     // blocks of rows
            auto load_keys = [&] {
                const int row = (blockIdx.x + keys_loaded * gridDim.x) * kTile;
                mbar_arrive_expect_tx(&keys_full, S::kKeys);
                for (int s = 0; s < S::kSubs; ++s)
                    tma_load_4d(s_keys + s * S::kKeySub, &map_k, &keys_full, s * 64, row, (int)bh, 0);
                ++keys_loaded;
            };
            auto load_queries = [&] {
                const int slot = loaded % kRing;
                mbar_arrive_expect_tx(&queries_full[slot], S::kQueries);
                for (int s = 0; s < S::kSubs; ++s)
                    tma_load_4d(s_queries + slot * S::kQueries + s * S::kQuerySub, &map_q, &queries_full[slot], s * 64, block_loaded * kRows,
                                (int)bh, 0);
                ++loaded;
                if (++block_loaded == blocks) block_loaded = 0;
            };
            load_keys();
            while (loaded < min((int64_t)kRing, units)) load_queries();
            bool ok = true;
            int tile = 0, block = 0, keys_seen = 0;
            int64_t seen = 0;  // what has landed
            for (int64_t u = 0; u < units; ++u) {
                const uint32_t slot = u % kRing, parity = (u / kRing) & 1;
                if (block == 0) {
                    if (!(ok = mbar_wait(&keys_full, tile & 1, p.status, kToKeys))) break;
                    keys_seen = tile + 1;
                }
                if (!(ok = mbar_wait(&queries_full[slot], parity, p.status, kToQueries))) break;
                seen = u + 1;
                if (u >= kRing && !(ok = mbar_wait(&buffer_free[slot], parity ^ 1, p.status, kToBuffer))) break;
                tc_fence_after();
                constexpr uint32_t idesc = make_idesc_bf16(kTile, kRows, 0, 0);
                const uint32_t a = smem_u32(s_keys), q = smem_u32(s_queries) + slot * S::kQueries;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_ss(tmem + slot * kRows, make_smem_desc_sw128(a + (k / 4) * S::kKeySub + (k % 4) * 32, 16, 1024),
                           make_smem_desc_sw128(q + (k / 4) * S::kQuerySub + (k % 4) * 32, 16, 1024), idesc, k > 0);
                mma_commit(&scores_full[slot]);
                // products that have run have read their operands, and the next ones take the place
                if (u >= 1 && loaded < units) {
                    if (!(ok = mbar_wait(&scores_full[(u - 1) % kRing], ((u - 1) / kRing) & 1, p.status, kToScores))) break;
                    load_queries();
                }
                if (++block == blocks) {
                    block = 0, ++tile;
                    if (keys_loaded < tiles) {
                        if (!(ok = mbar_wait(&scores_full[slot], parity, p.status, kToScores))) break;
                        load_keys();
                    }
                }
            }
            // after a wait that gave up: no copy may land in shared memory that is no longer this CTA's
            if (!ok) {
                if (keys_seen < keys_loaded) mbar_wait(&keys_full, keys_seen & 1, p.status, kToKeys);
                for (int64_t i = seen; i < loaded; ++i) mbar_wait(&queries_full[i % kRing], (i / kRing) & 1, p.status, kToQueries);
            }
        }
        __syncwarp();
    } else {
        const uint32_t lane_sel = (uint32_t)(warp * 32) << 16;
        const float2 scale = make_float2(p.scale_log2, p.scale_log2);
        const float* lse = p.lse + bh * rows;
        auto row_lse = [&](int block) {  // a row a thread; one that saw nothing, or is none, adds nothing
            const int64_t r = (int64_t)block * kRows + tid;
            return tid < kRows && r < rows ? lse[r] : -INFINITY;
        };
        float next = row_lse(0);
        bool ok = true;
        int64_t u = 0;
        for (int tile = 0; tile < tiles; ++tile) {
            const int t0 = (blockIdx.x + tile * gridDim.x) * kTile, t = t0 + tid;
            const bool all_seen = t0 + kTile - 1 <= len - p.seq_q;  // no row hides one of the tile's tokens
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            for (int block = 0; block < blocks; ++block, ++u) {
                const int slot = u % kRing, rows_slot = u & 1;
                bool hidden = !all_seen;
                if (tid < kRows) {  // what the block before last read from these places is two barriers ago
                    const bool none = next == -INFINITY;  // its query may be anything, so that the test and not the exponent hides it
                    s_lse[rows_slot][tid] = none ? 0.f : -next * kLog2e;
                    const unsigned r = (unsigned)block * kRows + tid;
                    s_last[rows_slot][tid] = none ? -1 : all_seen ? INT_MAX : (int)(len - p.seq_q + r % (unsigned)p.seq_q);
                    hidden |= none;
                }
                hidden = barrier_or(hidden);
                next = row_lse(block + 1 < blocks ? block + 1 : 0);
                if (ok) ok = __all_sync(kFullMask, mbar_wait(&scores_full[slot], (u / kRing) & 1, p.status, kToScores));
                if (!ok) continue;  // the other warps' barriers still count on this one
                tc_fence_after();
                // compiled with and without the test
                if (hidden) add_block<true>(sum, tmem + lane_sel + slot * kRows, s_lse[rows_slot], s_last[rows_slot], t, scale, &buffer_free[slot]);
                else add_block<false>(sum, tmem + lane_sel + slot * kRows, s_lse[rows_slot], s_last[rows_slot], t, scale, &buffer_free[slot]);
            }
            if (ok && t < len) p.weights[bh * p.max_seq + t] += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        tmem_dealloc(tmem, kRing * kRows);
    }
}

}  // namespace

cudaError_t launch_kv_weigh_tc(const void* q, const void* k_cache, const float* lse, float* weights, int64_t batch, int n_heads,
                               int n_kv, int64_t seq_q, int head_dim, int64_t max_seq, int64_t longest, const int32_t* kv_lens,
                               int64_t kv_len_uniform, float scale, cudaStream_t stream) {
    const int64_t groups = batch * n_kv, rows = n_heads / n_kv * seq_q;
    // TMA coordinates are 32 bits
    if (groups > 0x7fffffff || rows > 0x7fffff00) return cudaErrorNotSupported;
    CUtensorMap map_k, map_q;
    const int D = head_dim;
    if (!make_tensor_map_bf16_4d(&map_k, k_cache, 1, groups, max_seq, D, groups * max_seq * D, max_seq * D, D, kTile) ||
        !make_tensor_map_bf16_4d(&map_q, q, 1, groups, rows, D, groups * rows * D, rows * D, D, kRows))
        return cudaErrorNotSupported;
    WeighTcParams p;
    p.lse = lse, p.weights = weights, p.max_seq = max_seq, p.seq_q = seq_q, p.kv_lens = kv_lens, p.kv_len = (int)kv_len_uniform;
    p.n_kv = n_kv, p.group = n_heads / n_kv, p.scale_log2 = scale * kLog2e, p.status = device_status_ptr();
    if (!p.status) return cudaErrorInvalidSymbol;
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        // No more CTAs than are resident at a time (one for every tile, or one a head, where these are fewer or more): a second
        // wave of a few waits for all of the first.  The other side is two an SM at every D, rounded up: at D = 256, 256 rows,
        // 8 heads of 16,001 tokens 29.3 and 34.2 us, 12 of 20,000 61.1 and 75.9; D = 128, 56 heads of 8000 62.4 and 83.6.
        const int64_t tiles = (longest + kTile - 1) / kTile, each = std::max<int64_t>(1, WeighTc<D>::kPerSm * sm_count() / groups);
        const dim3 grid((unsigned)(tiles < each ? tiles : each), n_kv, (unsigned)batch);
        const cudaError_t e = set_max_dynamic_smem_once<kv_weigh_tc_kernel<D>>(WeighTc<D>::kSmem);
        if (e != cudaSuccess) return e;
        return launch_chained(kv_weigh_tc_kernel<D>, grid, kThreads, (size_t)WeighTc<D>::kSmem, stream, map_k, map_q, p);
    });
}

}  // namespace rt

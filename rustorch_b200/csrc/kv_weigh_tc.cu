// Softmax weights of many queries over a bf16 cache (a prompt's last ones), on tcgen05:
//   weights[t] += sum over the query rows r that share K of 2^(scale_log2 * q_r . k_t - lse_log2_r),  t <= last(r).
//
// A CTA owns 128 tokens of a (sequence, KV head).  Their keys are the A operand and stay in shared memory, blocks of 128 query
// rows pass by as B through a ring of two, and the 128 x 128 scores through two TMEM buffers.  A token is a TMEM lane, so
// a thread of the four epilogue warps has a token's scores to itself: it adds up their exponentials in a register, with
// the rows' log-sum-exps broadcast from shared memory, and writes the token's weight once.  One warp issues all loads and
// products.  Two CTAs an SM overlap one's set-up and waits with the other's exponentials.
//
// What bounds it: the exponentials, 16 a clock and SM (a block is 1024 clocks of them and 290 of products).  They are ex2's, not
// a short polynomial's, since the weights are f32 sums.  With a window of 64 queries on 16,001 tokens, 32 heads on 8:
// see the launch rule in kv_weigh.cu.
#include "cache_kernels.h"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace rt {

bool make_tensor_map_bf16_3d(CUtensorMap* map, const void* base, int64_t bh, int64_t seq, int dim);  // prefill_tc.cu

namespace {

using namespace ptx;

constexpr int kTile = 128;  // tokens, and query rows of a block
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
    static constexpr int kOperand = kTile * D * 2, kSub = kTile * 64 * 2, kSubs = D / 64;  // 64 columns a swizzled piece
    static constexpr int kSmem = 3 * kOperand + 1024 + 1024 + 2048;  // keys, two query blocks, alignment, barriers, rows
};

template <int D>
__global__ void __launch_bounds__(kThreads) kv_weigh_tc_kernel(const __grid_constant__ CUtensorMap map_k,
                                                               const __grid_constant__ CUtensorMap map_q, const WeighTcParams p) {
    using S = WeighTc<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *s_keys = smem, *s_queries = smem + S::kOperand;
    float* s_lse = reinterpret_cast<float*>(smem + 3 * S::kOperand);  // [2][128], negated
    int* s_last = reinterpret_cast<int*>(s_lse + 2 * kTile);          // [2][128]
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_last + 2 * kTile);
    uint64_t *keys_full = bars, *queries_full = bars + 1, *scores_full = bars + 3, *buffer_free = bars + 5;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 7);
    const int tid = threadIdx.x, warp = tid / 32;

    if (tid == 0) {
        mbar_init(keys_full, 1);
        for (int i = 0; i < 2; ++i) {
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
    const int t0 = blockIdx.x * kTile;
    if (t0 >= len) return;  // the whole CTA
    const int64_t rows = p.group * p.seq_q;
    const int blocks = (int)((rows + kTile - 1) / kTile);
    if (warp == 4) {
        tmem_alloc(tmem_slot, 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Not before: a CTA of the next kernel that has TMEM and waits for this one must not keep this one's from theirs.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 4) {
        if (elect_one()) {
            auto load_queries = [&](int i) {
                mbar_arrive_expect_tx(&queries_full[i & 1], S::kOperand);
                for (int s = 0; s < S::kSubs; ++s)
                    tma_load_3d(s_queries + (i & 1) * S::kOperand + s * S::kSub, &map_q, &queries_full[i & 1], s * 64, i * kTile, (int)bh);
            };
            mbar_arrive_expect_tx(keys_full, S::kOperand);
            for (int s = 0; s < S::kSubs; ++s) tma_load_3d(s_keys + s * S::kSub, &map_k, keys_full, s * 64, t0, (int)bh);
            int loaded = 0;
            for (; loaded < min(2, blocks); ++loaded) load_queries(loaded);
            bool ok = mbar_wait(keys_full, 0, p.status, kToKeys);
            int seen = 0;  // blocks whose loads have landed
            for (int i = 0; i < blocks && ok; ++i) {
                const uint32_t parity = (i >> 1) & 1;
                ok = mbar_wait(&queries_full[i & 1], parity, p.status, kToQueries);
                if (!ok) break;
                seen = i + 1;
                if (i >= 2 && !(ok = mbar_wait(&buffer_free[i & 1], parity ^ 1, p.status, kToBuffer))) break;
                tc_fence_after();
                constexpr uint32_t idesc = make_idesc_bf16(kTile, kTile, 0, 0);
                const uint32_t a = smem_u32(s_keys), q = smem_u32(s_queries) + (i & 1) * S::kOperand;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k / 4) * S::kSub + (k % 4) * 32;
                    mma_ss(tmem + (i & 1) * kTile, make_smem_desc_sw128(a + off, 16, 1024), make_smem_desc_sw128(q + off, 16, 1024),
                           idesc, k > 0);
                }
                mma_commit(&scores_full[i & 1]);
                // the products before these have read their queries: the next block's take the place
                if (i >= 1 && loaded < blocks) {
                    if (!(ok = mbar_wait(&scores_full[(i - 1) & 1], ((i - 1) >> 1) & 1, p.status, kToScores))) break;
                    load_queries(loaded++);
                }
            }
            // after a wait that gave up: no copy may land in shared memory that is no longer this CTA's
            if (!ok) mbar_wait(keys_full, 0, p.status, kToKeys);
            for (int i = seen; i < loaded; ++i) mbar_wait(&queries_full[i & 1], (i >> 1) & 1, p.status, kToQueries);
        }
        __syncwarp();
    } else {
        const uint32_t lane_sel = (uint32_t)(warp * 32) << 16;
        const int t = t0 + tid;
        const bool all_seen = t0 + kTile - 1 <= len - p.seq_q;  // no row of this tile's tokens hides one of them
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 scale = make_float2(p.scale_log2, p.scale_log2);
        const float* lse = p.lse + bh * rows;
        auto row_lse = [&](int i) {  // a row a thread; one that saw nothing, or is none, adds nothing
            const int64_t r = (int64_t)i * kTile + tid;
            return r < rows ? lse[r] : -INFINITY;
        };
        float next = row_lse(0);
        bool ok = true;
        for (int i = 0; i < blocks; ++i) {
            {  // what the block before last read from these places is two barriers ago
                const int64_t r = (int64_t)i * kTile + tid;
                s_lse[(i & 1) * kTile + tid] = next == -INFINITY ? -INFINITY : -next * kLog2e;
                s_last[(i & 1) * kTile + tid] = r < rows ? (int)(len - p.seq_q + r % p.seq_q) : -1;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (i + 1 < blocks) next = row_lse(i + 1);
            if (ok) ok = __all_sync(kFullMask, mbar_wait(&scores_full[i & 1], (i >> 1) & 1, p.status, kToScores));
            if (!ok) continue;  // the other warps' barriers still count on this one
            tc_fence_after();
            const bool hidden = !all_seen || (int64_t)(i + 1) * kTile > rows;
            const float* l_row = s_lse + (i & 1) * kTile;
            const int* last = s_last + (i & 1) * kTile;
#pragma unroll 1
            for (int c0 = 0; c0 < kTile; c0 += 32) {
                uint32_t s[32];
                tmem_ld32(tmem + lane_sel + (i & 1) * kTile + c0, s);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 32; c += 4) {
                    const float4 l = *reinterpret_cast<const float4*>(l_row + c0 + c);
                    const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale, make_float2(l.x, l.y)),
                                 y = __ffma2_rn(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), scale, make_float2(l.z, l.w));
                    float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y)), f = make_float2(fast_exp2(y.x), fast_exp2(y.y));
                    if (hidden) {
                        const int4 m = *reinterpret_cast<const int4*>(last + c0 + c);
                        e.x = t > m.x ? 0.f : e.x, e.y = t > m.y ? 0.f : e.y, f.x = t > m.z ? 0.f : f.x, f.y = t > m.w ? 0.f : f.y;
                    }
                    sum[0] = __fadd2_rn(sum[0], e);
                    sum[1] = __fadd2_rn(sum[1], f);
                }
            }
            tc_fence_before();
            mbar_arrive(&buffer_free[i & 1]);
        }
        if (ok && t < len) p.weights[bh * p.max_seq + t] += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        tmem_dealloc(tmem, 256);
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
    if (!make_tensor_map_bf16_3d(&map_k, k_cache, groups, max_seq, head_dim) || !make_tensor_map_bf16_3d(&map_q, q, groups, rows, head_dim))
        return cudaErrorNotSupported;
    WeighTcParams p;
    p.lse = lse, p.weights = weights, p.max_seq = max_seq, p.seq_q = seq_q, p.kv_lens = kv_lens, p.kv_len = (int)kv_len_uniform;
    p.n_kv = n_kv, p.group = n_heads / n_kv, p.scale_log2 = scale * kLog2e, p.status = device_status_ptr();
    if (!p.status) return cudaErrorInvalidSymbol;
    const dim3 grid((unsigned)((longest + kTile - 1) / kTile), n_kv, (unsigned)batch);
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const cudaError_t e = set_max_dynamic_smem_once<kv_weigh_tc_kernel<D>>(WeighTc<D>::kSmem);
        if (e != cudaSuccess) return e;
        return launch_chained(kv_weigh_tc_kernel<D>, grid, kThreads, (size_t)WeighTc<D>::kSmem, stream, map_k, map_q, p);
    });
}

}  // namespace rt

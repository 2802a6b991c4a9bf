// Single-token GQA attention over a 4-bit KV cache.
//
// out = sum_t p_t v_t, p = softmax(scale * q . k_t), with k, v = lo + scale * code per group of 32 values.  Per group
//     q . k = scale * sum(q * code) + lo * sum(q),        sum_t p_t v_t = sum_t p_t (scale_t code_t) + sum_t p_t lo_t.
// A code in the low bits of a 16-bit half is the f16 subnormal code * 2^-24, which mma.sync multiplies exactly, and so is a
// byte, two codes c0 + 16 c1: nothing is dequantised.  The scale of K goes onto the 16 x 8 products of a group, that of V, as
// a product sums over tokens, onto the probabilities of a group's product.
//
// A probability has f16's 11 bits, its product with a scale 22: it is used in two f16 parts.  One part alone is off by what
// sum(p scale code) and sum(p lo) do not share, and each of these is several times the values' size and cancels the other:
// where scores are nearly equal (a spread of 0.0003 in log2, 20,000 tokens, N(0, 1) values) the result was off by 1.8 %, and
// is by 0.2 now, bf16's own rounding.  A KV head of up to four queries has them twice in the products' eight columns, the
// second time with the second part; with more queries the second part takes products of its own.  64 sequences of 1024 to
// 8192 tokens, 32 heads on 8, D = 128: 84.7 us with one part, 87.9 with two by columns, 90.6 with products.
#include <algorithm>
#include <atomic>

#include "cache_kernels.h"
#include "cluster.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace rt {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kMaxGroup = 8;
constexpr int kStep = 32;    // tokens of a warp's step; the steps of a launch are dealt to its warps in equal runs
constexpr float kLazy = 6.f; // log2 of what a probability may exceed 1 by before the running maximum moves

template <int D>
struct Shape {
    using R = Kv4Row<D>;
    static constexpr int kGroups = R::kGroups, kSpanGroups = R::kSpanGroups, kSpans = D / R::kSpan;
    static constexpr int kRow = D / 2, kScaleRow = D / 8;
    // A row of V lies group by group, 16 bytes each.  Eight rows are read at a time: a pitch of 16 bytes more keeps them in
    // different banks.
    static constexpr int kVPitch = kRow + 16, kVScalePitch = kScaleRow < 16 ? 16 : kScaleRow;
    static constexpr int kKBytes = kStep * kRow, kVBytes = kStep * kVPitch, kScaleBytes = kStep * kScaleRow;
    static constexpr int kStage = kKBytes + kVBytes + kScaleBytes + kStep * kVScalePitch;
    static constexpr int kStages = D == 256 ? 2 : 3;  // steps of a warp in shared memory
    static constexpr int kPerSm = D == 256 ? 2 : 3;   // CTAs resident on an SM
    static constexpr int kSmem = kWarps * kStages * kStage;
    static_assert(kStage % 16 == 0, "copies are of 16 bytes");
};

struct DecodeParams {
    const __nv_bfloat16* q;
    const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    __nv_bfloat16* out;
    float* lse;
    float* weights;
    float* scores;   // [B * Hq, max_seq] scaled scores (log2), where weights are asked for
    float* part_o;   // [2 * workers][group][D]
    float2* part_ml; // [2 * workers][group]: the reference that the part's sums are relative to (log2), the sum of its weights
    int2* spans;     // [B * Hkv]: the first part of each and the worker that has the last one; x = -1 where there are no parts
    int64_t max_seq;
    const int32_t* kv_lens;
    int kv_len, batch, n_kv, group, workers;  // workers: warps that take a run of steps
    float scale_log2;
};

__device__ __forceinline__ int visible(const DecodeParams& p, int b) {
    return max(0, (int)min(p.kv_lens ? (int64_t)p.kv_lens[b] : (int64_t)p.kv_len, p.max_seq));
}
// A sequence without tokens has one step too: somebody has to write its zeros.
__device__ __forceinline__ int steps_of(int len) { return max(1, (len + kStep - 1) / kStep); }

// Steps are numbered sequence by sequence, KV head by KV head; worker i takes [i * all / workers, (i + 1) * all / workers),
// with no more workers than steps, so that every one has a part.
__device__ __forceinline__ int64_t share_start(int64_t i, int64_t all, int workers) { return i * all / workers; }

// Steps of all sequences, for all threads of the CTA.
__device__ __forceinline__ int64_t count_steps(const DecodeParams& p) {
    if (!p.kv_lens) return (int64_t)steps_of(visible(p, 0)) * p.batch * p.n_kv;
    __shared__ int64_t sums[kWarps];
    int64_t x = 0;
    for (int b = threadIdx.x; b < p.batch; b += kThreads) x += steps_of(visible(p, b));
#pragma unroll
    for (int off = 16; off; off >>= 1) x += __shfl_xor_sync(kFullMask, x, off);
    if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += sums[w];
    return x * p.n_kv;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(b));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // 8x8 matrix of 16-bit values, a row's pair a lane
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t rest_half2(uint32_t a, uint32_t b, uint32_t ab) {  // a b - ab
    const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              __hneg2(*reinterpret_cast<const __half2*>(&ab)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t max_half2(uint32_t a, uint32_t b) {
    const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t power_half2(int k) { return (uint32_t)(15 + k) * 0x04000400u; }  // 2^k twice, -15 < k < 16
__device__ __forceinline__ float low_half(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }

// Asynchronous copy of kBytes; `there` false writes zeros (and reads nothing).
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t to, const uint8_t* from, bool there) {
    const int n = there ? kBytes : 0;
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(to), "l"(from), "r"(n), "n"(kBytes) : "memory");
}

// kWords neighbouring words of shared memory.
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t (&w)[kWords], const uint8_t* p) {
    if constexpr (kWords == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x, w[1] = x.y;
    }
}

// One (sequence, KV head)'s queries as the B operand of the score products: lane (g, j) = (lane / 4, lane % 4) holds query
// g's octets of quarter j; with kTwice, queries 0 to 3 again as 4 to 7.  The queries are scaled by a power of two that brings
// their largest value to 2^14, where bf16's 8 bits fit f16 exactly down to 2^-31 of the largest, and to 2^-27 at the odd
// places, which are held 16 times smaller.  Smaller values are off by half of f16's last place at most, 2^-35 of the largest there.
template <int D>
struct Queries {
    uint32_t even[Shape<D>::kGroups][2], odd[Shape<D>::kGroups][2];  // pairs (0,4), (2,6) and (1,5)/16, (3,7)/16 of an octet
    uint32_t sums[Shape<D>::kSpans];     // lane j's group of a span: its sum / 64 in two f16 parts, 22 bits
    float factor[2];                     // scale_log2 * 2^24 / the power of two, of queries 2j and 2j + 1

    template <bool kTwice>
    __device__ __forceinline__ void load(const DecodeParams& p, int64_t bh, int lane) {
        using S = Shape<D>;
        const int g = kTwice ? lane / 4 % 4 : lane / 4, j = lane % 4;
        uint4 raw[S::kGroups];
        float top = 0.f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < S::kGroups; ++i) {
            const int octet = (i / S::kSpanGroups) * S::R::kSpanOctets + j * S::kSpanGroups + i % S::kSpanGroups;
            raw[i] = make_uint4(0, 0, 0, 0);
            if (g < p.group) raw[i] = *reinterpret_cast<const uint4*>(p.q + (bh * p.group + g) * D + 8 * octet);
            const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = bf16x2_to_float2(u[k]);
                top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                nan |= f.x != f.x || f.y != f.y;
            }
        }
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
        const int e = top > 0.f && top < INFINITY ? 14 - (((int)(__float_as_uint(top) >> 23) & 255) - 127) : 0;
        // 2^e in two factors: e may be past f32's exponents
        const float up0 = __uint_as_float((uint32_t)(127 + e / 2) << 23), up1 = __uint_as_float((uint32_t)(127 + e - e / 2) << 23);
        float total[S::kGroups];
#pragma unroll
        for (int i = 0; i < S::kGroups; ++i) {
            const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float x[8];
            total[i] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = bf16x2_to_float2(u[k]);
                x[2 * k] = f.x * up0 * up1, x[2 * k + 1] = f.y * up0 * up1;
                total[i] += x[2 * k] + x[2 * k + 1];
            }
            total[i] += __shfl_xor_sync(kFullMask, total[i], 1);
            total[i] += __shfl_xor_sync(kFullMask, total[i], 2);
            even[i][0] = pack_half2(x[0], x[4]), even[i][1] = pack_half2(x[2], x[6]);
            odd[i][0] = pack_half2(x[1] * 0.0625f, x[5] * 0.0625f), odd[i][1] = pack_half2(x[3] * 0.0625f, x[7] * 0.0625f);
        }
#pragma unroll
        for (int s = 0; s < S::kSpans; ++s) {
            float t = 0.f;  // lane j's group of the span
#pragma unroll
            for (int i = 0; i < S::kSpanGroups; ++i) t = j == i ? total[s * S::kSpanGroups + i] * 0.015625f : t;
            sums[s] = pack_half2(t, t - __half2float(__float2half_rn(t)));
        }
        // NaN and infinite queries: the row is NaN whatever the codes are
        float f = nan || top == INFINITY ? __uint_as_float(0x7fffffffu) : p.scale_log2 * exp2f((float)(24 - e));
        nan = (__ballot_sync(kFullMask, nan) >> (lane & ~3)) & 15u;
        if (nan) f = __uint_as_float(0x7fffffffu);
        factor[0] = __shfl_sync(kFullMask, f, 8 * j);
        factor[1] = __shfl_sync(kFullMask, f, 8 * j + 4);
    }
};

// What a warp has summed so far.  Lane (g, j) holds queries 2j and 2j + 1.  With kTwice the lanes j < 2 hold the sums of the
// products' first parts and j + 2 those of the second ones in `o`; all else is the same in both.
template <int D>
struct Sums {
    float o[D / 32][2][4];       // [group][0-1, 2-3 of a lane's four dims]: sum p scale c 2^(k - 24), {q 2j, 2j+1} x {c0, c0 + 16 c1}
    float lo[4], lo2[4];         // sum p * lo: row 2i + 1 = group i; see `step` for which of the rows count
    float ref[2], top[2], l[2];  // p = 2^(score - ref); running maximum; sum of p (this lane's tokens)
    // Of the lanes g = 2i, group i of each span: its scales are held times 2^k, which has the largest so far in [1/2, 1) (the
    // format's are below 2^14), k <= 15, and scale_limit is the largest f16 pattern for which k stands.  Other lanes' limit is
    // never passed.
    int k[D / Kv4Row<D>::kSpan];
    uint32_t scale_limit[D / Kv4Row<D>::kSpan];

    __device__ __forceinline__ void start(int lane) {
        *this = {};
        top[0] = top[1] = -INFINITY;
#pragma unroll
        for (uint32_t& limit : scale_limit) limit = lane / 4 % 2 || lane / 8 >= Kv4Row<D>::kSpanGroups ? 0xffffu : 0u;
    }
};
constexpr float kBase = 15.f - kLazy;  // log2 of what p is held times: the largest reaches 2^15

__device__ __forceinline__ void load_transposed(uint32_t (&r)[4], uint32_t at) {  // four 8x8 matrices of 16-bit values
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

// 32 tokens (valid of them) that lie in shared memory.  scores: [query][max_seq] from this step's first token on, or null.
template <int D, bool kTwice>
__device__ __forceinline__ void step(const uint8_t* stage, int valid, const Queries<D>& q, Sums<D>& a, int lane, float* scores,
                                     int64_t max_seq, int group) {
    using S = Shape<D>;
    const int g = lane / 4, j = lane % 4;
    const uint8_t *kc = stage, *vc = stage + S::kKBytes, *ks = vc + S::kVBytes, *vs = ks + S::kScaleBytes;
    float x[2][4];
#pragma unroll
    for (int tb = 0; tb < 2; ++tb) {
        const int r0 = tb * 16 + g, r1 = r0 + 8;
        float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < S::kSpans; ++s) {  // sum(q) * lo: lane j brings its group
            const int at = (s * S::kSpanGroups + (j & (S::kSpanGroups - 1))) * 4;
            const uint32_t a0 = __byte_perm(*reinterpret_cast<const uint32_t*>(ks + r0 * S::kScaleRow + at), 0, 0x3232),
                           a1 = __byte_perm(*reinterpret_cast<const uint32_t*>(ks + r1 * S::kScaleRow + at), 0, 0x3232);
            mma_f16_k8(m, a0, a1, q.sums[s]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) x[tb][k] = m[k] * 3.814697265625e-06f;  // 64 * 2^-24
#pragma unroll
        for (int s = 0; s < S::kSpans; ++s) {
            uint32_t w0[S::kSpanGroups], w1[S::kSpanGroups], s0[S::kSpanGroups], s1[S::kSpanGroups];
            // at D = 256 odd rows have their spans swapped, so that two rows fill all banks
            const int swap = S::kSpans == 2 ? (g & 1) : 0;
            load_words(w0, kc + r0 * S::kRow + (s ^ swap) * 64 + j * 4 * S::kSpanGroups);
            load_words(w1, kc + r1 * S::kRow + (s ^ swap) * 64 + j * 4 * S::kSpanGroups);
            load_words(s0, ks + r0 * S::kScaleRow + s * 4 * S::kSpanGroups);
            load_words(s1, ks + r1 * S::kScaleRow + s * 4 * S::kSpanGroups);
#pragma unroll
            for (int i = 0; i < S::kSpanGroups; ++i) {
                const int gi = s * S::kSpanGroups + i;
                float c[4];
                mma_f16_first(c, w0[i] & 0x000f000fu, w1[i] & 0x000f000fu, w0[i] & 0x00f000f0u, w1[i] & 0x00f000f0u, q.even[gi][0],
                              q.odd[gi][0]);
                const uint32_t h0 = w0[i] >> 8, h1 = w1[i] >> 8;
                mma_f16(c, h0 & 0x000f000fu, h1 & 0x000f000fu, h0 & 0x00f000f0u, h1 & 0x00f000f0u, q.even[gi][1], q.odd[gi][1]);
                const float f0 = low_half(s0[i]), f1 = low_half(s1[i]);
                x[tb][0] = fmaf(f0, c[0], x[tb][0]), x[tb][1] = fmaf(f0, c[1], x[tb][1]);
                x[tb][2] = fmaf(f1, c[2], x[tb][2]), x[tb][3] = fmaf(f1, c[3], x[tb][3]);
            }
        }
    }
    if (valid < kStep) {
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (tb * 16 + g + 4 * (k & 2) >= valid) x[tb][k] = -INFINITY;
    }
    if (scores) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
            if (2 * j + c < group) {
                float* row = scores + (2 * j + c) * max_seq;
#pragma unroll
                for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        if (tb * 16 + 8 * r + g < valid) row[tb * 16 + 8 * r + g] = x[tb][2 * r + c] * q.factor[c];
            }
    }
    // V and its scales come transposed: 16-bit unit g of a row (4 codes of a group, or a scale or minimum) to the lanes g, those
    // of tokens 2j and 2j + 1 in one register.
    // The scales of D = 256 are four matrices for 16 tokens, spans as rows 0-7 and 8-15 of one operand.  Else they are one
    // for 8 tokens: those of 32 tokens make an operand whose rows 0-7 count in the product with the tokens 0-7 and 16-23,
    // and rows 8-15 in that with the others.
    const uint32_t s_at = (uint32_t)__cvta_generic_to_shared(vs) +
                          (S::kSpans == 2 ? ((lane & 7) + (lane >> 4) * 8) * S::kVScalePitch + (lane >> 3 & 1) * 16 : lane * S::kVScalePitch);
    uint32_t vw[S::kSpans][4];
#pragma unroll
    for (int m = 0; m < S::kSpans; ++m) load_transposed(vw[m], s_at + m * 16 * S::kVScalePitch);
    uint32_t big[S::kSpans];  // the largest scale of V of this lane's group and tokens, of each span
    bool larger = false;
#pragma unroll
    for (int s = 0; s < S::kSpans; ++s) {
        constexpr int kLast = S::kSpans - 1;
        const uint32_t m = S::kSpans == 2 ? max_half2(max_half2(vw[0][s], vw[0][2 + s]), max_half2(vw[kLast][s], vw[kLast][2 + s]))
                                          : max_half2(max_half2(vw[0][0], vw[0][1]), max_half2(vw[0][2], vw[0][3]));
        big[s] = max(m & 0xffffu, m >> 16);
        larger |= big[s] > a.scale_limit[s];
    }
    float top[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        float m = fmaxf(fmaxf(x[0][c], x[0][c + 2]), fmaxf(x[1][c], x[1][c + 2]));
        m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 4));
        m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 8));
        top[c] = fmaxf(m, __shfl_xor_sync(kFullMask, m, 16)) * q.factor[c];
    }
    if (__any_sync(kFullMask, top[0] > a.top[0] + kLazy || top[1] > a.top[1] + kLazy || larger)) {
        float grow[S::kSpans];  // of the scales of this lane's group
#pragma unroll
        for (int s = 0; s < S::kSpans; ++s) {
            uint32_t most = max(big[s], __shfl_xor_sync(kFullMask, big[s], 1));
            most = max(most, __shfl_xor_sync(kFullMask, most, 2));
            grow[s] = 1.f;
            if (most > a.scale_limit[s]) {
                const int e = (int)(__float_as_uint(low_half(most)) >> 23) - 127, k = max(-14, min(-1 - e, 15));
                grow[s] = exp2f((float)(k - a.k[s]));
                a.k[s] = k;
                a.scale_limit[s] = (uint32_t)__half_as_ushort(__float2half_rn(exp2f((float)(e + 1)))) - 1;
            }
        }
        float alpha[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const bool first = a.top[c] == -INFINITY;
            a.top[c] = fmaxf(a.top[c], top[c]);
            const float ref = a.top[c] == -INFINITY ? 0.f : a.top[c] - kBase;
            alpha[c] = first ? 1.f : exp2f(a.ref[c] - ref);
            a.ref[c] = ref;
            a.l[c] *= alpha[c];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) a.lo[k] *= alpha[k & 1], a.lo2[k] *= alpha[k & 1];
#pragma unroll
        for (int i = 0; i < S::kGroups; ++i) {
            const float more = __shfl_sync(kFullMask, grow[i / S::kSpanGroups], 8 * (i % S::kSpanGroups));
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) a.o[i][t][k] *= alpha[k & 1] * more;
        }
    }
    uint32_t prob[2][2];  // query g, tokens 2j, 2j + 1 (and 8 more) of a block of 16
#pragma unroll
    for (int tb = 0; tb < 2; ++tb) {
        float e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            e[k] = fast_exp2(fmaf(x[tb][k], q.factor[k & 1], -a.ref[k & 1]));
            a.l[k & 1] += e[k];
        }
        // rounded to f16's 11 bits, an eighth of the result's own rounding to bf16
        prob[tb][0] = transposed(pack_half2(e[0], e[1]));
        prob[tb][1] = transposed(pack_half2(e[2], e[3]));
    }
    const uint32_t rest = kTwice && g < 4 ? 0u : 0xffffffffu;  // 0: this lane's column takes the first parts
    const uint32_t v_at = (uint32_t)__cvta_generic_to_shared(vc) + (lane & 15) * S::kVPitch + (lane >> 4) * 16;
    uint32_t f[2][2][S::kSpans];  // [16 tokens][8 tokens][span]
    if constexpr (S::kSpans == 2) {
        const uint32_t up[2] = {power_half2(a.k[0]), power_half2(a.k[1])};
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
            const uint32_t(&w)[4] = vw[tb];
            mma_f16(a.lo, w[0], w[1], w[2], w[3], prob[tb][0], prob[tb][1]);
#pragma unroll
            for (int k = 0; k < 4; ++k) f[tb][k / 2][k % 2] = mul_half2(w[k], up[k % 2]);
        }
    } else {
        const uint32_t up = power_half2(a.k[0]);
        const uint32_t(&w)[4] = vw[0];
        mma_f16(a.lo, w[0], w[1], w[2], w[3], prob[0][0], prob[1][0]);
        mma_f16(a.lo2, w[0], w[1], w[2], w[3], prob[0][1], prob[1][1]);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k / 2][k % 2][0] = mul_half2(w[k], up);
    }
#pragma unroll
    for (int tb = 0; tb < 2; ++tb) {
#pragma unroll
        for (int gi = 0; gi < S::kGroups; gi += 2) {
            uint32_t w[4];  // group gi, tokens 0-7 and 8-15; group gi + 1
            load_transposed(w, v_at + tb * 16 * S::kVPitch + gi * 16);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int s = (gi + c) / S::kSpanGroups, from = 8 * ((gi + c) % S::kSpanGroups) + j;
                const uint32_t f0 = __shfl_sync(kFullMask, f[tb][0][s], from), f1 = __shfl_sync(kFullMask, f[tb][1][s], from);
                uint32_t b0 = mul_half2(prob[tb][0], f0), b1 = mul_half2(prob[tb][1], f1);
                // what they were rounded by (exact), or, of a column with the first parts, themselves
                const uint32_t r0 = rest_half2(prob[tb][0], f0, b0 & rest), r1 = rest_half2(prob[tb][1], f1, b1 & rest);
                if (kTwice) b0 = r0, b1 = r1;
                const uint32_t u0 = w[2 * c], u1 = w[2 * c + 1], x0 = __byte_perm(u0, 0, 0x4341), x1 = __byte_perm(u1, 0, 0x4341);
                mma_f16(a.o[gi + c][0], u0 & 0x000f000fu, u0 & 0x00ff00ffu, u1 & 0x000f000fu, u1 & 0x00ff00ffu, b0, b1);
                mma_f16(a.o[gi + c][1], x0 & 0x000f000fu, x0, x1 & 0x000f000fu, x1, b0, b1);
                if (!kTwice) {
                    mma_f16(a.o[gi + c][0], u0 & 0x000f000fu, u0 & 0x00ff00ffu, u1 & 0x000f000fu, u1 & 0x00ff00ffu, r0, r1);
                    mma_f16(a.o[gi + c][1], x0 & 0x000f000fu, x0, x1 & 0x000f000fu, x1, r0, r1);
                }
            }
        }
    }
}

// A lane's places in the planes: the step's bytes are contiguous, neighbouring pieces a lane and copy.
struct LanePlanes {
    const uint8_t *k, *v, *ks, *vs;
};

// A warp's copies of 32 tokens, `valid` of them, into a stage.  Rows behind them become zeros.
template <int D>
__device__ __forceinline__ void fetch(uint32_t to, const LanePlanes& from, int64_t token, int valid, int lane) {
    using S = Shape<D>;
    constexpr int kChunks = S::kRow / 16, kWords = S::kRow / 4;  // of a row's codes
    constexpr int kPiece = S::kScaleRow < 16 ? S::kScaleRow : 16, kPieces = S::kScaleRow / kPiece;
    const int r = lane / kChunks, c = lane % kChunks, rv = lane / kWords, o = lane % kWords, rs = lane / kPieces;
    // at D = 256 odd rows have their spans swapped
    const uint32_t k_to = to + r * S::kRow + (S::kSpans == 2 ? c ^ ((r & 1) << 2) : c) * 16;
    // V word by word: octet o of a row is a group's word (o % kSpanOctets) / kSpanGroups
    const uint32_t v_to = to + S::kKBytes + rv * S::kVPitch + S::R::group_of_octet(o) * 16 + (o % S::R::kSpanOctets) / S::kSpanGroups * 4;
    const uint32_t ks_to = to + S::kKBytes + S::kVBytes + lane * kPiece;
    const uint32_t vs_to = to + S::kKBytes + S::kVBytes + S::kScaleBytes + rs * S::kVScalePitch + lane % kPieces * kPiece;
    const uint8_t *k = from.k + token * S::kRow, *v = from.v + token * S::kRow;
    const uint8_t *ks = from.ks + token * S::kScaleRow, *vs = from.vs + token * S::kScaleRow;
    static_assert((32 / kChunks) % 2 == 0, "a row's parity is the same in all copies of a lane");
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
        constexpr int kRows = 32 / kChunks;
        const bool there = valid >= kStep || r + n * kRows < valid;
        copy_async<16>(k_to + n * kRows * S::kRow, there ? k + n * 512 : from.k - lane * 16, there);
    }
#pragma unroll
    for (int n = 0; n < kWords; ++n) {
        constexpr int kRows = 32 / kWords;
        const bool there = valid >= kStep || rv + n * kRows < valid;
        copy_async<4>(v_to + n * kRows * S::kVPitch, there ? v + n * 128 : from.v - lane * 4, there);
    }
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
        constexpr int kRows = 32 / kPieces;
        const bool there = valid >= kStep || rs + n * kRows < valid;
        copy_async<kPiece>(ks_to + n * 32 * kPiece, there ? ks + n * 32 * kPiece : from.ks - lane * kPiece, there);
        copy_async<kPiece>(vs_to + n * kRows * S::kVScalePitch, there ? vs + n * 32 * kPiece : from.vs - lane * kPiece, there);
    }
}

// A warp's sums as rows: row(query, dim, four neighbouring dims, sum of p), and once a query total(query, reference, sum of p).
// They are relative to 2^reference and not yet divided.
template <int D, bool kTwice, class Row, class Total>
__device__ __forceinline__ void results(const Sums<D>& a, int lane, Row&& row, Total&& total) {
    using S = Shape<D>;
    const int g = lane / 4, j = lane % 4;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        float l = a.l[c];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(kFullMask, l, off);
#pragma unroll
        for (int i = 0; i < S::kGroups; ++i) {
            const int k = __shfl_sync(kFullMask, a.k[i / S::kSpanGroups], 8 * (i % S::kSpanGroups));
            const float even = exp2f((float)(24 - k)), odd = even * 0.0625f;
            // the minima's sum of the group is with the lanes 2i + 1
            const float sum = S::kSpans == 2 ? a.lo[c + 2 * (i / S::kSpanGroups)] : a.lo[c];
            float y = __shfl_sync(kFullMask, sum, 8 * (i % S::kSpanGroups) + 4 + j);
            if (S::kSpans == 1) y += __shfl_sync(kFullMask, a.lo2[c + 2], 8 * i + 4 + j);
            const int d = (i / S::kSpanGroups) * S::R::kSpan + (g >> 1) * (S::R::kSpan / 4) + 8 * (i % S::kSpanGroups) + 4 * (g & 1);
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[k] = a.o[i][k / 2][c + k % 2 * 2];
                if (kTwice) o[k] += __shfl_xor_sync(kFullMask, o[k], 2);
            }
            row(2 * j + c, d, make_float4(fmaf(o[0], even, y), fmaf(o[1] - o[0], odd, y), fmaf(o[2], even, y), fmaf(o[3] - o[2], odd, y)), l);
        }
        if (g == 0) total(2 * j + c, a.ref[c], l);
    }
}

// A warp is a worker: its run of steps may begin and end inside a (sequence, KV head) and pass over several.  What it has of
// one that others work on too is a part for the merge kernel: part 2 i of worker i is what its run begins with, 2 i + 1
// what it ends with.
template <int D, bool kTwice>
__global__ void __launch_bounds__(kThreads, Shape<D>::kPerSm) kv4_decode_kernel(const DecodeParams p) {
    using S = Shape<D>;
    constexpr int kStages = S::kStages;
    extern __shared__ __align__(16) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, G = p.group;
    const int64_t all = count_steps(p);
    const int workers = (int)min((int64_t)p.workers, all);
    const int worker = warp * gridDim.x + blockIdx.x;  // a launch of few spreads them over the SMs
    if (worker >= workers) return;
    int64_t at = share_start(worker, all, workers);
    const int64_t end = share_start(worker + 1, all, workers);
    // the sequence of the first step
    int b = 0;
    int64_t first = 0;  // its first step
    if (!p.kv_lens) {
        const int64_t n = (int64_t)steps_of(visible(p, 0)) * p.n_kv;
        b = (int)(at / n), first = b * n;
    } else {
        for (int b0 = 0;; b0 += 32) {
            const int64_t n = b0 + lane < p.batch ? (int64_t)steps_of(visible(p, b0 + lane)) * p.n_kv : 0;
            int64_t upto = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int64_t y = __shfl_up_sync(kFullMask, upto, off);
                if (lane >= off) upto += y;
            }
            const unsigned owner = __ballot_sync(kFullMask, first + upto > at);
            if (owner || b0 + 32 >= p.batch) {
                const int o = owner ? __ffs(owner) - 1 : 31;
                b = b0 + o, first += __shfl_sync(kFullMask, upto - n, o);
                break;
            }
            first += __shfl_sync(kFullMask, upto, 31);
        }
    }
    uint8_t* ring = smem + warp * kStages * S::kStage;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    constexpr int kPiece = S::kScaleRow < 16 ? S::kScaleRow : 16;
    const LanePlanes planes{p.k_codes + lane * 16, p.v_codes + lane * 4, p.k_scales + lane * kPiece, p.v_scales + lane * kPiece};
    for (bool head = true; at < end; head = false) {
        const int len = visible(p, b), n = steps_of(len);
        const int h = (int)((at - first) / n), step0 = (int)((at - first) % n);
        const int steps = (int)min(end - at, (int64_t)(n - step0));
        const int lo = step0 * kStep, hi = min(len, lo + steps * kStep);
        const int64_t bh = (int64_t)b * p.n_kv + h, rows = bh * p.max_seq;
        auto prefetch = [&](int s, int slot) {
            const int valid = hi - lo - s * kStep;
            const uint32_t to = ring_at + slot * S::kStage;
            if (valid >= kStep) fetch<D>(to, planes, rows + lo + s * kStep, kStep, lane);  // compiled without the tests
            else if (valid > 0) fetch<D>(to, planes, rows + lo + s * kStep, valid, lane);
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncwarp();  // all lanes are done with what lies in the ring
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) prefetch(i, i);
        Queries<D> q;
        q.template load<kTwice>(p, bh, lane);
        Sums<D> a;
        a.start(lane);
        int slot = 0;
        for (int t0 = lo, s = 0; t0 < hi; t0 += kStep, ++s) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            int next = slot + kStages - 1;
            if (next >= kStages) next -= kStages;
            prefetch(s + kStages - 1, next);
            step<D, kTwice>(ring + slot * S::kStage, hi - t0, q, a, lane, p.scores ? p.scores + rows * G + t0 : nullptr, p.max_seq, G);
            if (++slot == kStages) slot = 0;
        }
        // ---- the result, or a part of it
        const bool whole = steps == n;
        const int64_t part = (2 * (int64_t)worker + !head) * G;
        if (lane == 0) {
            if (step0 == 0) p.spans[bh].x = whole ? -1 : 2 * worker + !head;
            if (step0 + steps == n) p.spans[bh].y = worker;
        }
        results<D, kTwice>(
            a, lane,
            [&](int h_q, int d, float4 o, float l) {
                if (h_q >= G) return;
                if (!whole) {
                    *reinterpret_cast<float4*>(p.part_o + (part + h_q) * D + d) = o;
                    return;
                }
                const float inv = hi > lo ? 1.f / l : 0.f;
                *reinterpret_cast<uint2*>(p.out + (bh * G + h_q) * D + d) =
                    make_uint2(float2_to_bf16x2(o.x * inv, o.y * inv), float2_to_bf16x2(o.z * inv, o.w * inv));
            },
            [&](int h_q, float ref, float l) {
                if (h_q >= G) return;
                if (!whole) p.part_ml[part + h_q] = make_float2(ref, l);
                else if (p.lse) p.lse[bh * G + h_q] = hi > lo ? ref * kLn2 + logf(l) : -INFINITY;
            });
        at += steps;
        if (h == p.n_kv - 1 && step0 + steps == n) first += (int64_t)n * p.n_kv, ++b;
    }
}

// Short sequences in one launch: a cluster of CTAs is one (sequence, KV head), its warps take the steps in turn, and the
// results meet in shared memory: the CTA's four warps', then the cluster's CTAs'.  Scores stay there too until the
// log-sum-exp is known, so that the weights need no launch of their own.  On the device, here and with workers and merge
// (and weights) launches, 8 KV heads, 32 queries:
//                          D = 64                         D = 128                        D = 256
//                          plain          weighed         plain          weighed         plain          weighed
//      1 x  1000 tokens    5.4 |  7.5      7.0 | 10.4     6.4 |  8.7      8.0 | 11.7     8.8 | 11.4     10.1 | 14.1
//      1 x  8000           9.0 | 14.9     13.7 | 18.0    11.4 | 17.1     16.0 | 20.1    16.9 | 26.3     21.3 | 29.4
//      1 x 16,000         12.9 | 16.0     21.3 | 19.5    16.5 | 19.1     25.0 | 22.3    25.4 | 24.3     33.8 | 28.0
//      4 x  8000          12.7 | 15.3     17.7 | 19.1    15.2 | 21.1     20.3 | 24.9    25.2 | 29.3     35.2 | 34.1
//     18 x  1000           8.1 | 13.8     11.2 | 16.9     9.2 | 15.5     12.5 | 18.8    one CTA an SM: workers
//     18 x  4000          19.2 | 25.3     workers        21.8 | 32.5     workers        workers
// So wherever all clusters are resident at once, up to 8 steps a warp, or 16 where no weights are asked for and D is below 256.
template <int D>
struct ClusterShape {
    using S = Shape<D>;
    static constexpr int kPitch = D + 4;  // of a query's sums
    static constexpr int kResults = kWarps * kMaxGroup * kPitch * 4;
    static size_t smem(int score_steps, int group) { return S::kSmem + kResults + (size_t)score_steps * kWarps * kStep * group * 4; }
};
constexpr size_t kHalfSm = 112 * 1024;              // shared memory with which two CTAs fit an SM
constexpr int kMostCluster = 8, kWeighedTurns = 8;  // CTAs of a cluster; steps of a warp whose scores are kept
constexpr int most_turns(int head_dim, bool weighed) { return weighed || head_dim == 256 ? kWeighedTurns : 16; }

// score_steps: steps of a warp at most, where weights are asked for.
template <int D, bool kTwice>
__global__ void __launch_bounds__(kThreads, 1) kv4_cluster_kernel(const DecodeParams p, int score_steps) {
    using S = Shape<D>;
    using C = ClusterShape<D>;
    constexpr int kStages = S::kStages;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 ml[kWarps][kMaxGroup], cta_ml[kMaxGroup];  // reference (-inf: no tokens) and sum of a query's weights
    __shared__ float lse2[kMaxGroup];
    float* sums = reinterpret_cast<float*>(smem + S::kSmem);  // [warp][query][kPitch]; the CTA's own in warp 0's place
    float* scores = reinterpret_cast<float*>(smem + S::kSmem + C::kResults);  // [query][local token]
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, G = p.group, ctas = gridDim.x, rank = blockIdx.x;
    const int64_t b = blockIdx.z, bh = b * p.n_kv + blockIdx.y, rows = bh * p.max_seq;
    const int len = visible(p, (int)b), steps = (len + kStep - 1) / kStep, every = ctas * kWarps, first = rank * kWarps + warp;
    uint8_t* ring = smem + warp * kStages * S::kStage;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    constexpr int kPiece = S::kScaleRow < 16 ? S::kScaleRow : 16;
    const LanePlanes planes{p.k_codes + lane * 16, p.v_codes + lane * 4, p.k_scales + lane * kPiece, p.v_scales + lane * kPiece};
    auto prefetch = [&](int s, int slot) {
        const int valid = len - s * kStep;
        const uint32_t to = ring_at + slot * S::kStage;
        if (valid >= kStep) fetch<D>(to, planes, rows + s * kStep, kStep, lane);
        else if (valid > 0) fetch<D>(to, planes, rows + s * kStep, valid, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i)
        if (first + (int64_t)i * every < steps) prefetch(first + i * every, i);
        else asm volatile("cp.async.commit_group;" ::: "memory");
    Queries<D> q;
    q.template load<kTwice>(p, bh, lane);
    Sums<D> a;
    a.start(lane);
    int slot = 0, turn = 0;
    const int local = score_steps * kWarps * kStep;  // tokens of a query's scores
    for (int s = first; s < steps; s += every, ++turn) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        int next = slot + kStages - 1;
        if (next >= kStages) next -= kStages;
        prefetch(s + (kStages - 1) * every, next);
        step<D, kTwice>(ring + slot * S::kStage, len - s * kStep, q, a, lane, score_steps ? scores + (turn * kWarps + warp) * kStep : nullptr, local, G);
        if (++slot == kStages) slot = 0;
    }
    const bool any = first < steps;
    results<D, kTwice>(
        a, lane,
        [&](int h, int d, float4 o, float) {
            if (h < G) *reinterpret_cast<float4*>(sums + (warp * kMaxGroup + h) * C::kPitch + d) = o;
        },
        [&](int h, float ref, float l) { ml[warp][h] = make_float2(any ? ref : -INFINITY, l); });
    __syncthreads();
    // ---- the CTA's: a thread keeps to its places, so that warp 0's can be overwritten
    for (int i = tid; i < G * (D / 4); i += kThreads) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w][h].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 x = ml[w][h];
            if (x.x == -INFINITY) continue;
            const float f = exp2f(x.x - m);
            const float4 y = *reinterpret_cast<const float4*>(sums + (w * kMaxGroup + h) * C::kPitch + d);
            o.x = fmaf(y.x, f, o.x), o.y = fmaf(y.y, f, o.y), o.z = fmaf(y.z, f, o.z), o.w = fmaf(y.w, f, o.w);
            l = fmaf(x.y, f, l);
        }
        *reinterpret_cast<float4*>(sums + h * C::kPitch + d) = o;
        if (d == 0) cta_ml[h] = make_float2(m, l);
    }
    cluster_barrier();
    // ---- the cluster's: each CTA a share of the places
    auto total_of = [&](int h, float& m, float& l) {
        m = -INFINITY, l = 0.f;
        for (int r = 0; r < ctas; ++r) m = fmaxf(m, load_remote(&cta_ml[h], r).x);
        for (int r = 0; r < ctas; ++r) {
            const float2 x = load_remote(&cta_ml[h], r);
            if (x.x != -INFINITY) l = fmaf(x.y, exp2f(x.x - m), l);
        }
    };
    for (int i = rank * kThreads + tid; i < G * (D / 4); i += ctas * kThreads) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float m, l;
        total_of(h, m, l);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < ctas; ++r) {
            const float2 x = load_remote(&cta_ml[h], r);
            const float4 y = load_remote(reinterpret_cast<const float4*>(sums + h * C::kPitch + d), r);
            const float f = x.x == -INFINITY ? 0.f : exp2f(x.x - m);
            o.x = fmaf(y.x, f, o.x), o.y = fmaf(y.y, f, o.y), o.z = fmaf(y.z, f, o.z), o.w = fmaf(y.w, f, o.w);
        }
        const float inv = len > 0 ? 1.f / l : 0.f;
        *reinterpret_cast<uint2*>(p.out + (bh * G + h) * D + d) =
            make_uint2(float2_to_bf16x2(o.x * inv, o.y * inv), float2_to_bf16x2(o.z * inv, o.w * inv));
        if (d == 0 && p.lse) p.lse[bh * G + h] = len > 0 ? m * kLn2 + logf(l) : -INFINITY;
    }
    if (score_steps) {
        if (tid < G) {
            float m, l;
            total_of(tid, m, l);
            lse2[tid] = m + log2f(l);
        }
        __syncthreads();
        for (int i = tid; i < local; i += kThreads) {
            const int64_t t = ((int64_t)first - warp + i / (kWarps * kStep) * every) * kStep + i % (kWarps * kStep);
            if (t >= len) break;  // the later ones are further on
            float w = 0.f;
            for (int h = 0; h < G; ++h) w += exp2f(scores[h * local + i] - lse2[h]);
            p.weights[rows + t] += w;
        }
    }
    cluster_barrier();  // nobody leaves while its shared memory is read
}

constexpr int kMergeWarps = 8, kMergeParts = 256;

// The parts of a row (sequence, query head) that several workers have.  kWide: a CTA a row, every eighth part a warp; else
// a warp a row.
template <int D, bool kWide>
__global__ void __launch_bounds__(32 * kMergeWarps) kv4_merge_kernel(const DecodeParams p) {
    constexpr int kPer = D / 32;  // dims of a lane: neighbours
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, G = p.group;
    const int row = kWide ? blockIdx.x : blockIdx.x * kMergeWarps + warp;
    if (row >= p.batch * p.n_kv * G) return;
    const int bh = row / G, h = row % G;
    const int2 span = p.spans[bh];
    if (span.x < 0) return;  // one worker had all of it
    const int i0 = span.x / 2, n = span.y - i0 + 1;
    auto part = [&](int r) { return (int64_t)(r == 0 ? span.x : 2 * (i0 + r)) * G + h; };
    float m = -INFINITY;
    for (int r = kWide ? threadIdx.x : lane; r < n; r += kWide ? 32 * kMergeWarps : 32) m = fmaxf(m, p.part_ml[part(r)].x);
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, off));
    float o[kPer] = {}, l = 0.f;
    // `count` rows from part r on, every `every`-th, times their factors: the loads of a batch are in flight at once
    constexpr int kBatch = 16 / (kPer / 2);
    auto add = [&](int r, int count, int every, auto&& factor_of) {
        for (int k0 = 0; k0 < count; k0 += kBatch) {
            float2 v[kBatch][kPer / 2];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const float* from = p.part_o + part(r + min(k0 + u, count - 1) * every) * D + lane * kPer;
#pragma unroll
                for (int k = 0; k < kPer / 2; ++k) v[u][k] = *reinterpret_cast<const float2*>(from + 2 * k);
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (k0 + u >= count) break;
                const float f = factor_of(r + (k0 + u) * every);
#pragma unroll
                for (int k = 0; k < kPer / 2; ++k) o[2 * k] = fmaf(v[u][k].x, f, o[2 * k]), o[2 * k + 1] = fmaf(v[u][k].y, f, o[2 * k + 1]);
            }
        }
    };
    if constexpr (kWide) {
        __shared__ float sums[kMergeWarps][D], totals[kMergeWarps], tops[kMergeWarps], factor[kMergeParts];
        if (lane == 0) tops[warp] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) m = fmaxf(m, tops[w]);
        for (int r0 = 0; r0 < n; r0 += kMergeParts) {  // the factors first, so that the rows' loads wait for nothing
            const int count = min(kMergeParts, n - r0);
            if (r0) __syncthreads();
            if (threadIdx.x < count) {
                const float2 x = p.part_ml[part(r0 + threadIdx.x)];
                const float f = exp2f(x.x - m);
                factor[threadIdx.x] = f;
                l += x.y * f;
            }
            __syncthreads();
            if (warp < count)
                add(r0 + warp, (count - warp + kMergeWarps - 1) / kMergeWarps, kMergeWarps, [&](int r) { return factor[r - r0]; });
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) l += __shfl_xor_sync(kFullMask, l, off);
#pragma unroll
        for (int k = 0; k < kPer; k += 2) *reinterpret_cast<float2*>(&sums[warp][kPer * lane + k]) = make_float2(o[k], o[k + 1]);
        if (lane == 0) totals[warp] = l;
        __syncthreads();
        l = 0.f;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) l += totals[w];
        if (threadIdx.x < D) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kMergeWarps; ++w) v += sums[w][threadIdx.x];
            p.out[(int64_t)row * D + threadIdx.x] = __float2bfloat16(v / l);
        }
    } else {
        for (int r0 = 0; r0 < n; r0 += 32) {  // a factor a lane
            const int count = min(32, n - r0);
            float f = 0.f;
            if (lane < count) {
                const float2 x = p.part_ml[part(r0 + lane)];
                f = exp2f(x.x - m);
                l = fmaf(x.y, f, l);
            }
            add(r0, count, 1, [&](int r) { return __shfl_sync(kFullMask, f, r - r0); });
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) l += __shfl_xor_sync(kFullMask, l, off);
#pragma unroll
        for (int k = 0; k < kPer; k += 2)
            *reinterpret_cast<uint32_t*>(p.out + (int64_t)row * D + kPer * lane + k) = float2_to_bf16x2(o[k] / l, o[k + 1] / l);
    }
    if ((kWide ? threadIdx.x : lane) == 0 && p.lse) p.lse[row] = m * kLn2 + logf(l);
}

// weights[t] += sum over the group of 2^(score - lse): a thread four neighbouring tokens, and further ones of a CTA's places.
// The weighed call on 64 sequences of 1000 tokens, 8 KV heads, D = 128: 38 us in a cache of 1024 rows, 36 in one of 131,072, where
// a CTA for every 512 rows of cache took 165.
__global__ void __launch_bounds__(kThreads) kv4_weights_kernel(const DecodeParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t b = blockIdx.z, bh = b * p.n_kv + blockIdx.y;
    const int len = visible(p, (int)b), fours = (len + 3) / 4;
    const bool four = p.max_seq % 4 == 0 && (reinterpret_cast<uintptr_t>(p.weights) & 15) == 0;  // rows begin at 16 bytes
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < fours; i += gridDim.x * kThreads) {
        const int t = 4 * i;
        const float* x = p.scores + bh * p.group * p.max_seq + t;
        float* to = p.weights + bh * p.max_seq + t;
        float w[4] = {};
#pragma unroll
        for (int h = 0; h < kMaxGroup; ++h) {
            if (h >= p.group) continue;
            const float l = p.lse[bh * p.group + h] * kLog2e;
            float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (four) {  // tokens behind the length hold anything: they are not written
                v = *reinterpret_cast<const float4*>(x + h * p.max_seq);
            } else {
                v.x = x[h * p.max_seq];
                if (t + 1 < len) v.y = x[h * p.max_seq + 1];
                if (t + 2 < len) v.z = x[h * p.max_seq + 2];
                if (t + 3 < len) v.w = x[h * p.max_seq + 3];
            }
            w[0] += exp2f(v.x - l), w[1] += exp2f(v.y - l), w[2] += exp2f(v.z - l), w[3] += exp2f(v.w - l);
        }
        if (four && t + 3 < len) {
            float4 v = *reinterpret_cast<float4*>(to);
            v.x += w[0], v.y += w[1], v.z += w[2], v.w += w[3];
            *reinterpret_cast<float4*>(to) = v;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (t + k < len) to[k] += w[k];
        }
    }
}

// f(head dim, whether a KV head's queries fit an operand twice)
template <class F>
cudaError_t for_form(int head_dim, int group, F&& f) {
    return for_head_dim(head_dim, [&](auto d) { return group <= 4 ? f(d, std::true_type{}) : f(d, std::false_type{}); });
}

// Clusters of `size` CTAs with that much shared memory that the device has resident at a time, asked for once.
template <int D, bool kTwice>
cudaError_t cluster_slots(int size, size_t smem, int& slots) {
    static std::atomic<int> known[64][4][2];  // [device][log2 size][shared memory: up to half of an SM's, or more]
    int dev = 0;
    const cudaError_t at = cudaGetDevice(&dev);
    if (at != cudaSuccess) return at;
    const int log2 = size == 8 ? 3 : size == 4 ? 2 : 1, large = smem > kHalfSm;
    std::atomic<int>* entry = dev < 64 ? &known[dev][log2][large] : nullptr;
    if (entry && (slots = entry->load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size, 1024);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = large ? ClusterShape<D>::smem(kWeighedTurns, kMaxGroup) : kHalfSm;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&slots, kv4_cluster_kernel<D, kTwice>, &cfg);
    if (e == cudaSuccess && entry) entry->store(std::max(slots, 1), std::memory_order_relaxed);
    return e;
}

// The largest cluster that all groups can have at once and whose warps have a step each at least; 0: none, or too many steps.
template <int D, bool kTwice>
cudaError_t pick_cluster(int64_t groups, int64_t steps, bool weighed, int group, int& cluster, int& turns, size_t& smem) {
    const cudaError_t at = set_max_dynamic_smem_once<kv4_cluster_kernel<D, kTwice>>((int)std::max(ClusterShape<D>::smem(kWeighedTurns, kMaxGroup), kHalfSm));
    if (at != cudaSuccess) return at;
    for (cluster = kMostCluster; cluster > 1; cluster /= 2) {
        turns = (int)((steps + cluster * kWarps - 1) / (cluster * kWarps));
        if (turns > most_turns(D, weighed)) break;  // smaller clusters have more
        if (steps < cluster * kWarps) continue;
        smem = ClusterShape<D>::smem(weighed ? turns : 0, group);
        int slots = 0;
        const cudaError_t e = cluster_slots<D, kTwice>(cluster, smem, slots);
        if (e != cudaSuccess) return e;
        if (groups <= slots) return cudaSuccess;
    }
    cluster = 0;
    return cudaSuccess;
}

// Workers of a launch: as many warps as fit at a time, or one for every step.
int workers_of(int64_t batch, int n_kv, int head_dim, int64_t max_seq) {
    const int per_sm = kWarps * (head_dim == 64 ? Shape<64>::kPerSm : head_dim == 128 ? Shape<128>::kPerSm : Shape<256>::kPerSm);
    const int64_t steps = batch * n_kv * ((max_seq + kStep - 1) / kStep);
    return (int)std::min(steps, (int64_t)per_sm * sm_count());
}

inline size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t kv4_decode_workspace_bytes(int64_t batch, int n_heads, int n_kv, int head_dim, int64_t max_seq, bool weighed) {
    const size_t rows = 2 * (size_t)workers_of(batch, n_kv, head_dim, max_seq) * (n_heads / n_kv + (n_heads % n_kv != 0));
    return round16(rows * head_dim * sizeof(float)) + round16(rows * sizeof(float2)) + round16((size_t)batch * n_kv * sizeof(int2)) +
           (weighed ? round16((size_t)batch * n_heads * sizeof(float)) + round16((size_t)batch * n_heads * max_seq * sizeof(float)) : 0);
}

cudaError_t launch_kv4_decode(const Kv4Cache& c, const void* q, void* out, float* lse, float* weights, int64_t batch,
                              int n_heads, int n_kv, int head_dim, int64_t max_seq, const int32_t* kv_lens,
                              int64_t kv_len_uniform, float scale, void* workspace, cudaStream_t stream) {
    DecodeParams p = {};
    p.q = (const __nv_bfloat16*)q;
    p.k_codes = (const uint8_t*)c.k_codes, p.v_codes = (const uint8_t*)c.v_codes;
    p.k_scales = (const uint8_t*)c.k_scales, p.v_scales = (const uint8_t*)c.v_scales;
    p.out = (__nv_bfloat16*)out, p.weights = weights;
    p.max_seq = max_seq, p.kv_lens = kv_lens, p.kv_len = (int)kv_len_uniform, p.batch = (int)batch;
    p.n_kv = n_kv, p.group = n_heads / n_kv, p.workers = workers_of(batch, n_kv, head_dim, max_seq);
    p.scale_log2 = scale * kLog2e;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const size_t rows = 2 * (size_t)p.workers * p.group;
    p.part_o = (float*)ws, ws += round16(rows * head_dim * sizeof(float));
    p.part_ml = (float2*)ws, ws += round16(rows * sizeof(float2));
    p.spans = (int2*)ws, ws += round16((size_t)batch * n_kv * sizeof(int2));
    if (weights) {
        if (!lse) lse = (float*)ws;
        ws += round16((size_t)batch * n_heads * sizeof(float));
        p.scores = (float*)ws;
    }
    p.lse = lse;
    // One launch where all clusters are resident at once and a warp has few steps.
    const int64_t groups = batch * n_kv, longest = kv_lens ? max_seq : kv_len_uniform, steps = (longest + kStep - 1) / kStep;
    if (steps <= (int64_t)kMostCluster * kWarps * most_turns(head_dim, weights != nullptr) && groups <= sm_count()) {
        int cluster = 0, turns = 0;
        size_t smem = 0;
        const cudaError_t e = for_form(head_dim, p.group, [&](auto d, auto t) {
            return pick_cluster<decltype(d)::value, decltype(t)::value>(groups, steps, weights != nullptr, p.group, cluster, turns, smem);
        });
        if (e != cudaSuccess) return e;
        if (cluster) return for_form(head_dim, p.group, [&](auto d, auto t) {
            constexpr int D = decltype(d)::value;
            constexpr bool kTwice = decltype(t)::value;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(cluster, n_kv, (unsigned)batch);
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = smem;
            cfg.stream = stream;
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
            attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[1].val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 2;
            return cudaLaunchKernelEx(&cfg, kv4_cluster_kernel<D, kTwice>, p, weights ? turns : 0);
        });
    }
    return for_form(head_dim, p.group, [&](auto d, auto t) {
        constexpr int D = decltype(d)::value;
        constexpr bool kTwice = decltype(t)::value;
        cudaError_t e = set_max_dynamic_smem_once<kv4_decode_kernel<D, kTwice>>(Shape<D>::kSmem);
        if (e != cudaSuccess) return e;
        e = launch_chained(kv4_decode_kernel<D, kTwice>, dim3((p.workers + kWarps - 1) / kWarps), kThreads, Shape<D>::kSmem, stream, p);
        if (e == cudaSuccess && p.workers > 1) {
            // A row has about workers * group / rows parts: a CTA a row from 8 on.  The whole call with a CTA a row and a warp a row,
            // D = 128: 32 rows of 20,000 tokens (222 parts) 19.9 and 69.0 us, 128 of 20,000 (56) 31.2 and 43.9, 512 of 4000 (14)
            // 30.6 and 32.4, 1024 of 4000 (7) 43.1 and 43.1.
            const int64_t n = batch * n_heads;
            e = p.workers * (int64_t)p.group >= 8 * n
                    ? launch_chained(kv4_merge_kernel<D, true>, dim3((unsigned)n), 32 * kMergeWarps, 0, stream, p)
                    : launch_chained(kv4_merge_kernel<D, false>, dim3((unsigned)((n + kMergeWarps - 1) / kMergeWarps)), 32 * kMergeWarps, 0,
                                     stream, p);
        }
        if (e == cudaSuccess && weights)
            e = launch_chained(kv4_weights_kernel,
                               dim3((unsigned)bounded_blocks((longest + 4 * kThreads - 1) / (4 * kThreads), groups, 32), n_kv, (unsigned)batch),
                               kThreads, 0, stream, p);
        return e;
    });
}

}  // namespace rt

// Rows into and out of a 4-bit KV cache: quantising append (with and without the rotary embedding) and read-back in bf16.
//
// One thread handles an octet (8 bf16 values, 16 bytes; one word of 8 codes), D/8 neighbouring threads a row.  A group's
// four octets lie kSpanGroups threads apart, so its minimum and maximum are two shuffles each.
#include "cache_kernels.h"
#include "kv4.cuh"

namespace rt {
namespace {

__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = bf16x2_to_float2(u[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}

// Codes of the calling thread's octet, and the {scale, lo} word of its group.  All threads of the warp call it.
template <int D>
__device__ __forceinline__ uint32_t quantise_octet(uint4 raw, uint32_t& scale_word) {
    using R = Kv4Row<D>;
    const int lane = threadIdx.x & 31;
    float x[8];
    unpack8(raw, x);
    bool nan = false;
    float lo = 65504.f, hi = -65504.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        nan |= x[i] != x[i];
        x[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
        lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int off = R::kSpanGroups; off <= 2 * R::kSpanGroups; off *= 2) {
        lo = fminf(lo, __shfl_xor_sync(kFullMask, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(kFullMask, hi, off));
    }
    constexpr unsigned kMembers = 1u | 1u << R::kSpanGroups | 1u << 2 * R::kSpanGroups | 1u << 3 * R::kSpanGroups;
    const int first = (lane & ~(R::kSpanOctets - 1)) | (lane & (R::kSpanGroups - 1));
    const bool group_nan = (__ballot_sync(kFullMask, nan) >> first) & kMembers;
    const __half lo16 = __float2half_rn(lo);
    const float lo32 = __half2float(lo16);
    const __half s16 = __float2half_rn(__fdiv_rn(fmaxf(hi - lo32, 0.f), 15.f));
    const float s = __half2float(s16);
    uint32_t codes = 0;
    if (s > 0.f && !group_nan) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i] - lo32, s)), 0.f), 15.f);
            codes |= (uint32_t)c << (4 * i);
        }
    }
    const uint32_t low = group_nan ? 0u : (uint32_t)__half_as_ushort(s16);
    const uint32_t high = group_nan ? 0x7fffu : (uint32_t)__half_as_ushort(lo16);
    scale_word = low | high << 16;
    return codes;
}

struct Kv4Planes {
    uint32_t *k_codes, *k_scales, *v_codes, *v_scales;
};

// Writes a row's octet `o` (and, once per group, the group's word).
template <int D>
__device__ __forceinline__ void store_octet(uint32_t* codes, uint32_t* scales, int64_t row, int o, uint32_t c, uint32_t s) {
    using R = Kv4Row<D>;
    codes[row * R::kOctets + o] = c;
    if (o % R::kSpanOctets < R::kSpanGroups) scales[row * R::kGroups + R::group_of_octet(o)] = s;
}

struct AppendParams {
    Kv4Planes cache;
    const __nv_bfloat16 *k, *v;
    int64_t ks[3], vs[3];  // batch, head, row
    int64_t items, rows, max_seq, pos;
    int n_kv;
    const int32_t *positions, *lens;
};

template <int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendParams p) {
    using R = Kv4Row<D>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int o = threadIdx.x % R::kOctets;
    const int64_t item = (int64_t)blockIdx.x * (256 / R::kOctets) + threadIdx.x / R::kOctets;
    // neighbouring rows are the heads of a token: together in the projections' layout
    const int64_t it = min(item, p.items - 1);
    const int h = (int)(it % p.n_kv);
    const int64_t bt = it / p.n_kv, t = bt % p.rows, b = bt / p.rows;
    const int64_t at = (p.positions ? (int64_t)p.positions[b] : p.pos) + t;
    const bool write = item < p.items && at >= 0 && at < p.max_seq && (!p.lens || t < p.lens[b]);
    const uint4 k = *reinterpret_cast<const uint4*>(p.k + b * p.ks[0] + h * p.ks[1] + t * p.ks[2] + 8 * o);
    const uint4 v = *reinterpret_cast<const uint4*>(p.v + b * p.vs[0] + h * p.vs[1] + t * p.vs[2] + 8 * o);
    uint32_t k_scale, v_scale;
    const uint32_t kc = quantise_octet<D>(k, k_scale), vc = quantise_octet<D>(v, v_scale);
    if (write) {
        const int64_t row = (b * p.n_kv + h) * p.max_seq + at;
        store_octet<D>(p.cache.k_codes, p.cache.k_scales, row, o, kc, k_scale);
        store_octet<D>(p.cache.v_codes, p.cache.v_scales, row, o, vc, v_scale);
    }
}

struct RopeParams {
    Kv4Planes cache;
    __nv_bfloat16* q;
    const __nv_bfloat16 *k, *v;
    const float* inv_freq;
    int64_t rows, max_seq, pos, slot;
    int n_heads, n_kv, style;
    const int32_t *positions, *slots;
};

// Row r of a sequence: its Hq query heads, then the Hkv keys, then the Hkv values.
template <int D>
__global__ void __launch_bounds__(128) kv4_rope_append_kernel(const RopeParams p) {
    using R = Kv4Row<D>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int o = threadIdx.x % R::kOctets;
    const int64_t item = (int64_t)blockIdx.x * (128 / R::kOctets) + threadIdx.x / R::kOctets;
    const int64_t it = min(item, p.rows - 1);
    const int per = p.n_heads + 2 * p.n_kv;
    const int64_t b = it / per;
    const int r = (int)(it % per);
    const int64_t pos = p.positions ? (int64_t)p.positions[b] : p.pos;
    const int64_t slot = p.slots ? (int64_t)p.slots[b] : (p.slot >= 0 ? p.slot : pos);
    const bool valid = item < p.rows && pos >= 0 && slot >= 0 && slot < p.max_seq;
    const bool is_q = r < p.n_heads, is_k = !is_q && r < p.n_heads + p.n_kv;
    const int h = is_q ? r : (is_k ? r - p.n_heads : r - p.n_heads - p.n_kv);
    const __nv_bfloat16* src = is_q ? p.q + (b * p.n_heads + h) * D : (is_k ? p.k : p.v) + (b * p.n_kv + h) * D;
    uint4 raw = *reinterpret_cast<const uint4*>(src + 8 * o);
    if (__any_sync(kFullMask, is_q || is_k)) {
        // the other half's octet, for pairs (i, i + D/2)
        const uint4 other = make_uint4(__shfl_xor_sync(kFullMask, raw.x, R::kOctets / 2), __shfl_xor_sync(kFullMask, raw.y, R::kOctets / 2),
                                       __shfl_xor_sync(kFullMask, raw.z, R::kOctets / 2), __shfl_xor_sync(kFullMask, raw.w, R::kOctets / 2));
        if (is_q || is_k) {
            float x[8], y[8], z[8];
            unpack8(raw, x);
            unpack8(other, y);
            const float at = (float)pos;
            if (p.style == 0) {
                const bool upper = o >= R::kOctets / 2;
                const int base = 8 * (upper ? o - R::kOctets / 2 : o);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float s, c;
                    sincosf(at * p.inv_freq[base + i], &s, &c);
                    z[i] = upper ? x[i] * c + y[i] * s : x[i] * c - y[i] * s;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float s, c;
                    sincosf(at * p.inv_freq[4 * o + i / 2], &s, &c);
                    z[i] = x[i] * c - x[i + 1] * s;
                    z[i + 1] = x[i + 1] * c + x[i] * s;
                }
            }
            raw = make_uint4(float2_to_bf16x2(z[0], z[1]), float2_to_bf16x2(z[2], z[3]), float2_to_bf16x2(z[4], z[5]),
                             float2_to_bf16x2(z[6], z[7]));
        }
    }
    uint32_t scale;
    const uint32_t codes = quantise_octet<D>(raw, scale);
    if (!valid) return;
    if (is_q) {
        *reinterpret_cast<uint4*>(p.q + (b * p.n_heads + h) * D + 8 * o) = raw;
        return;
    }
    const int64_t row = (b * p.n_kv + h) * p.max_seq + slot;
    store_octet<D>(is_k ? p.cache.k_codes : p.cache.v_codes, is_k ? p.cache.k_scales : p.cache.v_scales, row, o, codes, scale);
}

struct ReadParams {
    const uint32_t *k_codes, *k_scales, *v_codes, *v_scales;
    __nv_bfloat16 *k, *v;
    int64_t items, rows, max_seq, start;
    int n_kv;
    const int32_t *starts, *kv_lens;
};

template <int D>
__device__ __forceinline__ uint4 octet_values(uint32_t codes, uint32_t scale_word) {
    const float2 s = kv4_scale(scale_word);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = float2_to_bf16x2(kv4_value(s, codes >> (8 * i) & 15u), kv4_value(s, codes >> (8 * i + 4) & 15u));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadParams p) {
    using R = Kv4Row<D>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int o = threadIdx.x % R::kOctets;
    const int64_t item = (int64_t)blockIdx.x * (256 / R::kOctets) + threadIdx.x / R::kOctets;
    if (item >= p.items) return;
    const int64_t i = item % p.rows, bh = item / p.rows, b = bh / p.n_kv;
    const int64_t at = (p.starts ? (int64_t)p.starts[b] : p.start) + i;
    const int64_t len = p.kv_lens ? min((int64_t)p.kv_lens[b], p.max_seq) : p.max_seq;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (at >= 0 && at < len) {
        const int64_t row = bh * p.max_seq + at;
        const int g = R::group_of_octet(o);
        k = octet_values<D>(p.k_codes[row * R::kOctets + o], p.k_scales[row * R::kGroups + g]);
        v = octet_values<D>(p.v_codes[row * R::kOctets + o], p.v_scales[row * R::kGroups + g]);
    }
    *reinterpret_cast<uint4*>(p.k + item * D + 8 * o) = k;
    *reinterpret_cast<uint4*>(p.v + item * D + 8 * o) = v;
}

inline unsigned blocks(int64_t items, int per) { return (unsigned)((items + per - 1) / per); }

}  // namespace

cudaError_t launch_kv4_append(const Kv4Cache& c, const void* k, const void* v, const int64_t* ks, const int64_t* vs,
                              int64_t batch, int n_kv, int64_t rows, int head_dim, int64_t max_seq, int64_t pos,
                              const int32_t* positions, const int32_t* lens, cudaStream_t stream) {
    AppendParams p;
    p.cache = Kv4Planes{(uint32_t*)c.k_codes, (uint32_t*)c.k_scales, (uint32_t*)c.v_codes, (uint32_t*)c.v_scales};
    p.k = (const __nv_bfloat16*)k, p.v = (const __nv_bfloat16*)v;
    for (int i = 0; i < 3; ++i) p.ks[i] = ks[i], p.vs[i] = vs[i];
    p.items = batch * rows * n_kv;
    p.rows = rows, p.max_seq = max_seq, p.pos = pos, p.n_kv = n_kv, p.positions = positions, p.lens = lens;
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_chained(kv4_append_kernel<D>, dim3(blocks(p.items, 256 * 8 / D)), 256, 0, stream, p);
    });
}

cudaError_t launch_rope_kv4_append(const Kv4Cache& c, void* q, const void* k, const void* v, const float* inv_freq,
                                   int64_t batch, int n_heads, int n_kv, int head_dim, int64_t max_seq, int64_t pos,
                                   const int32_t* positions, int64_t slot, const int32_t* slots, int style,
                                   cudaStream_t stream) {
    RopeParams p;
    p.cache = Kv4Planes{(uint32_t*)c.k_codes, (uint32_t*)c.k_scales, (uint32_t*)c.v_codes, (uint32_t*)c.v_scales};
    p.q = (__nv_bfloat16*)q, p.k = (const __nv_bfloat16*)k, p.v = (const __nv_bfloat16*)v;
    p.inv_freq = inv_freq;
    p.rows = batch * ((int64_t)n_heads + 2 * n_kv);
    p.max_seq = max_seq, p.pos = pos, p.slot = slot, p.n_heads = n_heads, p.n_kv = n_kv, p.style = style;
    p.positions = positions, p.slots = slots;
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_chained(kv4_rope_append_kernel<D>, dim3(blocks(p.rows, 128 * 8 / D)), 128, 0, stream, p);
    });
}

cudaError_t launch_kv4_read(const Kv4Cache& c, void* k, void* v, int64_t batch, int n_kv, int head_dim, int64_t max_seq,
                            int64_t rows, int64_t start, const int32_t* starts, const int32_t* kv_lens, cudaStream_t stream) {
    ReadParams p;
    p.k_codes = (const uint32_t*)c.k_codes, p.k_scales = (const uint32_t*)c.k_scales;
    p.v_codes = (const uint32_t*)c.v_codes, p.v_scales = (const uint32_t*)c.v_scales;
    p.k = (__nv_bfloat16*)k, p.v = (__nv_bfloat16*)v;
    p.items = batch * n_kv * rows;
    p.rows = rows, p.max_seq = max_seq, p.start = start, p.n_kv = n_kv, p.starts = starts, p.kv_lens = kv_lens;
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_chained(kv4_read_kernel<D>, dim3(blocks(p.items, 256 * 8 / D)), 256, 0, stream, p);
    });
}

}  // namespace rt

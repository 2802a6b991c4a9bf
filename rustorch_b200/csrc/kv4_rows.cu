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

__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {  // of two bf16 at a time; NaN stays
    uint32_t c;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    return c;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t c;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    return c;
}

// Two f32 at a time.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 split(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t c;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c) : "l"(a), "l"(b));
    return c;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// Codes of the calling thread's octet, and the {scale, lo} word of its group.  All threads of the warp call it.
//
// A code is the IEEE quotient (x - lo) / scale rounded to a whole number.  It is first taken from a product with 1 / scale,
// which is within 2^-18 of it; only an octet in which that leaves a value in doubt (within 2^-15 of the middle between two
// codes, or outside 0 to 15) takes the quotient itself and clamps it.  10,194 tokens of 8 heads, D = 128, with their
// read-back: 80.6 us with all values divided, 37.3 with a reciprocal and each value clamped (29 instructions a value at 0.74
// of the issue rate), 31 with pairs of values and the rare cases apart (18 a value; 20.8 us of it here, 2.6 TB/s).
template <int D>
__device__ __forceinline__ uint32_t quantise_octet(uint4 raw, uint32_t& scale_word) {
    using R = Kv4Row<D>;
    // {min, -max} of the octet, then of the group, as a pair of bf16
    const uint32_t lo2 = min2(min2(raw.x, raw.y), min2(raw.z, raw.w)), hi2 = max2(max2(raw.x, raw.y), max2(raw.z, raw.w)) ^ 0x80008000u;
    uint32_t ends = min2(__byte_perm(lo2, hi2, 0x5410), __byte_perm(lo2, hi2, 0x7632));
    ends = min2(ends, __shfl_xor_sync(kFullMask, ends, R::kSpanGroups));
    ends = min2(ends, __shfl_xor_sync(kFullMask, ends, 2 * R::kSpanGroups));
    const float2 e = bf16x2_to_float2(ends);
    const bool nan = e.x != e.x;
    const float lo = fminf(fmaxf(e.x, -65504.f), 65504.f), hi = fminf(fmaxf(-e.y, -65504.f), 65504.f);
    const __half lo16 = __float2half_rn(lo);
    const float lo32 = __half2float(lo16);
    // range / 15, correctly rounded: a product with the rounded reciprocal and one correction by its remainder (Markstein)
    const float range = fmaxf(hi - lo32, 0.f), fifteenth = 1.f / 15.f, about = range * fifteenth;
    const __half s16 = __float2half_rn(fmaf(fmaf(-15.f, about, range), fifteenth, about));
    const float s = __half2float(s16);
    const bool plain = s > 0.f && !nan;  // else all codes are 0
    scale_word = nan ? 0x7fff0000u : (uint32_t)__half_as_ushort(s16) | (uint32_t)__half_as_ushort(lo16) << 16;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    // value i beside value i + 4
    float x[8];
    unpack8(raw, x);
    constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: a sum with it is rounded to a whole number, to the even one of two
    const uint64_t less = pair(-lo32, -lo32), by = pair(inv, inv), whole = pair(kWhole, kWhole), back = pair(-kWhole, -kWhole);
    uint64_t c[4];
    // the group's own ends say whether a value can be outside: lo rounded up, a subnormal scale, values past 65504
    float off = (e.x - lo32) * inv < -0.49f || (-e.y - lo32) * inv > 15.49f ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t d = add2(pair(x[i], x[i + 4]), less);
        c[i] = add2(fma2(d, by, whole), back);
        const float2 k = split(c[i]), r = split(fma2(d, by, pair(-k.x, -k.y)));
        off = max3(off, fabsf(r.x), fabsf(r.y));
    }
    if (plain && off > 0.49996f) {
        // The quotients, by the same correction.  This is not rare: values and scales have few bits, so that 0.07 % of N(0, 1)
        // values lie exactly between two codes, an octet in a sixth of the warps.
        const float exact_inv = __frcp_rn(s);
        const uint64_t y = pair(exact_inv, exact_inv), minus_s = pair(-s, -s), zero = pair(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t d = add2(pair(fminf(fmaxf(x[i], -65504.f), 65504.f), fminf(fmaxf(x[i + 4], -65504.f), 65504.f)), less);
            const uint64_t q0 = fma2(d, y, zero);
            const float2 q = split(fma2(fma2(q0, minus_s, d), y, q0));
            c[i] = add2(add2(pair(fminf(fmaxf(q.x, 0.f), 15.f), fminf(fmaxf(q.y, 0.f), 15.f)), whole), back);
        }
    }
    // four codes are a whole number below 2^16, exact in f32; the sum with 2^23 has it in its low bits
    const float2 sums = split(fma2(c[3], pair(4096.f, 4096.f), fma2(c[2], pair(256.f, 256.f),
                                                                    fma2(c[1], pair(16.f, 16.f), add2(c[0], pair(8388608.f, 8388608.f))))));
    return plain ? __byte_perm(__float_as_uint(sums.x), __float_as_uint(sums.y), 0x5410) : 0u;
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
    int64_t max_seq, pos;
    int rows, n_kv;
    const int32_t *positions, *lens;
};

constexpr int kRowThreads = 256;

// Grid: (blocks of rows, KV head, sequence).  A thread has kRows rows, a block's apart, all their loads in flight at once.
template <int D, int kRows>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(const AppendParams p) {
    using R = Kv4Row<D>;
    constexpr int kApart = kRowThreads / R::kOctets;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int o = threadIdx.x % R::kOctets, h = blockIdx.y, b = blockIdx.z;
    const int t0 = blockIdx.x * (kApart * kRows) + threadIdx.x / R::kOctets;
    const int rows = p.lens ? min(p.rows, p.lens[b]) : p.rows;
    const int64_t at = (p.positions ? (int64_t)p.positions[b] : p.pos) + t0;
    const __nv_bfloat16 *k_from = p.k + b * p.ks[0] + h * p.ks[1] + t0 * p.ks[2] + 8 * o,
                        *v_from = p.v + b * p.vs[0] + h * p.vs[1] + t0 * p.vs[2] + 8 * o;
    uint4 k[kRows], v[kRows];
    bool write[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int t = t0 + i * kApart;
        write[i] = t < rows && at + i * kApart >= 0 && at + i * kApart < p.max_seq;
        k[i] = v[i] = make_uint4(0, 0, 0, 0);
        if (write[i]) {
            k[i] = ld_stream_16B(k_from + i * kApart * p.ks[2]);
            v[i] = ld_stream_16B(v_from + i * kApart * p.vs[2]);
        }
    }
    const int64_t row = ((int64_t)b * p.n_kv + h) * p.max_seq + at;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (!__any_sync(kFullMask, write[i])) continue;
        uint32_t k_scale, v_scale;
        const uint32_t kc = quantise_octet<D>(k[i], k_scale), vc = quantise_octet<D>(v[i], v_scale);
        if (write[i]) {
            store_octet<D>(p.cache.k_codes, p.cache.k_scales, row + i * kApart, o, kc, k_scale);
            store_octet<D>(p.cache.v_codes, p.cache.v_scales, row + i * kApart, o, vc, v_scale);
        }
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
    int64_t max_seq, start;
    int rows, n_kv;
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
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(const ReadParams p) {
    using R = Kv4Row<D>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int o = threadIdx.x % R::kOctets, b = blockIdx.z;
    const int i = blockIdx.x * (kRowThreads / R::kOctets) + threadIdx.x / R::kOctets;
    if (i >= p.rows) return;
    const int64_t bh = (int64_t)b * p.n_kv + blockIdx.y;
    const int64_t at = (p.starts ? (int64_t)p.starts[b] : p.start) + i;
    const int64_t len = p.kv_lens ? min((int64_t)p.kv_lens[b], p.max_seq) : p.max_seq;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (at >= 0 && at < len) {
        const int64_t row = bh * p.max_seq + at;
        const int g = R::group_of_octet(o);
        const uint32_t kc = p.k_codes[row * R::kOctets + o], ks = p.k_scales[row * R::kGroups + g],
                       vc = p.v_codes[row * R::kOctets + o], vs = p.v_scales[row * R::kGroups + g];
        k = octet_values<D>(kc, ks);
        v = octet_values<D>(vc, vs);
    }
    const int64_t to = (bh * p.rows + i) * D + 8 * o;
    *reinterpret_cast<uint4*>(p.k + to) = k;
    *reinterpret_cast<uint4*>(p.v + to) = v;
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
    p.rows = (int)rows, p.max_seq = max_seq, p.pos = pos, p.n_kv = n_kv, p.positions = positions, p.lens = lens;
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        constexpr int kApart = kRowThreads * 8 / D;
        if (rows <= kApart)  // a block of rows: the short form
            return launch_chained(kv4_append_kernel<D, 1>, dim3(1, n_kv, (unsigned)batch), kRowThreads, 0, stream, p);
        // two: 20.8 us for 10,194 tokens of 8 heads, as four, 22.5 with one; the next step's loads begin sooner
        return launch_chained(kv4_append_kernel<D, 2>, dim3(blocks(rows, 2 * kApart), n_kv, (unsigned)batch), kRowThreads, 0, stream, p);
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
    p.rows = (int)rows, p.max_seq = max_seq, p.start = start, p.n_kv = n_kv, p.starts = starts, p.kv_lens = kv_lens;
    return for_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_chained(kv4_read_kernel<D>, dim3(blocks(rows, kRowThreads * 8 / D), n_kv, (unsigned)batch), kRowThreads, 0,
                              stream, p);
    });
}

}  // namespace rt

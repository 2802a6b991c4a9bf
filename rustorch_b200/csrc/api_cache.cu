// extern "C" boundary of the 4-bit KV cache and of eviction: argument validation and dispatch.
#include <cmath>

#include "../../include/rustorch_attn.h"
#include "cache_kernels.h"

namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline float default_scale(float scale, int dim) { return scale > 0.f ? scale : 1.0f / std::sqrt((float)dim); }
inline bool head_dim_ok(int d) { return d == 64 || d == 128 || d == 256; }

// Lengths and counts are 32-bit in the kernels, places in a tensor 64-bit.
constexpr int64_t kMostSeq = 0x7fff0000;

// The planes of a 4-bit cache: there and aligned.
inline int check_planes(const rt::Kv4Cache& c) {
    for (const void* p : {c.k_codes, c.k_scales, c.v_codes, c.v_scales})
        if (!p) return RT_ERR_NULL_POINTER;
    for (const void* p : {c.k_codes, c.k_scales, c.v_codes, c.v_scales})
        if (!aligned16(p)) return RT_ERR_ALIGNMENT;
    return RT_OK;
}

// Shape checks that the entries share.
inline int check_shape(int64_t batch, int64_t n_kv, int head_dim, int64_t max_seq) {
    if (head_dim == 0) return RT_ERR_ZERO_DIM;
    if (batch < 0 || n_kv < 0 || head_dim < 0 || max_seq < 0) return RT_ERR_BAD_LENGTH;
    if (!head_dim_ok(head_dim) || batch > 65535 || n_kv > 65535 || max_seq > kMostSeq) return RT_ERR_UNSUPPORTED;
    return RT_OK;
}

struct Bytes {
    const void* at;
    size_t n;
};
inline bool overlap(const Bytes& a, const Bytes& b) {
    const auto x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return x < y + b.n && y < x + a.n;
}

}  // namespace

extern "C" {

int rt_kv4_append(void* k_codes, void* k_scales, void* v_codes, void* v_scales, const void* k, const void* v,
                  const int64_t* k_strides, const int64_t* v_strides, int64_t batch, int n_kv, int64_t rows,
                  int head_dim, int64_t max_seq, int64_t pos, const int32_t* positions, const int32_t* lens,
                  void* stream) {
    if (const int rc = check_shape(batch, n_kv, head_dim, max_seq)) return rc;
    if (rows < 0) return RT_ERR_BAD_LENGTH;
    if (!positions && (pos < 0 || pos > max_seq || rows > max_seq - pos)) return RT_ERR_BAD_LENGTH;
    if (batch == 0 || n_kv == 0 || rows == 0) return RT_OK;
    const rt::Kv4Cache c{k_codes, k_scales, v_codes, v_scales};
    if (!k || !v) return RT_ERR_NULL_POINTER;
    if (const int rc = check_planes(c)) return rc;
    if (!aligned16(k) || !aligned16(v)) return RT_ERR_ALIGNMENT;
    if (rows > kMostSeq) return RT_ERR_UNSUPPORTED;
    const int64_t dense[3] = {n_kv * rows * head_dim, rows * head_dim, head_dim};
    const int64_t *ks = k_strides ? k_strides : dense, *vs = v_strides ? v_strides : dense;
    for (int i = 0; i < 3; ++i)
        if (ks[i] % 8 || vs[i] % 8) return RT_ERR_ALIGNMENT;
    return (int)rt::launch_kv4_append(c, k, v, ks, vs, batch, n_kv, rows, head_dim, max_seq, pos, positions, lens,
                                      as_stream(stream));
}

int rt_rope_kv4_append(void* q, const void* k_in, const void* v_in, void* k_codes, void* k_scales, void* v_codes,
                       void* v_scales, const float* inv_freq, int64_t batch, int n_heads, int n_kv, int head_dim,
                       int64_t max_seq, int64_t pos, const int32_t* positions, int64_t slot, const int32_t* slots,
                       int rope_style, void* stream) {
    if (const int rc = check_shape(batch, n_kv, head_dim, max_seq)) return rc;
    if (n_heads < 0) return RT_ERR_BAD_LENGTH;
    if (n_heads > 65535 || (rope_style != RT_ROPE_HALF_SPLIT && rope_style != RT_ROPE_ADJACENT)) return RT_ERR_UNSUPPORTED;
    if (!positions && (pos < 0 || pos > kMostSeq)) return RT_ERR_BAD_LENGTH;
    if (!slots && (slot >= 0 ? slot >= max_seq : !positions && pos >= max_seq)) return RT_ERR_BAD_LENGTH;
    if (batch == 0 || n_heads + n_kv == 0) return RT_OK;
    if (!inv_freq || (n_heads > 0 && !q) || (n_kv > 0 && (!k_in || !v_in))) return RT_ERR_NULL_POINTER;
    const rt::Kv4Cache c{k_codes, k_scales, v_codes, v_scales};
    if (n_kv > 0)
        if (const int rc = check_planes(c)) return rc;
    if (!aligned16(q) || !aligned16(k_in) || !aligned16(v_in)) return RT_ERR_ALIGNMENT;
    return (int)rt::launch_rope_kv4_append(c, q, k_in, v_in, inv_freq, batch, n_heads, n_kv, head_dim, max_seq, pos, positions,
                                           slot, slots, rope_style, as_stream(stream));
}

int rt_kv4_read(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* k_out,
                void* v_out, int64_t batch, int n_kv, int head_dim, int64_t max_seq, int64_t rows, int64_t start,
                const int32_t* starts, const int32_t* kv_lens, void* stream) {
    if (const int rc = check_shape(batch, n_kv, head_dim, max_seq)) return rc;
    if (rows < 0) return RT_ERR_BAD_LENGTH;
    if (batch == 0 || n_kv == 0 || rows == 0) return RT_OK;
    const rt::Kv4Cache c{k_codes, k_scales, v_codes, v_scales};
    if (!k_out || !v_out) return RT_ERR_NULL_POINTER;
    if (const int rc = check_planes(c)) return rc;
    if (!aligned16(k_out) || !aligned16(v_out)) return RT_ERR_ALIGNMENT;
    if (rows > kMostSeq || start > kMostSeq || start < -kMostSeq) return RT_ERR_UNSUPPORTED;
    return (int)rt::launch_kv4_read(c, k_out, v_out, batch, n_kv, head_dim, max_seq, rows, start, starts, kv_lens,
                                    as_stream(stream));
}

size_t rt_kv4_decode_workspace_bytes(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int head_dim, int64_t max_seq,
                                     int weighed) {
    if (batch <= 0 || n_kv_heads <= 0 || n_heads <= 0 || max_seq <= 0 || n_heads > 8 * n_kv_heads ||
        check_shape(batch, n_kv_heads, head_dim, max_seq) != RT_OK)
        return 0;
    return rt::kv4_decode_workspace_bytes(batch, (int)n_heads, (int)n_kv_heads, head_dim, max_seq, weighed != 0);
}

int rt_kv4_decode(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                  void* out, float* lse, float* weights, int64_t batch, int64_t n_heads, int64_t n_kv_heads,
                  int head_dim, int64_t max_seq, const int32_t* kv_lens, int64_t kv_len_uniform, float scale,
                  void* workspace, size_t workspace_bytes, void* stream) {
    if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads != 0) return RT_ERR_HEAD_COUNT;
    if (const int rc = check_shape(batch, n_kv_heads, head_dim, max_seq)) return rc;
    if (max_seq == 0 || (!kv_lens && (kv_len_uniform < 0 || kv_len_uniform > max_seq))) return RT_ERR_BAD_LENGTH;
    if (n_heads / n_kv_heads > 8 || batch * n_heads > 0x7fffffff) return RT_ERR_UNSUPPORTED;
    if (batch == 0) return RT_OK;
    const rt::Kv4Cache c{k_codes, k_scales, v_codes, v_scales};
    if (!q || !out) return RT_ERR_NULL_POINTER;
    if (const int rc = check_planes(c)) return rc;
    if (!aligned16(q) || !aligned16(out)) return RT_ERR_ALIGNMENT;
    const size_t need = rt_kv4_decode_workspace_bytes(batch, n_heads, n_kv_heads, head_dim, max_seq, weights != nullptr);
    if (need && (!workspace || workspace_bytes < need)) return RT_ERR_WORKSPACE;
    if (need && !aligned16(workspace)) return RT_ERR_ALIGNMENT;
    return (int)rt::launch_kv4_decode(c, q, out, lse, weights, batch, (int)n_heads, (int)n_kv_heads, head_dim, max_seq,
                                      kv_lens, kv_len_uniform, default_scale(scale, head_dim), workspace, as_stream(stream));
}

int rt_kv_weigh_bf16(const void* q, const void* k_cache, const float* lse, float* weights, int64_t batch,
                     int64_t n_heads, int64_t n_kv_heads, int64_t seq_q, int head_dim, int64_t max_seq,
                     const int32_t* kv_lens, int64_t kv_len_uniform, float scale, void* stream) {
    if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads != 0) return RT_ERR_HEAD_COUNT;
    if (const int rc = check_shape(batch, n_kv_heads, head_dim, max_seq)) return rc;
    if (seq_q < 0 || max_seq == 0 || (!kv_lens && (kv_len_uniform < 0 || kv_len_uniform > max_seq))) return RT_ERR_BAD_LENGTH;
    if (n_heads / n_kv_heads > 8 || seq_q > kMostSeq / 8) return RT_ERR_UNSUPPORTED;
    if (batch == 0 || seq_q == 0) return RT_OK;
    if (!q || !k_cache || !lse || !weights) return RT_ERR_NULL_POINTER;
    if (!aligned16(q) || !aligned16(k_cache)) return RT_ERR_ALIGNMENT;
    return (int)rt::launch_kv_weigh(q, k_cache, lse, weights, batch, (int)n_heads, (int)n_kv_heads, seq_q, head_dim, max_seq,
                                    kv_lens, kv_len_uniform, default_scale(scale, head_dim), as_stream(stream));
}

int rt_kv_evict(const void* const* src, void* const* dst, const int32_t* row_bytes, int n_planes, const float* weights,
                float* weights_out, int32_t* kept, int32_t* lens_out, int64_t batch, int64_t n_kv_heads,
                int64_t max_seq, int64_t max_seq_out, const int32_t* kv_lens, int64_t kv_len_uniform, int64_t keep,
                int64_t recent, void* stream) {
    if (batch < 0 || n_kv_heads < 0 || max_seq <= 0 || max_seq_out <= 0 || keep < 1 || keep > max_seq_out || recent < 0 ||
        recent > keep || (!kv_lens && (kv_len_uniform < 0 || kv_len_uniform > max_seq)))
        return RT_ERR_BAD_LENGTH;
    if (n_planes < 1 || n_planes > rt::EvictPlanes::kMost || batch > 65535 || n_kv_heads > 65535 || max_seq > kMostSeq ||
        max_seq_out > kMostSeq || batch * n_kv_heads > 65535)
        return RT_ERR_UNSUPPORTED;
    if (batch == 0 || n_kv_heads == 0) return RT_OK;
    if (!src || !dst || !row_bytes || !weights || !weights_out || !kept || !lens_out) return RT_ERR_NULL_POINTER;
    rt::EvictPlanes p = {};
    p.n = n_planes;
    const size_t rows_in = (size_t)(batch * n_kv_heads) * max_seq, rows_out = (size_t)(batch * n_kv_heads) * max_seq_out;
    for (int i = 0; i < n_planes; ++i) {
        if (!src[i] || !dst[i]) return RT_ERR_NULL_POINTER;
        if (row_bytes[i] <= 0 || row_bytes[i] % 8 || row_bytes[i] > 4096) return RT_ERR_UNSUPPORTED;
        if (!aligned16(src[i]) || !aligned16(dst[i])) return RT_ERR_ALIGNMENT;
        p.src[i] = src[i], p.dst[i] = dst[i], p.row_bytes[i] = row_bytes[i];
    }
    // The selection and the move have no order: what is written must be nothing that is read, and nothing twice.
    constexpr int kMost = rt::EvictPlanes::kMost;
    Bytes read[kMost + 2], written[kMost + 3];
    int n_read = 0, n_written = 0;
    for (int i = 0; i < n_planes; ++i) {
        read[n_read++] = {src[i], rows_in * row_bytes[i]};
        written[n_written++] = {dst[i], rows_out * row_bytes[i]};
    }
    read[n_read++] = {weights, rows_in * sizeof(float)};
    if (kv_lens) read[n_read++] = {kv_lens, batch * sizeof(int32_t)};
    written[n_written++] = {weights_out, rows_out * sizeof(float)};
    written[n_written++] = {kept, (size_t)(batch * n_kv_heads) * keep * sizeof(int32_t)};
    written[n_written++] = {lens_out, batch * sizeof(int32_t)};
    for (int i = 0; i < n_written; ++i) {
        for (int j = 0; j < n_read; ++j)
            if (overlap(written[i], read[j])) return RT_ERR_UNSUPPORTED;
        for (int j = 0; j < i; ++j)
            if (overlap(written[i], written[j])) return RT_ERR_UNSUPPORTED;
    }
    return (int)rt::launch_kv_evict(p, weights, weights_out, kept, lens_out, batch, (int)n_kv_heads, max_seq, max_seq_out,
                                    kv_lens, kv_len_uniform, keep, recent, as_stream(stream));
}

}  // extern "C"

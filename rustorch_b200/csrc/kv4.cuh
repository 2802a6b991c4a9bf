// The 4-bit KV cache's format (include/rustorch_attn.h states it) as device helpers.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace rt {

// A row's shape.  Its octets (8 values, 4 bytes of codes) are dealt to the groups in turn, span by span: octet o of a span
// belongs to the span's group o % kSpanGroups.
template <int D>
struct Kv4Row {
    static constexpr int kSpan = D < 128 ? D : 128;
    static constexpr int kSpanGroups = kSpan / 32, kSpanOctets = kSpan / 8;
    static constexpr int kGroups = D / 32, kOctets = D / 8;
    static constexpr int kCodeBytes = D / 2, kScaleBytes = D / 8;
    __host__ __device__ static constexpr int group_of_octet(int o) {
        return (o / kSpanOctets) * kSpanGroups + o % kSpanGroups;
    }
};

// {scale, lo} of a group as f32.
__device__ __forceinline__ float2 kv4_scale(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// The value of code c (0..15).
__device__ __forceinline__ float kv4_value(float2 s, uint32_t c) { return fmaf(s.x, (float)c, s.y); }

}  // namespace rt

// Device helpers of the paged key-value cache: conversions, page lookup.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv_cache.cuh"

namespace eosb {

// ---------------------------------------------------------------- conversions
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bf16x2_of(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 f16x2_floats(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 bf16x2_floats(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// two e4m3 / e2m1 codes, the first in the low bits
__device__ __forceinline__ uint32_t e4m3x2_of(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e2m1x2_of(float lo, float hi) {
    uint32_t r;
    asm("{\n .reg .b8 c;\n cvt.rn.satfinite.e2m1x2.f32 c, %1, %2;\n cvt.u32.u8 %0, c;\n}" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// four e4m3 codes -> two f16 pairs
__device__ __forceinline__ void f16_of_e4m3x4(uint32_t w, uint32_t& a, uint32_t& b) {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(a), "=r"(b)
        : "r"(w));
}
// eight e2m1 codes -> four f16 pairs
__device__ __forceinline__ void f16_of_e2m1x8(uint32_t w, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm("{\n .reg .b8 p, q, r, s;\n mov.b32 {p, q, r, s}, %4;\n cvt.rn.f16x2.e2m1x2 %0, p;\n cvt.rn.f16x2.e2m1x2 %1, q;\n"
        " cvt.rn.f16x2.e2m1x2 %2, r;\n cvt.rn.f16x2.e2m1x2 %3, s;\n}"
        : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
        : "r"(w));
}
// value of a scale byte: 2^(e - 127) for 1 <= e <= 254, NaN for 255 (a block that holds a non-finite value)
__device__ __forceinline__ float kv_scale_value(uint32_t e) { return e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(e << 23); }

// ---------------------------------------------------------------- pages
// The record of `rec` (record index in sequence b) and head h; null when the table or the page id is out of range.
__device__ __forceinline__ uint8_t* kv_record(const KvPool& pool, const KvSeqs& s, int b, int rec, int h) {
    const int slot = rec / pool.records_per_page;
    if (slot >= s.max_pages) return nullptr;
    const int page = __ldg(s.table + (int64_t)b * s.max_pages + slot);
    if (page < 0 || page >= pool.pages) return nullptr;
    return pool.base + (((int64_t)page * pool.heads + h) * pool.records_per_page + (rec - slot * pool.records_per_page)) *
                           (int64_t)pool.record_bytes;
}

// ---------------------------------------------------------------- rows of a call's tensors
// N (4 or 8) consecutive elements as floats / from floats; vec: the address is aligned for 16-byte (or, for four
// 16-bit elements, 8-byte) accesses.
template <int N>
__device__ __forceinline__ void load_row(const void* p, int64_t at, int type, int vec, float (&x)[N]) {
    if (type == kTypeF32) {
        const float* f = static_cast<const float*>(p) + at;
        if (vec) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const float4 v = *reinterpret_cast<const float4*>(f + i);
                x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = f[i];
        }
        return;
    }
    const uint16_t* h = static_cast<const uint16_t*>(p) + at;
    uint32_t w[N / 2];
    if (vec) {
        if constexpr (N == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(h);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(h);
            w[0] = v.x, w[1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float2 v = type == kTypeF16 ? f16x2_floats(w[i]) : bf16x2_floats(w[i]);
        x[2 * i] = v.x, x[2 * i + 1] = v.y;
    }
}
// 16 bytes from an address that is aligned to 2 bytes only, out of line
__device__ __noinline__ inline uint4 load16_unaligned(const uint8_t* p) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    uint4 v;
    v.x = (uint32_t)h[0] | (uint32_t)h[1] << 16, v.y = (uint32_t)h[2] | (uint32_t)h[3] << 16;
    v.z = (uint32_t)h[4] | (uint32_t)h[5] << 16, v.w = (uint32_t)h[6] | (uint32_t)h[7] << 16;
    return v;
}
// elements one by one, out of line: for rows that are not aligned
__device__ __noinline__ inline void store_elements(void* p, int type, int n, float a, float b, float c, float d) {
    for (int i = 0; i < n; ++i) {
        const float y = i == 0 ? a : i == 1 ? b : i == 2 ? c : d;
        if (type == kTypeF32) static_cast<float*>(p)[i] = y;
        else static_cast<uint16_t*>(p)[i] = (uint16_t)(type == kTypeF16 ? f16x2_of(y, 0.f) : bf16x2_of(y, 0.f));
    }
}
template <int N>
__device__ __forceinline__ void store_row(void* p, int64_t at, int type, int vec, const float (&x)[N]) {
    uint8_t* dst = static_cast<uint8_t*>(p) + at * (type == kTypeF32 ? 4 : 2);
    if (!vec) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            store_elements(dst + i * (type == kTypeF32 ? 4 : 2), type, 4, x[i], x[i + 1], x[i + 2], x[i + 3]);
        return;
    }
    if (type == kTypeF32) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        return;
    }
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = type == kTypeF16 ? f16x2_of(x[2 * i], x[2 * i + 1]) : bf16x2_of(x[2 * i], x[2 * i + 1]);
    if constexpr (N == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
}

}  // namespace eosb

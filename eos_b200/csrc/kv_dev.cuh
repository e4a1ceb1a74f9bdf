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

// two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

// ---------------------------------------------------------------- records
// The bytes of one lane at `plane0`, BYTES of them (see kv_lane_offset)
template <int BYTES>
__device__ __forceinline__ void load_lane(const uint8_t* plane0, int lane, uint32_t (&w)[BYTES / 4]) {
#pragma unroll
    for (int p = 0; p + 16 <= BYTES; p += 16) {
        const uint4 v = *reinterpret_cast<const uint4*>(plane0 + p * 32 + lane * 16);
        w[p / 4] = v.x, w[p / 4 + 1] = v.y, w[p / 4 + 2] = v.z, w[p / 4 + 3] = v.w;
    }
    constexpr int r = BYTES & 15, p = BYTES - r;
    if constexpr (r >= 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(plane0 + p * 32 + lane * 8);
        w[p / 4] = v.x, w[p / 4 + 1] = v.y;
    }
    if constexpr ((r & 7) != 0)
        w[BYTES / 4 - 1] = *reinterpret_cast<const uint32_t*>(plane0 + p * 32 + (r >= 8 ? 256 : 0) + lane * 4);
}

// Scale bytes of one token's key, packed four to a word
template <int NB>
__device__ __forceinline__ void load_scales(const uint8_t* p, uint32_t (&a)[(NB + 3) / 4]) {
    if constexpr (NB == 1) a[0] = *p;
    else if constexpr (NB == 2) a[0] = *reinterpret_cast<const uint16_t*>(p);
    else if constexpr (NB <= 4) a[0] = *reinterpret_cast<const uint32_t*>(p);
    else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        a[0] = w.x, a[1] = w.y;
    }
}
// Scale bytes of a token pair's values: block b in byte 2 (b % 2) (first token) and the next (second) of word b / 2
template <int NB>
__device__ __forceinline__ void load_pair_scales(const uint8_t* p, uint32_t (&w)[(NB + 1) / 2]) {
    if constexpr (NB == 1) w[0] = *reinterpret_cast<const uint16_t*>(p);
    else if constexpr (NB == 2) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (NB <= 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z;
        if constexpr (NB > 6) w[3] = v.w;
    }
}
// ---------------------------------------------------------------- errors
// Counts an error that a call met (see KvWork).
__device__ __forceinline__ void kv_report(uint64_t* errors, int code) {
    atomicAdd(reinterpret_cast<unsigned long long*>(errors) + (code - kStatusPipelineTimeout), 1ull);
}

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
// 16 bytes from an address that is aligned to 2 bytes only, out of line
__device__ __noinline__ inline uint4 load16_unaligned(const uint8_t* p) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    uint4 v;
    v.x = (uint32_t)h[0] | (uint32_t)h[1] << 16, v.y = (uint32_t)h[2] | (uint32_t)h[3] << 16;
    v.z = (uint32_t)h[4] | (uint32_t)h[5] << 16, v.w = (uint32_t)h[6] | (uint32_t)h[7] << 16;
    return v;
}
// four elements of an aligned row
__device__ __forceinline__ void store_row(void* p, int64_t at, int type, const float (&x)[4]) {
    if (type == kTypeF32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + at) = make_float4(x[0], x[1], x[2], x[3]);
        return;
    }
    const uint32_t a = type == kTypeF16 ? f16x2_of(x[0], x[1]) : bf16x2_of(x[0], x[1]);
    const uint32_t b = type == kTypeF16 ? f16x2_of(x[2], x[3]) : bf16x2_of(x[2], x[3]);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + at) = make_uint2(a, b);
}

}  // namespace eosb

// Paged key-value cache: quantising tokens as they are written, and reading them back (kernel templates, one instance per
// format, head size and element type; kv_io_*.cu compile them).
//
// Formats.  f16 / bf16 hold each element rounded to nearest.  mx8 (e4m3) and mx4 (e2m1) hold, for every 32 consecutive
// elements of a head's vector, one scale 2^e with the smallest e >= -126 for which max|x| <= top 2^e (top = 448 or 6,
// the type's largest value, so nothing saturates) and the codes x / 2^e rounded to nearest, ties to even.  The scale is
// a power of two: the division is exact, every code has one right answer, and a code times its scale is exact in fp32.
// A block that holds an infinity or a NaN is stored as NaN (scale byte 255, codes zero).
//
// One warp per (record, head): it owns all 16 tokens of the record that the call writes, so a record that is completed
// by several calls needs no atomics, and neighbouring tokens' codes are merged by a plain read-modify-write.  Loads are
// issued together before the first is used, and codes are built in registers in the order of the record.
//
// What bounds them (131072 tokens of 8 heads of 128, 16-bit rows): the 16-bit formats HBM -- append and read 163 us each, 6.6
// TB/s.  mx8 append 131 us, 6.2 TB/s: a warp's two rounds of loads with the quantisation between them (137 when the page was
// looked up before the first); read 131 us, 6.2 TB/s.  mx4 append 124 us, 5.5 TB/s, read 111 us, 6.1
// TB/s.  (DRAM moves the rows and the records once: 537 + 249 MB and 279 + 484 MB at mx8, what an append leaves in the L2 of
// its 279 MB aside.)  One token for each of 64 sequences, the read back included: 10 to 11 us, two launches and the latency of
// starts, rows and page table, and the record's old bytes one after the other.
#pragma once
#include "kv_dev.cuh"
#include "kv_split.cuh"

namespace eosb {

constexpr int kKvIoWarps = 8;

// The sequence and record that work unit u of a call stands for.  Warp-wide search, 32 probes a step; lanes agree on the result.
__device__ __forceinline__ KvUnit kv_unit(const KvSeqs& s, int64_t tokens, int64_t u, int lane, uint64_t* errors) {
    KvUnit r;
    r.ok = false;
    int64_t row, n, first = 0;
    int64_t start;   // (asked for together with the row offsets)
    if (s.cu == nullptr) {
        r.b = (int)u, row = u, n = 1;
        start = __ldg(s.starts + r.b);
    } else {
        int lo = 0, hi = s.batch;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) >> 5;
            const int probe = lo + lane * step;
            const bool below = lane == 0 || (probe < hi && kv_unit_start(__ldg(s.cu + probe), probe) <= u);
            const int top = 31 - __clz(__ballot_sync(0xffffffffu, below));
            lo += top * step;
            hi = min(hi, lo + step);
        }
        r.b = lo;
        row = __ldg(s.cu + lo);
        start = __ldg(s.starts + lo);
        n = (int64_t)__ldg(s.cu + lo + 1) - row;
        first = u - kv_unit_start((int)row, lo);
    }
    if (n == 0) return r;
    if (n < 0 || row < 0 || row + n > tokens || start < 0 || start + n > 0x7fffffffLL) {
        if (lane == 0) kv_report(errors, kStatusBadSequence);
        return r;
    }
    r.ok = kv_place(r, row, n, start, first);
    return r;
}

// The row offsets of a call, looked over by one block (the last; the work's own would not meet all that is wrong, for where offsets
// descend the search above passes sequences by): ascending from 0 or more to `tokens` or less.
__device__ __forceinline__ void kv_check_offsets(const KvSeqs& s, int64_t tokens, uint64_t* errors) {
    bool bad = false;
    for (int b = threadIdx.x; b < s.batch; b += blockDim.x) {
        const int from = __ldg(s.cu + b), to = __ldg(s.cu + b + 1);
        bad |= from < 0 || to < from || to > tokens;
    }
    if (__syncthreads_or(bad) && threadIdx.x == 0) kv_report(errors, kStatusBadSequence);
}

// ---------------------------------------------------------------- elements
// N (4 or 8) consecutive elements of a call's tensor, as they lie in memory
template <int TYPE, int N>
struct KvRow {
    static constexpr int kWords = TYPE == kTypeF32 ? N : N / 2;
    uint32_t w[kWords];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void load(const uint8_t* p, int vec) {
        if (vec) {
            if constexpr (kWords == 2) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
                w[0] = v.x, w[1] = v.y;
            } else if constexpr (kWords == 8) {   // a lane's 32 bytes are a whole sector
                if (vec > 1) {
                    ld_global_v8(p, w);
                } else {
#pragma unroll
                    for (int i = 0; i < kWords; i += 4) {
                        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
                        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
                    }
                }
            } else {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
            }
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = (uint32_t)h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ float2 pair(int i) const {   // elements 2i, 2i + 1
        if constexpr (TYPE == kTypeF32) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else if constexpr (TYPE == kTypeF16) return f16x2_floats(w[i]);
        else return bf16x2_floats(w[i]);
    }
    // Largest magnitude, as bits that compare like it with infinities and NaN on top: of fp32, or two 16-bit halves
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            m = TYPE == kTypeF32 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
        return m;
    }
};
// the larger half of a 16-bit pair's, as its fp32 bits
template <int TYPE>
__device__ __forceinline__ uint32_t top_bits(uint32_t h) {   // h < 2^16
    if constexpr (TYPE == kTypeF16) return __float_as_uint(f16x2_floats(h).x);
    return h << 16;
}

// scale byte of a block with the largest magnitude amax (its fp32 bits): its exponent less that of the largest code, one
// more where the mantissa passes that code's (448 = 1.75 2^8, 6 = 1.5 2^2); 255 for infinities and NaN
template <int FMT>
__device__ __forceinline__ uint32_t kv_scale_byte(uint32_t amax_bits) {
    const int byte = (int)((amax_bits + (FMT == kKvMx8 ? 0x1fffffu : 0x3fffffu)) >> 23) - (FMT == kKvMx8 ? 8 : 2);
    return amax_bits >= 0x7f800000u ? 255u : (uint32_t)max(byte, 1);
}
// 2^-e of a scale byte; 0 for a block stored as NaN
__device__ __forceinline__ float kv_inverse_scale(uint32_t byte) { return __uint_as_float(byte == 255u ? 0u : (254u - byte) << 23); }

__device__ __forceinline__ uint32_t e4m3x4_of(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
__device__ __forceinline__ uint32_t e2m1x8_of(float a, float b, float c, float d, float e, float f, float g, float h) {
    uint32_t r;
    asm("{\n .reg .b8 p, q, r, s;\n cvt.rn.satfinite.e2m1x2.f32 p, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 q, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 r, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 s, %8, %7;\n mov.b32 %0, {p, q, r, s};\n}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d), "f"(e), "f"(f), "f"(g), "f"(h));
    return r;
}

// The bytes of one lane (see kv_lane_offset)
template <int BYTES>
__device__ __forceinline__ void store_lane(uint8_t* plane0, int lane, const uint32_t (&w)[BYTES / 4]) {
#pragma unroll
    for (int p = 0; p + 16 <= BYTES; p += 16)
        *reinterpret_cast<uint4*>(plane0 + p * 32 + lane * 16) = make_uint4(w[p / 4], w[p / 4 + 1], w[p / 4 + 2], w[p / 4 + 3]);
    constexpr int r = BYTES & 15, p = BYTES - r;
    if constexpr (r >= 8) *reinterpret_cast<uint2*>(plane0 + p * 32 + lane * 8) = make_uint2(w[p / 4], w[p / 4 + 1]);
    if constexpr ((r & 7) != 0) *reinterpret_cast<uint32_t*>(plane0 + p * 32 + (r >= 8 ? 256 : 0) + lane * 4) = w[BYTES / 4 - 1];
}

// ---------------------------------------------------------------- append
// Raw words that a lane holds of the keys, or of the values.  The block-scaled formats are bound by latency, so the values
// are loaded when the keys are done with, and the registers that saves go to more warps (16-bit rows of 128 to mx8: 32
// warps an SM 159 us with the read back (155 now), 24 warps 168, 16 warps with all loads first 176; fetching the values' rows into
// the L2 meanwhile brings nothing); the plain formats run at HBM's rate with all loads first.  The warps are bought with spills
// (-Xptxas -v, bytes stored and loaded a thread): 16-bit rows of 128 to mx8 64 registers, 124 and 140, to mx4 48 and 80; of 192
// 80 registers, 168 to 176 and 196 to 204, to mx4 80 to 88 and 128 to 140; of 256 to mx8 32 and 32; of 96 64 and 96; fp32 rows 4 to 48.
__host__ __device__ constexpr int kv_raw_words(int nb, int type) { return type == kTypeF32 ? 16 * nb : 8 * nb; }
__host__ __device__ constexpr int kv_append_blocks(int fmt, int nb, int type) {
    return fmt < kKvMx8 ? 1 : kv_raw_words(nb, type) <= 32 ? 4 : kv_raw_words(nb, type) <= 48 ? 3 : kv_raw_words(nb, type) <= 64 ? 2 : 1;
}
template <int FMT, int NB, int TYPE>
__global__ void __launch_bounds__(kKvIoWarps * 32, kv_append_blocks(FMT, NB, TYPE))
    kv_append_kernel(KvPool pool, KvSeqs seqs, KvRows key, KvRows value, int64_t tokens, int64_t units, uint64_t* errors) {
    constexpr bool kMx = FMT >= kKvMx8;
    constexpr int KP = kv_key_piece(FMT), VP = kv_value_piece(FMT), NS = kv_scale_stride(NB), ES = TYPE == kTypeF32 ? 4 : 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t w = (int64_t)blockIdx.x * kKvIoWarps + (threadIdx.x >> 5);
    const int64_t u = w / pool.heads;
    if (u >= units) {   // (all warps of the last block)
        if (seqs.cu != nullptr && blockIdx.x == gridDim.x - 1) kv_check_offsets(seqs, tokens, errors);
        return;
    }
    const int h = (int)(w - u * pool.heads);
    const KvUnit un = kv_unit(seqs, tokens, u, lane, errors);
    if (!un.ok) return;
    const int base = un.rec * kKvRecord;
    const bool full = un.hi - un.lo == kKvRecord && key.vec && value.vec;   // the usual record of a prompt: no conditions on the loads
    // ---- keys: lane (g, t) owns 8 elements of the tokens g and g + 8 in every block
    bool kmine[2];
    KvRow<TYPE, 8> kx[2][NB];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int pos = base + 8 * j + g;
        kmine[j] = pos >= un.lo && pos < un.hi;
        const uint8_t* p = static_cast<const uint8_t*>(key.p) + ((un.row0 + pos) * key.token_stride + (int64_t)h * key.head_stride + 8 * t) * ES;
        if (full) {
#pragma unroll
            for (int b = 0; b < NB; ++b) kx[j][b].load(p + 32 * b * ES, key.vec);
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                kx[j][b].zero();
                if (kmine[j]) kx[j][b].load(p + 32 * b * ES, key.vec);
            }
        }
    }
    // the rows are on their way while the page is looked up
    uint8_t* rec = kv_record(pool, seqs, un.b, un.rec, h);
    if (rec == nullptr) {
        if (lane == 0) kv_report(errors, kStatusBadPage);
        return;
    }
    // ---- values: lane (g, t) owns elements 4 g .. + 3 of every block for the tokens 2t, 2t+1, 2t+8, 2t+9
    bool vmine[4];
    const uint8_t* vp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = base + 2 * t + (i & 1) + 8 * (i >> 1);
        vmine[i] = pos >= un.lo && pos < un.hi;
        vp[i] = static_cast<const uint8_t*>(value.p) + ((un.row0 + pos) * value.token_stride + (int64_t)h * value.head_stride + 4 * g) * ES;
    }
    KvRow<TYPE, 4> vx[4][NB];
    auto load_values = [&]() {
        if (full) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) vx[i][b].load(vp[i] + 32 * b * ES, 1);
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vx[i][b].zero();
                    if (vmine[i]) vx[i][b].load(vp[i] + 32 * b * ES, value.vec);
                }
        }
    };
    constexpr bool kLate = kMx || kv_raw_words(NB, TYPE) >= 96;   // (fp32 rows of 192 elements do not fit the registers beside the keys)
    if constexpr (!kLate) load_values();
    // the values' codes that this call leaves alone
    const bool any = vmine[0] || vmine[1] || vmine[2] || vmine[3], all = vmine[0] && vmine[1] && vmine[2] && vmine[3];
    uint32_t old[NB * VP / 4];
    if (any && !all) load_lane<NB * VP>(rec + kv_value_offset(FMT, NB), lane, old);

    if constexpr (!kMx) {
        // words of the two tokens in turn
        uint32_t kw[NB * 8];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 x = kx[j][b].pair(i);
                    kw[8 * b + 4 * (i >> 1) + 2 * (i & 1) + j] = TYPE == FMT + 1 ? kx[j][b].w[i % KvRow<TYPE, 8>::kWords]   // (f16 to f16, bf16 to bf16)
                                                                 : FMT == kKvF16 ? f16x2_of(x.x, x.y) : bf16x2_of(x.x, x.y);
                }
        if (kmine[0] && kmine[1]) {
            store_lane<NB * 32>(rec, lane, kw);
        } else if (kmine[0] || kmine[1]) {
#pragma unroll
            for (int i = 0; i < NB * 8; i += 2)
                *reinterpret_cast<uint32_t*>(rec + kv_lane_offset(NB * 32, lane, 4 * i + (kmine[1] ? 4 : 0))) = kmine[1] ? kw[i + 1] : kw[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t codes[NB * KP / 4];
            uint32_t bytes[2] = {0u, 0u};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                uint32_t m = kx[j][b].top();
                if constexpr (TYPE == kTypeF32) {
                    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                } else {
                    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    m = top_bits<TYPE>(max(m & 0xffffu, m >> 16));
                }
                const uint32_t byte = kv_scale_byte<FMT>(m);
                const float inv = kv_inverse_scale(byte);
                bytes[b / 4] |= byte << (8 * (b & 3));
                float2 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = mul2(kx[j][b].pair(i), make_float2(inv, inv));
                if (__any_sync(0xffffffffu, inv == 0.f)) {   // (a NaN or infinity times 0 is a NaN; its code is to be zero)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (inv == 0.f) x[i] = make_float2(0.f, 0.f);
                }
                if constexpr (FMT == kKvMx8) {
                    codes[2 * b] = e4m3x4_of(x[0].x, x[0].y, x[1].x, x[1].y);
                    codes[2 * b + 1] = e4m3x4_of(x[2].x, x[2].y, x[3].x, x[3].y);
                } else {
                    codes[b] = e2m1x8_of(x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y);
                }
            }
            if (kmine[j]) {
                store_lane<NB * KP>(rec + j * 32 * NB * KP, lane, codes);
                if (t == 0) {
                    uint8_t* p = rec + kv_key_scale_offset(FMT, NB) + (8 * j + g) * NS;
                    if constexpr (NS == 1) *p = (uint8_t)bytes[0];
                    else if constexpr (NS == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)bytes[0];
                    else if constexpr (NS == 4) *reinterpret_cast<uint32_t*>(p) = bytes[0];
                    else *reinterpret_cast<uint2*>(p) = make_uint2(bytes[0], bytes[1]);
                }
            }
        }
    }

    // ---- values
    if constexpr (kLate) load_values();
    uint32_t v[NB * VP / 4], keep[4];   // keep: bits of a block's words that belong to tokens of other calls
    uint32_t scales[4][2] = {};         // of each token: the blocks' scale bytes, and the largest and smallest of them
    uint32_t top[4] = {0u, 0u, 0u, 0u}, least[4] = {255u, 255u, 255u, 255u};
    if constexpr (!kMx) {
        keep[0] = (vmine[0] ? 0u : 0x0000ffffu) | (vmine[1] ? 0u : 0xffff0000u);
        keep[1] = (vmine[2] ? 0u : 0x0000ffffu) | (vmine[3] ? 0u : 0xffff0000u);
    } else if constexpr (FMT == kKvMx8) {
        keep[0] = (vmine[0] ? 0u : 0xffu) | (vmine[1] ? 0u : 0xff00u) | (vmine[2] ? 0u : 0xff0000u) | (vmine[3] ? 0u : 0xff000000u);
    } else {
        keep[0] = ((vmine[0] ? 0u : 0xfu) | (vmine[1] ? 0u : 0xf0u) | (vmine[2] ? 0u : 0xf00u) | (vmine[3] ? 0u : 0xf000u)) * 0x10001u;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        float x[4][4];   // [token][element]
        if constexpr (kMx) {
            uint32_t m[4];   // fp32 bits of the tokens' largest magnitudes
            if constexpr (TYPE == kTypeF32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    m[i] = vx[i][b].top();
                    m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 4));
                    m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 8));
                    m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 16));
                }
            } else {
                // two tokens a word
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint32_t a = vx[2 * p][b].top(), c = vx[2 * p + 1][b].top();
                    uint32_t y = __vmaxu2(__byte_perm(a, c, 0x5410), __byte_perm(a, c, 0x7632));
                    y = __vmaxu2(y, __shfl_xor_sync(0xffffffffu, y, 4));
                    y = __vmaxu2(y, __shfl_xor_sync(0xffffffffu, y, 8));
                    y = __vmaxu2(y, __shfl_xor_sync(0xffffffffu, y, 16));
                    m[2 * p] = top_bits<TYPE>(y & 0xffffu), m[2 * p + 1] = top_bits<TYPE>(y >> 16);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t byte = kv_scale_byte<FMT>(m[i]);
                const float inv = kv_inverse_scale(byte);
                scales[i][b / 4] |= byte << (8 * (b & 3));
                top[i] = max(top[i], byte);
                least[i] = min(least[i], byte);
                const float2 y = mul2(vx[i][b].pair(0), make_float2(inv, inv)), z = mul2(vx[i][b].pair(1), make_float2(inv, inv));
                x[i][0] = y.x, x[i][1] = y.y, x[i][2] = z.x, x[i][3] = z.y;
            }
            if (__any_sync(0xffffffffu, max(max(top[0], top[1]), max(top[2], top[3])) == 255u)) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((scales[i][b / 4] >> (8 * (b & 3)) & 0xffu) == 255u) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 y = vx[i][b].pair(0), z = vx[i][b].pair(1);
                x[i][0] = y.x, x[i][1] = y.y, x[i][2] = z.x, x[i][3] = z.y;
            }
        }
        if constexpr (!kMx) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int at = 8 * b + 4 * (e >> 1) + 2 * p + (e & 1);
                    if constexpr (TYPE == FMT + 1)
                        v[at] = __byte_perm(vx[2 * p][b].w[e >> 1], vx[2 * p + 1][b].w[e >> 1], e & 1 ? 0x7632 : 0x5410);
                    else
                        v[at] = FMT == kKvF16 ? f16x2_of(x[2 * p][e], x[2 * p + 1][e]) : bf16x2_of(x[2 * p][e], x[2 * p + 1][e]);
                }
        } else if constexpr (FMT == kKvMx8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * b + e] = e4m3x4_of(x[0][e], x[1][e], x[2][e], x[3][e]);
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                v[2 * b + e] = e2m1x8_of(x[0][2 * e], x[1][2 * e], x[2][2 * e], x[3][2 * e], x[0][2 * e + 1], x[1][2 * e + 1],
                                         x[2][2 * e + 1], x[3][2 * e + 1]);
        }
    }
    if (any) {
        if (!all) {
#pragma unroll
            for (int i = 0; i < NB * VP / 4; ++i) {
                const uint32_t k = kMx ? keep[0] : keep[i >> 1 & 1];
                v[i] = (v[i] & ~k) | (old[i] & k);
            }
        }
        store_lane<NB * VP>(rec + kv_value_offset(FMT, NB), lane, v);
    }
    if constexpr (kMx) {   // scales and tops: two token pairs a lane t, lanes g = 0 and 1 one each
        uint32_t odd[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) odd[i] = least[i] + kKvNear < top[i] ? 1u : 0u;
        if (__any_sync(0xffffffffu, max(max(top[0], top[1]), max(top[2], top[3])) == 255u)) {   // a block stored as NaN
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (top[i] != 255u) continue;
                odd[i] = 1u;
                top[i] = 1u;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint32_t e = scales[i][b / 4] >> (8 * (b & 3)) & 0xffu;
                    if (e != 255u) top[i] = max(top[i], e);
                }
            }
        }
        if (g < 2) {
            const bool second = g == 1;
            uint32_t sa[2], sb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) sa[i] = second ? scales[2][i] : scales[0][i], sb[i] = second ? scales[3][i] : scales[1][i];
            const bool ma = second ? vmine[2] : vmine[0], mb = second ? vmine[3] : vmine[1];
            const uint32_t word = (second ? top[2] : top[0]) | (second ? top[3] : top[1]) << 8 | (second ? odd[2] : odd[0]) << 16 |
                                  (second ? odd[3] : odd[1]) << 24;
            uint8_t* sp = rec + kv_value_scale_offset(FMT, NB) + (t + 4 * g) * 2 * NS;
            uint8_t* tp = rec + kv_value_top_offset(FMT, NB) + 4 * (t + 4 * g);
            if (ma && mb) {
                uint32_t out[(NB + 1) / 2];
#pragma unroll
                for (int i = 0; i < (NB + 1) / 2; ++i)   // bytes (a, b) of blocks 2i and 2i + 1
                    out[i] = __byte_perm(sa[i / 2], sb[i / 2], i & 1 ? 0x7362 : 0x5140);
                if constexpr (NB == 1) *reinterpret_cast<uint16_t*>(sp) = (uint16_t)out[0];
                else {
#pragma unroll
                    for (int i = 0; i < (NB + 1) / 2; ++i) *reinterpret_cast<uint32_t*>(sp + 4 * i) = out[i];
                }
                *reinterpret_cast<uint32_t*>(tp) = word;
            } else if (ma || mb) {
                const int at = ma ? 0 : 1;
#pragma unroll
                for (int b = 0; b < NB; ++b) sp[2 * b + at] = (uint8_t)((ma ? sa[b / 4] : sb[b / 4]) >> (8 * (b & 3)));
                tp[at] = (uint8_t)(word >> (8 * at));
                tp[2 + at] = (uint8_t)(word >> (16 + 8 * at));
            }
        }
    }
}

// ---------------------------------------------------------------- read
template <int TYPE, int N>
__device__ __forceinline__ void store_out(uint8_t* p, int vec, const float (&x)[N]) {
    constexpr int kWords = TYPE == kTypeF32 ? N : N / 2;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        if constexpr (TYPE == kTypeF32) w[2 * i] = __float_as_uint(x[2 * i]), w[2 * i + 1] = __float_as_uint(x[2 * i + 1]);
        else w[i] = TYPE == kTypeF16 ? f16x2_of(x[2 * i], x[2 * i + 1]) : bf16x2_of(x[2 * i], x[2 * i + 1]);
    }
    if (vec) {
        if constexpr (kWords == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else if constexpr (kWords == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if (vec > 1) st_global_v8(p, w);
        else {
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            *(reinterpret_cast<uint4*>(p) + 1) = make_uint4(w[4], w[5], w[6], w[7]);
        }
    } else {
        uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < kWords; ++i) h[2 * i] = (uint16_t)w[i], h[2 * i + 1] = (uint16_t)(w[i] >> 16);
    }
}

template <int FMT, int NB, int TYPE>
__global__ void __launch_bounds__(kKvIoWarps * 32)
    kv_read_kernel(KvPool pool, KvSeqs seqs, KvRows key, KvRows value, int64_t tokens, int64_t units, uint64_t* errors) {
    constexpr bool kMx = FMT >= kKvMx8;
    constexpr int KP = kv_key_piece(FMT), VP = kv_value_piece(FMT), NS = kv_scale_stride(NB), ES = TYPE == kTypeF32 ? 4 : 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t w = (int64_t)blockIdx.x * kKvIoWarps + (threadIdx.x >> 5);
    const int64_t u = w / pool.heads;
    if (u >= units) {   // (all warps of the last block)
        if (seqs.cu != nullptr && blockIdx.x == gridDim.x - 1) kv_check_offsets(seqs, tokens, errors);
        return;
    }
    const int h = (int)(w - u * pool.heads);
    const KvUnit un = kv_unit(seqs, tokens, u, lane, errors);
    if (!un.ok) return;
    const uint8_t* rec = kv_record(pool, seqs, un.b, un.rec, h);
    if (rec == nullptr) {
        if (lane == 0) kv_report(errors, kStatusBadPage);
        return;
    }
    const int base = un.rec * kKvRecord;
    // all loads first
    constexpr int kKeyWords = kMx ? NB * KP / 4 : NB * 8;
    uint32_t k0[kKeyWords], k1[kMx ? NB * KP / 4 : 1], v[NB * VP / 4], e0[(NB + 3) / 4], e1[(NB + 3) / 4], f0[(NB + 1) / 2], f1[(NB + 1) / 2];
    if constexpr (kMx) {
        load_lane<NB * KP>(rec, lane, k0);
        load_lane<NB * KP>(rec + 32 * NB * KP, lane, k1);
        load_scales<NB>(rec + kv_key_scale_offset(FMT, NB) + g * NS, e0);
        load_scales<NB>(rec + kv_key_scale_offset(FMT, NB) + (g + 8) * NS, e1);
        load_pair_scales<NB>(rec + kv_value_scale_offset(FMT, NB) + t * 2 * NS, f0);
        load_pair_scales<NB>(rec + kv_value_scale_offset(FMT, NB) + (t + 4) * 2 * NS, f1);
    } else {
        load_lane<NB * 32>(rec, lane, k0);
    }
    load_lane<NB * VP>(rec + kv_value_offset(FMT, NB), lane, v);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int pos = base + 8 * j + g;
        if (pos < un.lo || pos >= un.hi) continue;
        uint8_t* p = static_cast<uint8_t*>(key.p) + ((un.row0 + pos) * key.token_stride + (int64_t)h * key.head_stride + 8 * t) * ES;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t c[4];
            if constexpr (!kMx) {
                c[0] = k0[8 * b + j], c[1] = k0[8 * b + 2 + j], c[2] = k0[8 * b + 4 + j], c[3] = k0[8 * b + 6 + j];
            } else if constexpr (FMT == kKvMx8) {
                f16_of_e4m3x4(j ? k1[2 * b] : k0[2 * b], c[0], c[1]);
                f16_of_e4m3x4(j ? k1[2 * b + 1] : k0[2 * b + 1], c[2], c[3]);
            } else {
                f16_of_e2m1x8(j ? k1[b] : k0[b], c[0], c[1], c[2], c[3]);
            }
            const float s = kMx ? kv_scale_value((j ? e1[b / 4] : e0[b / 4]) >> (8 * (b & 3)) & 0xffu) : 1.f;
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = FMT == kKvBf16 ? bf16x2_floats(c[i]) : f16x2_floats(c[i]);
                x[2 * i] = kMx ? f.x * s : f.x;
                x[2 * i + 1] = kMx ? f.y * s : f.y;
            }
            store_out<TYPE, 8>(p + 32 * b * ES, key.vec, x);
        }
    }
    bool mine[4];
    uint8_t* p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = base + 2 * t + (i & 1) + 8 * (i >> 1);
        mine[i] = pos >= un.lo && pos < un.hi;
        p[i] = static_cast<uint8_t*>(value.p) + ((un.row0 + pos) * value.token_stride + (int64_t)h * value.head_stride + 4 * g) * ES;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        uint32_t c[8];   // [element][token pair]
        if constexpr (!kMx) {
#pragma unroll
            for (int e = 0; e < 4; ++e) c[2 * e] = v[8 * b + 4 * (e >> 1) + (e & 1)], c[2 * e + 1] = v[8 * b + 4 * (e >> 1) + 2 + (e & 1)];
        } else if constexpr (FMT == kKvMx8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f16_of_e4m3x4(v[4 * b + e], c[2 * e], c[2 * e + 1]);
        } else {
            f16_of_e2m1x8(v[2 * b], c[0], c[1], c[2], c[3]);
            f16_of_e2m1x8(v[2 * b + 1], c[4], c[5], c[6], c[7]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!mine[i]) continue;
            const float s = kMx ? kv_scale_value(((i >> 1) ? f1[b / 2] : f0[b / 2]) >> (16 * (b & 1) + 8 * (i & 1)) & 0xffu) : 1.f;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = FMT == kKvBf16 ? bf16x2_floats(c[2 * e + (i >> 1)]) : f16x2_floats(c[2 * e + (i >> 1)]);
                const float y = (i & 1) ? f.y : f.x;
                x[e] = kMx ? y * s : y;
            }
            store_out<TYPE, 4>(p[i] + 32 * b * ES, value.vec, x);
        }
    }
}

// ---------------------------------------------------------------- launches
template <bool READ, int FMT, int NB, int TYPE>
void kv_io_launch(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int64_t tokens, uint64_t* errors,
                  cudaStream_t stream) {
    const int64_t units = kv_units(seqs.cu != nullptr, tokens, seqs.batch);
    const unsigned blocks = (unsigned)((units * pool.heads + kKvIoWarps - 1) / kKvIoWarps) + (seqs.cu != nullptr ? 1u : 0u);   // (kv_check_offsets)
    if constexpr (READ) kv_read_kernel<FMT, NB, TYPE><<<blocks, kKvIoWarps * 32, 0, stream>>>(pool, seqs, key, value, tokens, units, errors);
    else kv_append_kernel<FMT, NB, TYPE><<<blocks, kKvIoWarps * 32, 0, stream>>>(pool, seqs, key, value, tokens, units, errors);
}
template <bool READ, int FMT, int NB>
void kv_io_type(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                uint64_t* errors, cudaStream_t stream) {
    switch (type) {
        case kTypeF32: return kv_io_launch<READ, FMT, NB, kTypeF32>(pool, seqs, key, value, tokens, errors, stream);
        case kTypeF16: return kv_io_launch<READ, FMT, NB, kTypeF16>(pool, seqs, key, value, tokens, errors, stream);
        default: return kv_io_launch<READ, FMT, NB, kTypeBf16>(pool, seqs, key, value, tokens, errors, stream);
    }
}
template <bool READ, int FMT>
void kv_io_format(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                  uint64_t* errors, cudaStream_t stream) {
    switch (pool.blocks) {
        case 1: return kv_io_type<READ, FMT, 1>(pool, seqs, key, value, type, tokens, errors, stream);
        case 2: return kv_io_type<READ, FMT, 2>(pool, seqs, key, value, type, tokens, errors, stream);
        case 3: return kv_io_type<READ, FMT, 3>(pool, seqs, key, value, type, tokens, errors, stream);
        case 4: return kv_io_type<READ, FMT, 4>(pool, seqs, key, value, type, tokens, errors, stream);
        case 6: return kv_io_type<READ, FMT, 6>(pool, seqs, key, value, type, tokens, errors, stream);
        default: return kv_io_type<READ, FMT, 8>(pool, seqs, key, value, type, tokens, errors, stream);
    }
}

// Loads the kernels of a cache (their first launch may be inside a stream capture, which loading does not get along with).
template <int FMT, int NB>
cudaError_t kv_io_blocks_init() {
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, kv_append_kernel<FMT, NB, kTypeF32>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, kv_append_kernel<FMT, NB, kTypeF16>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, kv_append_kernel<FMT, NB, kTypeBf16>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, kv_read_kernel<FMT, NB, kTypeF32>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, kv_read_kernel<FMT, NB, kTypeF16>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, kv_read_kernel<FMT, NB, kTypeBf16>);
    return e;
}
template <int FMT>
cudaError_t kv_io_format_init(int blocks) {
    switch (blocks) {
        case 1: return kv_io_blocks_init<FMT, 1>();
        case 2: return kv_io_blocks_init<FMT, 2>();
        case 3: return kv_io_blocks_init<FMT, 3>();
        case 4: return kv_io_blocks_init<FMT, 4>();
        case 6: return kv_io_blocks_init<FMT, 6>();
        default: return kv_io_blocks_init<FMT, 8>();
    }
}

#define EOSB_KV_IO(name)                                                                                                   \
    void kv_append_##name(const KvPool&, const KvSeqs&, const KvRows&, const KvRows&, int, int64_t, uint64_t*, cudaStream_t);   \
    void kv_read_##name(const KvPool&, const KvSeqs&, const KvRows&, const KvRows&, int, int64_t, uint64_t*, cudaStream_t);     \
    cudaError_t kv_io_##name##_init(int blocks);
EOSB_KV_IO(f16)
EOSB_KV_IO(bf16)
EOSB_KV_IO(mx8)
EOSB_KV_IO(mx4)
#undef EOSB_KV_IO

}  // namespace eosb

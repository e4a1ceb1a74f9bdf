// Paged key-value cache: quantising tokens as they are written, and reading them back.
//
// Formats.  f16 / bf16 hold each element rounded to nearest.  mx8 (e4m3) and mx4 (e2m1) hold, for every 32 consecutive
// elements of a head's vector, one scale 2^e with the smallest e >= -126 for which max|x| <= top 2^e (top = 448 or 6,
// the type's largest value, so nothing saturates) and the codes x / 2^e rounded to nearest, ties to even.  The scale is
// a power of two: the division is exact, every code has one right answer, and a code times its scale is exact in fp32.
// A block that holds an infinity or a NaN is stored as NaN (scale byte 255).
//
// One warp per (record, head): it owns all 16 tokens of the record that the call writes, so a record that is completed
// by several calls needs no atomics and neighbouring 4-bit codes of two tokens are merged by a plain read-modify-write.
#include "kv_cache.cuh"

#include "kv_attend.cuh"
#include "kv_dev.cuh"

namespace eosb {

namespace {

constexpr int kKvWarps = 8;

// The sequence and record that work unit u of a call stands for.  Sequence b starts at unit cu[b] / 16 + 2 b: n tokens
// that start anywhere in a record touch at most floor((n + 30) / 16) records, and the gap to sequence b + 1 is at least
// that.  Warp-wide search, 32 probes a step; lanes agree on the result.
struct KvUnit {
    int b, rec;       // sequence, record index within the sequence
    int lo, hi;       // positions [lo, hi) of the record that the call covers
    int64_t row0;     // row of position 0 of the sequence (may be negative: rows are row0 + position)
    bool ok;
};
__device__ __forceinline__ KvUnit kv_unit(const KvSeqs& s, int64_t tokens, int64_t u, int lane, int* status) {
    KvUnit r;
    r.ok = false;
    int64_t row, n, first = 0;
    if (s.cu == nullptr) {
        r.b = (int)u, row = u, n = 1;
    } else {
        int lo = 0, hi = s.batch;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) >> 5;
            const int probe = lo + lane * step;
            const bool below = lane == 0 || (probe < hi && (int64_t)(__ldg(s.cu + probe) >> 4) + 2 * (int64_t)probe <= u);
            const int top = 31 - __clz(__ballot_sync(0xffffffffu, below));
            lo += top * step;
            hi = min(hi, lo + step);
        }
        r.b = lo;
        row = __ldg(s.cu + lo);
        n = (int64_t)__ldg(s.cu + lo + 1) - row;
        first = u - ((int64_t)(row >> 4) + 2 * (int64_t)lo);
    }
    if (n == 0) return r;
    const int64_t start = __ldg(s.starts + r.b);
    if (n < 0 || row < 0 || row + n > tokens || start < 0 || start + n > 0x7fffffffLL) {
        if (lane == 0) atomicExch(status, kStatusBadSequence);
        return r;
    }
    const int64_t rec = (start >> 4) + first;
    if (first < 0 || rec * kKvRecord >= start + n) return r;
    r.rec = (int)rec;
    r.lo = (int)max(start, rec * kKvRecord);
    r.hi = (int)min(start + n, (rec + 1) * kKvRecord);
    r.row0 = row - start;
    r.ok = true;
    return r;
}

// scale byte of a block with the largest magnitude amax (its fp32 bits)
template <int FMT>
__device__ __forceinline__ uint32_t kv_scale_byte(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23, m = amax_bits & 0x7fffffu;
    if (e == 255u) return 255u;
    const int byte = FMT == kKvMx8 ? (int)e - 8 + (m > 0x600000u) : (int)e - 2 + (m > 0x400000u);   // 448 = 1.75 2^8, 6 = 1.5 2^2
    return (uint32_t)max(byte, 1);
}
// 2^-e of a scale byte; 0 for a block stored as NaN, whose codes are all zero
__device__ __forceinline__ float kv_inverse_scale(uint32_t byte) { return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float kv_scaled(float x, uint32_t byte, float inv) { return byte == 255u ? 0.f : x * inv; }

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int FMT>
__global__ void __launch_bounds__(kKvWarps * 32)
    kv_append_kernel(KvPool pool, KvSeqs seqs, KvRows key, KvRows value, int type, int64_t tokens, int64_t units, int* status) {
    constexpr bool kMx = FMT >= kKvMx8;
    constexpr int KP = kv_key_piece(FMT), VP = kv_value_piece(FMT);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t w = (int64_t)blockIdx.x * kKvWarps + (threadIdx.x >> 5);
    const int64_t u = w / pool.heads;
    if (u >= units) return;
    const int h = (int)(w - u * pool.heads);
    const KvUnit un = kv_unit(seqs, tokens, u, lane, status);
    if (!un.ok) return;
    uint8_t* rec = kv_record(pool, seqs, un.b, un.rec, h);
    if (rec == nullptr) {
        if (lane == 0) atomicExch(status, kStatusBadPage);
        return;
    }
    const int nb = pool.blocks, ns = kv_scale_stride(nb), base = un.rec * kKvRecord;
    // ---- keys: lane (g, t) owns 8 elements of token 8 j + g in every block
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int pos = base + 8 * j + g;
        const bool mine = pos >= un.lo && pos < un.hi;
        if (!__any_sync(0xffffffffu, mine)) continue;
        const int64_t at = (un.row0 + pos) * key.token_stride + (int64_t)h * key.head_stride + 8 * t;
        uint8_t* codes = rec + (kMx ? j * 32 * nb * KP : 0);
#pragma unroll 4
        for (int b = 0; b < nb; ++b) {
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (mine) load_row<8>(key.p, at + 32 * b, type, key.vec, x);
            uint8_t* dst = codes + kv_lane_offset(nb * KP, lane, b * KP);
            if constexpr (!kMx) {
                // words 0, 1 and 2, 3 of the token go to words j, j + 2 of the block's first and second 16 bytes
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t v = FMT == kKvF16 ? f16x2_of(x[2 * i], x[2 * i + 1]) : bf16x2_of(x[2 * i], x[2 * i + 1]);
                    if (mine) *reinterpret_cast<uint32_t*>(codes + kv_lane_offset(2 * nb * KP, lane, 32 * b + 16 * (i >> 1) + 8 * (i & 1) + 4 * j)) = v;
                }
            } else {
                uint32_t m = 0;   // as integers: an infinity or a NaN stays the largest
#pragma unroll
                for (int i = 0; i < 8; ++i) m = max(m, abs_bits(x[i]));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const uint32_t byte = kv_scale_byte<FMT>(m);
                const float inv = kv_inverse_scale(byte);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = kv_scaled(x[i], byte, inv);
                if (mine) {
                    if constexpr (FMT == kKvMx8) {
                        uint2 v;
                        v.x = e4m3x2_of(x[0], x[1]) | (e4m3x2_of(x[2], x[3]) << 16);
                        v.y = e4m3x2_of(x[4], x[5]) | (e4m3x2_of(x[6], x[7]) << 16);
                        *reinterpret_cast<uint2*>(dst) = v;
                    } else {
                        *reinterpret_cast<uint32_t*>(dst) = e2m1x2_of(x[0], x[1]) | (e2m1x2_of(x[2], x[3]) << 8) |
                                                            (e2m1x2_of(x[4], x[5]) << 16) | (e2m1x2_of(x[6], x[7]) << 24);
                    }
                    if (t == 0) rec[kv_key_scale_offset(FMT, nb) + (8 * j + g) * ns + b] = (uint8_t)byte;
                }
            }
        }
    }
    // ---- values: lane (g, t) owns elements 4 g .. + 3 of every block for the tokens 2t, 2t+1, 2t+8, 2t+9
    bool mine[4];
    int64_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = base + 2 * t + (i & 1) + 8 * (i >> 1);
        mine[i] = pos >= un.lo && pos < un.hi;
        at[i] = (un.row0 + pos) * value.token_stride + (int64_t)h * value.head_stride + 4 * g;
    }
    const bool any = mine[0] || mine[1] || mine[2] || mine[3], all = mine[0] && mine[1] && mine[2] && mine[3];
    uint8_t* codes = rec + kv_value_offset(FMT, nb);
    uint64_t scales[4] = {0, 0, 0, 0};   // of each token: the blocks' scale bytes, 0 for a block of zeros
#pragma unroll 2
    for (int b = 0; b < nb; ++b) {
        float x[4][4];   // [token][element]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
            if (mine[i]) load_row<4>(value.p, at[i] + 32 * b, type, value.vec, x[i]);
        }
        uint32_t v[VP / 4], keep[VP / 4];
        if constexpr (!kMx) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a = x[2 * i][e], c = x[2 * i + 1][e];
                    const int at_word = 4 * (e >> 1) + 2 * i + (e & 1);
                    v[at_word] = FMT == kKvF16 ? f16x2_of(a, c) : bf16x2_of(a, c);
                    keep[at_word] = (mine[2 * i] ? 0u : 0x0000ffffu) | (mine[2 * i + 1] ? 0u : 0xffff0000u);
                }
        } else {
            uint32_t byte[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t m = max(max(abs_bits(x[i][0]), abs_bits(x[i][1])), max(abs_bits(x[i][2]), abs_bits(x[i][3])));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
                byte[i] = kv_scale_byte<FMT>(m);
                const float inv = kv_inverse_scale(byte[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = kv_scaled(x[i][e], byte[i], inv);
                scales[i] |= (uint64_t)(m == 0 ? 0u : byte[i]) << (8 * b);
            }
            if constexpr (FMT == kKvMx8) {
                const uint32_t k = (mine[0] ? 0u : 0xffu) | (mine[1] ? 0u : 0xff00u) | (mine[2] ? 0u : 0xff0000u) |
                                   (mine[3] ? 0u : 0xff000000u);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = e4m3x2_of(x[0][e], x[1][e]) | (e4m3x2_of(x[2][e], x[3][e]) << 16);
                    keep[e] = k;
                }
            } else {
                const uint32_t k = (mine[0] ? 0u : 0xfu) | (mine[1] ? 0u : 0xf0u) | (mine[2] ? 0u : 0xf00u) | (mine[3] ? 0u : 0xf000u);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    v[e] = e2m1x2_of(x[0][2 * e], x[1][2 * e]) | (e2m1x2_of(x[2][2 * e], x[3][2 * e]) << 8) |
                           (e2m1x2_of(x[0][2 * e + 1], x[1][2 * e + 1]) << 16) |
                           (e2m1x2_of(x[2][2 * e + 1], x[3][2 * e + 1]) << 24);
                    keep[e] = k | (k << 16);
                }
            }
        }
        if (!any) continue;
        // pieces of 16 bytes (8 for mx4); tokens of the record that this call does not write keep their bits
        if constexpr (VP == 8) {
            uint2* dst = reinterpret_cast<uint2*>(codes + kv_lane_offset(nb * VP, lane, b * VP));
            if (!all) {
                const uint2 old = *dst;
                v[0] = (v[0] & ~keep[0]) | (old.x & keep[0]);
                v[1] = (v[1] & ~keep[1]) | (old.y & keep[1]);
            }
            *dst = make_uint2(v[0], v[1]);
        } else {
#pragma unroll
            for (int p = 0; p < VP / 16; ++p) {
                uint4* dst = reinterpret_cast<uint4*>(codes + kv_lane_offset(nb * VP, lane, b * VP + 16 * p));
                uint32_t* q = v + 4 * p;
                const uint32_t* k = keep + 4 * p;
                if (!all) {
                    const uint4 old = *dst;
                    q[0] = (q[0] & ~k[0]) | (old.x & k[0]);
                    q[1] = (q[1] & ~k[1]) | (old.y & k[1]);
                    q[2] = (q[2] & ~k[2]) | (old.z & k[2]);
                    q[3] = (q[3] & ~k[3]) | (old.w & k[3]);
                }
                *dst = make_uint4(q[0], q[1], q[2], q[3]);
            }
        }
    }
    if constexpr (kMx) {   // lane (g, t) stores the scales of block g; the tops by the lanes of block 0
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t top = 1, odd = 0;
            for (int b = 0; b < nb; ++b) {
                const uint32_t e = (uint32_t)(scales[i] >> (8 * b)) & 0xffu;
                if (e == 255u) odd = 1;
                else top = max(top, e);
            }
            for (int b = 0; b < nb; ++b) {
                const uint32_t e = (uint32_t)(scales[i] >> (8 * b)) & 0xffu;
                if (e != 0u && e + kKvNear < top) odd = 1;
            }
            if (!mine[i]) continue;
            const int pair = t + 4 * (i >> 1);
            if (g < nb) {
                const uint32_t e = (uint32_t)(scales[i] >> (8 * g)) & 0xffu;
                rec[kv_value_scale_offset(FMT, nb) + (pair * ns + g) * 2 + (i & 1)] = (uint8_t)(e == 0u ? top : e);
            }
            if (g == 0) {
                uint8_t* tops = rec + kv_value_top_offset(FMT, nb) + 4 * pair + (i & 1);
                tops[0] = (uint8_t)top;
                tops[2] = (uint8_t)odd;
            }
        }
    }
}

template <int FMT>
__global__ void __launch_bounds__(kKvWarps * 32)
    kv_read_kernel(KvPool pool, KvSeqs seqs, KvRows key, KvRows value, int type, int64_t tokens, int64_t units, int* status) {
    constexpr bool kMx = FMT >= kKvMx8;
    constexpr int KP = kv_key_piece(FMT), VP = kv_value_piece(FMT);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t w = (int64_t)blockIdx.x * kKvWarps + (threadIdx.x >> 5);
    const int64_t u = w / pool.heads;
    if (u >= units) return;
    const int h = (int)(w - u * pool.heads);
    const KvUnit un = kv_unit(seqs, tokens, u, lane, status);
    if (!un.ok) return;
    const uint8_t* rec = kv_record(pool, seqs, un.b, un.rec, h);
    if (rec == nullptr) {
        if (lane == 0) atomicExch(status, kStatusBadPage);
        return;
    }
    const int nb = pool.blocks, ns = kv_scale_stride(nb), base = un.rec * kKvRecord;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int pos = base + 8 * j + g;
        if (pos < un.lo || pos >= un.hi) continue;
        const int64_t at = (un.row0 + pos) * key.token_stride + (int64_t)h * key.head_stride + 8 * t;
        const uint8_t* codes = rec + (kMx ? j * 32 * nb * KP : 0);
#pragma unroll 4
        for (int b = 0; b < nb; ++b) {
            const uint8_t* src = codes + kv_lane_offset(nb * KP, lane, b * KP);
            float x[8];
            uint32_t c[4];
            if constexpr (!kMx) {
                const uint4 v = *reinterpret_cast<const uint4*>(codes + kv_lane_offset(2 * nb * KP, lane, 32 * b));
                const uint4 y = *reinterpret_cast<const uint4*>(codes + kv_lane_offset(2 * nb * KP, lane, 32 * b + 16));
                c[0] = j ? v.y : v.x, c[1] = j ? v.w : v.z, c[2] = j ? y.y : y.x, c[3] = j ? y.w : y.z;
            } else if constexpr (FMT == kKvMx8) {
                const uint2 v = *reinterpret_cast<const uint2*>(src);
                f16_of_e4m3x4(v.x, c[0], c[1]);
                f16_of_e4m3x4(v.y, c[2], c[3]);
            } else {
                f16_of_e2m1x8(*reinterpret_cast<const uint32_t*>(src), c[0], c[1], c[2], c[3]);
            }
            const float s = kMx ? kv_scale_value(rec[kv_key_scale_offset(FMT, nb) + (8 * j + g) * ns + b]) : 1.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = FMT == kKvBf16 ? bf16x2_floats(c[i]) : f16x2_floats(c[i]);
                x[2 * i] = kMx ? f.x * s : f.x;
                x[2 * i + 1] = kMx ? f.y * s : f.y;
            }
            store_row<8>(key.p, at + 32 * b, type, key.vec, x);
        }
    }
    bool mine[4];
    int64_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = base + 2 * t + (i & 1) + 8 * (i >> 1);
        mine[i] = pos >= un.lo && pos < un.hi;
        at[i] = (un.row0 + pos) * value.token_stride + (int64_t)h * value.head_stride + 4 * g;
    }
    if (!(mine[0] || mine[1] || mine[2] || mine[3])) return;
    const uint8_t* codes = rec + kv_value_offset(FMT, nb);
#pragma unroll 2
    for (int b = 0; b < nb; ++b) {
        uint32_t c[8];   // [element][token pair]
        if constexpr (!kMx) {
            const uint4 a = *reinterpret_cast<const uint4*>(codes + kv_lane_offset(nb * VP, lane, b * VP));
            const uint4 d = *reinterpret_cast<const uint4*>(codes + kv_lane_offset(nb * VP, lane, b * VP + 16));
            c[0] = a.x, c[2] = a.y, c[1] = a.z, c[3] = a.w, c[4] = d.x, c[6] = d.y, c[5] = d.z, c[7] = d.w;
        } else if constexpr (FMT == kKvMx8) {
            const uint4 a = *reinterpret_cast<const uint4*>(codes + kv_lane_offset(nb * VP, lane, b * VP));
            f16_of_e4m3x4(a.x, c[0], c[1]);
            f16_of_e4m3x4(a.y, c[2], c[3]);
            f16_of_e4m3x4(a.z, c[4], c[5]);
            f16_of_e4m3x4(a.w, c[6], c[7]);
        } else {
            const uint2 a = *reinterpret_cast<const uint2*>(codes + kv_lane_offset(nb * VP, lane, b * VP));
            f16_of_e2m1x8(a.x, c[0], c[1], c[2], c[3]);
            f16_of_e2m1x8(a.y, c[4], c[5], c[6], c[7]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!mine[i]) continue;
            const float s = kMx ? kv_scale_value(rec[kv_value_scale_offset(FMT, nb) + ((t + 4 * (i >> 1)) * ns + b) * 2 + (i & 1)]) : 1.f;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = FMT == kKvBf16 ? bf16x2_floats(c[2 * e + (i >> 1)]) : f16x2_floats(c[2 * e + (i >> 1)]);
                const float y = (i & 1) ? f.y : f.x;
                x[e] = kMx ? y * s : y;
            }
            store_row<4>(value.p, at[i] + 32 * b, type, value.vec, x);
        }
    }
}

// Work units of a call: see kv_unit.  The rows behind the last sequence belong to no unit.
int64_t kv_units(const KvSeqs& s, int64_t tokens) { return s.cu == nullptr ? tokens : (tokens >> 4) + 2 * (int64_t)s.batch; }

template <int FMT>
void launch_append(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                   int* status, cudaStream_t stream) {
    const int64_t units = kv_units(seqs, tokens), blocks = (units * pool.heads + kKvWarps - 1) / kKvWarps;
    kv_append_kernel<FMT><<<(unsigned)blocks, kKvWarps * 32, 0, stream>>>(pool, seqs, key, value, type, tokens, units, status);
}
template <int FMT>
void launch_read(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                 int* status, cudaStream_t stream) {
    const int64_t units = kv_units(seqs, tokens), blocks = (units * pool.heads + kKvWarps - 1) / kKvWarps;
    kv_read_kernel<FMT><<<(unsigned)blocks, kKvWarps * 32, 0, stream>>>(pool, seqs, key, value, type, tokens, units, status);
}

}  // namespace

void launch_kv_append(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type,
                      int64_t tokens, int* status, cudaStream_t stream) {
    switch (pool.format) {
        case kKvF16: return launch_append<kKvF16>(pool, seqs, key, value, type, tokens, status, stream);
        case kKvBf16: return launch_append<kKvBf16>(pool, seqs, key, value, type, tokens, status, stream);
        case kKvMx8: return launch_append<kKvMx8>(pool, seqs, key, value, type, tokens, status, stream);
        default: return launch_append<kKvMx4>(pool, seqs, key, value, type, tokens, status, stream);
    }
}

void launch_kv_read(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                    int* status, cudaStream_t stream) {
    switch (pool.format) {
        case kKvF16: return launch_read<kKvF16>(pool, seqs, key, value, type, tokens, status, stream);
        case kKvBf16: return launch_read<kKvBf16>(pool, seqs, key, value, type, tokens, status, stream);
        case kKvMx8: return launch_read<kKvMx8>(pool, seqs, key, value, type, tokens, status, stream);
        default: return launch_read<kKvMx4>(pool, seqs, key, value, type, tokens, status, stream);
    }
}

int launch_kv_attend(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, int* status,
                     cudaStream_t stream) {
    switch (pool.format) {
        case kKvF16: return kv_attend_f16(pool, seqs, a, work, status, stream);
        case kKvBf16: return kv_attend_bf16(pool, seqs, a, work, status, stream);
        case kKvMx8: return kv_attend_mx8(pool, seqs, a, work, status, stream);
        default: return kv_attend_mx4(pool, seqs, a, work, status, stream);
    }
}

cudaError_t kv_attend_init(int format, int blocks) {
    switch (format) {
        case kKvF16: return kv_attend_f16_init(blocks);
        case kKvBf16: return kv_attend_bf16_init(blocks);
        case kKvMx8: return kv_attend_mx8_init(blocks);
        default: return kv_attend_mx4_init(blocks);
    }
}

}  // namespace eosb

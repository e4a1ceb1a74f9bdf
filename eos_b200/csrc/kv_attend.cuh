// One new token a sequence attends over its cached keys and values: the kernel template (one instance per format, head
// size and row tiles; kv_attend_*.cu compile them).
//
//     out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = scale log2(e) q . k_j,   one pass with a running maximum m
//
// A warp takes one or two records (16 tokens of one key head each) at a time with mma.sync m16n8k16, and both products are
// formed transposed: S^T = K q^T with the tokens as the 16 rows and 8 query heads of the key head as the columns, then
// O^T += V^T P^T with 16 elements of the values as the rows.  The few query heads that share a key head fill the narrow
// side of the instruction, keys and values its wide one, and the accumulators take half of what heads as rows would.
// (tcgen05 wants 128 rows and its operands in shared memory or TMEM.  Its 16-bit kinds would have the codes converted and written
// back there first, and the weights once more; its block-scaled kinds take the codes as they are, but then query and weights have
// to be sums of several e4m3 numbers, and the value scales, one for 32 elements of a token, run along the wrong axis.  The 16-bit
// formats are at HBM's rate without it.)
//
// Every fp32 factor -- the weights, and a query that does not fit the operand type (fp32, or f16 over a bf16 cache) -- is
// the sum of two 16-bit operands, so the products carry 22 bits.  Over a bf16 cache, whose operands hold 8, it is the sum of
// three for fp32 queries and results, 24 bits, and of two, 16, for 16-bit ones, which keep 11 at most (an f16 query is exact in
// two; its lse stays that of 32 bits, for it is taken before the split; weights of three operands there took 32.2 us instead of
// 30.5 for one key head of 256 under a window, and left the error as it is to three digits).  The cached value is never split: it is
// exact in its operand type.  (Weights in one f16 operand where the result is bf16 saved 7 us of 90 over mx4 and 1 of 64 over mx8, and moved
// one result in twenty to a neighbouring bf16 number.)
//
// The maxima are integers, and lag: m is set 7 below the largest score and moves only when a score passes m + 15, so most
// records do no rescaling and no shuffles, and weights use f16's range from both ends: they stay below 2^15, and what
// f16 cannot hold (2^-25) is 2^-31 of the row's largest weight.  A weight and its value's scale are multiplied before the
// split: w = 2^(x - m + e - d) with e the largest scale exponent of the token's blocks and d a second lagging maximum,
// relative to the first, so that the bound holds whatever the scales; the blocks' own exponents, relative to e, are f16 factors of
// the split weights (four multiplications a block where scaling the codes takes eight), so the codes enter the mma as they are.
//
// What bounds it (GPU time of a call, heads of 128 unless said; floor: the records' bytes at 6540 GB/s).  f16, 32 sequences of
// 8192 tokens, 8 key heads with 8 query heads each: 174 to 179 us, 6.0 to 6.2 TB/s, floor 164: HBM.  mx8, one sequence of
// 131071 tokens, 8 key heads with 4 query heads each: 55 us, 5.0 TB/s, floor 42: the loop runs at HBM's rate, and the rest is
// a call's constant part -- launch and exit 2.5 us, lengths, page ids and the first records one after the other 4 us, joins
// 4 to 5 us, of which 3 to 4 are those across CTAs.  mx4, 16 sequences of 4000 to 32768 tokens, 8 key heads with 8 query
// heads each: 90 us, 3.4 TB/s, floor 47: no one unit -- 425 instructions a warp and record, of which 173 run at half rate, fill 55 %
// of the issue slots and 38 % of that pipe; the rest is the latency of dependent instructions that four warps a scheduler do not
// hide (wait 1.8, math pipe 0.8, barriers 0.7, shared memory 0.6 stalls an instruction), and 10 to 12 us of prologue and joins.  Spills are
// two loads in 425 instructions.  One short sequence: 8 us, launch and latencies.
#pragma once
#include <algorithm>

#include "kv_dev.cuh"
#include "kv_split.cuh"

namespace eosb {

// A value that the compiler takes for a new one each time: a condition on it inside a loop does not double the loop.  The
// code that runs once or seldom is most of the kernel, and comes from the L2 while the records do.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+r"(x));
    return x;
}

// The least fp32 number: no score is below it.  Finite, so that 2^(x - m) of a masked score is 0 and not NaN.  (A distance from it
// may be infinite: a first score above 0 less it, and the second maximum by which it moves.  Both are then taken anew.)
constexpr float kKvMaxInit = -3.402823466e38f;
constexpr float kKvHead = 7.f, kKvLag = 15.f;   // m = ceil(largest score) - 7; weights up to 2^15
constexpr int kKvQueryExp = 13;                  // query rows are scaled to a largest magnitude in [2^13, 2^14)

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&y);
}
template <bool kBf>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
    if constexpr (kBf)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// a pair of fp32 values as the sum of PARTS 16-bit pairs, the largest first
template <bool kBf, int PARTS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&part)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        part[i] = kBf ? bf16x2_of(a, b) : f16x2_of(a, b);
        const float2 f = kBf ? bf16x2_floats(part[i]) : f16x2_floats(part[i]);
        a -= f.x, b -= f.y;
    }
}

// transposes an 8 x 8 matrix of 16-bit values held by a warp (lane 4 g + t: row g, columns 2t and 2t+1)
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}

// byte i of a word as a float 2^(byte - 127); 255 becomes infinity, which times the zero codes of such a block is NaN
__device__ __forceinline__ float scale_at(uint32_t word, int i) { return __uint_as_float(__byte_perm(word, 0, 0x4440 | i) << 23); }

// RT: tiles of 8 query heads; HALVES: operands of the query (1: its type fits the operand type; 3: f32 over a bf16 cache).
template <int FMT, int NB, int RT, int HALVES>
struct KvWarp {
    static constexpr bool kMx = FMT >= kKvMx8, kBf = FMT == kKvBf16;
    static constexpr int KP = kv_key_piece(FMT), VP = kv_value_piece(FMT), D = 32 * NB;
    static constexpr int kParts = HALVES == 3 ? 3 : 2;           // operands of the weights
    static constexpr bool kWide = HALVES == (kBf ? 3 : 2);       // the query is fp32
    using Weights = uint32_t[RT][kParts][2];

    uint32_t q[RT][NB][4 * HALVES];   // head g of each tile, elements 32 b + 8 t .. + 7: the largest parts, then the next
    float2 qs[RT];                    // heads 2t and 2t + 1: factor of the raw sums, scale log2(e) 2^(query exponent), less ks
    float ks;                         // (mx formats) factor of the key scales, a power of two
    float2 nm[RT], nd[RT];            // heads 2t, 2t + 1: minus the lagging maxima of x; of x + e relative to those (mx formats)
    float l[RT][2];                   // this lane's part of the sum of weights
    float o[RT][NB][2][4];            // [block][i]: elements 32 b + 4 g + 2 i (0, 1) and + 2 i + 1 (2, 3) of heads 2t, 2t + 1

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int i = 0; i < 2; ++i) l[r][i] = 0.f;
            nm[r] = make_float2(-kKvMaxInit, -kKvMaxInit);
            nd[r] = make_float2(0.f, 0.f);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) o[r][b][i >> 2][i & 3] = 0.f;
        }
    }

    // Query rows [row0, row0 + 8 RT) of a unit, those from `rows` on are zero: first the raw loads, all of them on their way
    // at once and waited for in convert_query, ...
    __device__ __forceinline__ void load_query(const KvAttend& a, int64_t at, int row0, int rows, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const int vec = opaque(a.vec);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = row0 + 8 * r + g;
            const uint8_t* base = static_cast<const uint8_t*>(a.query) + (at + (int64_t)row * a.head_stride + 8 * t) * (kWide ? 4 : 2);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < (kWide ? 8 : 4); i += 4) {   // two 16-byte loads a block, or one
                    uint4 x = make_uint4(0u, 0u, 0u, 0u);
                    const uint8_t* from = base + b * (kWide ? 128 : 64) + 4 * i;
                    if (row < rows) {
                        if (vec) x = *reinterpret_cast<const uint4*>(from);
                        else x = load16_unaligned(from);
                    }
                    q[r][b][i] = x.x, q[r][b][i + 1] = x.y, q[r][b][i + 2] = x.z, q[r][b][i + 3] = x.w;
                }
        }
    }
    // ... then the operands.  f16: each row is divided by a power of two first, so that no magnitude leaves f16's range.  It is
    // multiplied back behind the sum -- over block-scaled keys, whose sum with it might leave fp32's range where the score does
    // not, as far as it is common to the rows and below 1, into the key scales (one packed product a block, 1 % over mx4).
    // One operand: the type is f16 or bf16 (over a bf16 cache bf16); more: f32 (over a bf16 cache two: f16).
    __device__ __forceinline__ void convert_query(const KvAttend& a, int lane) {
        const bool f16 = opaque(a.type) == kTypeF16;
        auto pair = [&](int r, int b, int i) {
            if constexpr (!kWide) {
                const uint32_t w = q[r][b][i];
                if constexpr (kBf) return HALVES == 1 ? bf16x2_floats(w) : f16x2_floats(w);
                const float2 x = f16x2_floats(w), y = bf16x2_floats(w);
                return make_float2(f16 ? x.x : y.x, f16 ? x.y : y.y);
            } else {
                return make_float2(__uint_as_float(q[r][b][2 * i]), __uint_as_float(q[r][b][2 * i + 1]));
            }
        };
        uint32_t e[RT], back = 127u + kKvQueryExp;   // exponents of the rows; what they are taken back relative to behind the sum
        if constexpr (!kBf) {
            uint32_t most = 0;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                uint32_t top = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 x = pair(r, b, i);
                        top = max(top, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
                    }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                e[r] = min(max(top >> 23, kKvQueryExp + 1u), 254u);
                most = max(most, e[r]);
            }
            if constexpr (kMx) {
                back = min(back, __reduce_max_sync(0xffffffffu, most));
                ks = __uint_as_float((back - kKvQueryExp) << 23);
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) split_row(r, lane, e[r], back, a.scale_log2, [&](int b, int i) { return pair(r, b, i); });
    }
    template <typename F>
    __device__ __forceinline__ void split_row(int r, int lane, uint32_t e, uint32_t back, float factor, F&& pair) {
        float inv = 1.f;
        if constexpr (!kBf) {
            inv = __uint_as_float((254u + kKvQueryExp - e) << 23);
            factor *= __uint_as_float((127u + e - back) << 23);   // (e and back are at least 14: an exponent of -126 or more)
        }
        // the factors of heads 2t and 2t + 1 are those of the lanes with g = 2t and 2t + 1
        qs[r].x = __shfl_sync(0xffffffffu, factor, 8 * (lane & 3));
        qs[r].y = __shfl_sync(0xffffffffu, factor, 8 * (lane & 3) + 4);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float2 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = pair(b, i);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t part[HALVES];
                split_pair<kBf>(x[i].x * inv, x[i].y * inv, part);
#pragma unroll
                for (int u = 0; u < HALVES; ++u) q[r][b][4 * u + i] = part[u];
            }
        }
    }

    __device__ __forceinline__ void scale_rows(int r, float2 f) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float* c = &o[r][b][i >> 2][i & 3];
                const float2 y = mul2(make_float2(c[0], c[1]), f);
                c[0] = y.x, c[1] = y.y;
            }
    }

    // Raw scores of a record's tokens g (0, 1) and g + 8 (2, 3) with heads 2t, 2t + 1.
    __device__ __forceinline__ void scores(const uint8_t* rec, float (&s)[RT][4], int lane) const {
        const int g = lane >> 2;
        if constexpr (!kMx) {
            uint32_t k[NB * 8];
            load_lane<NB * 32>(rec, lane, k);
            float c[RT][2][4];   // two sums: chains of dependent mma half as long
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i) c[r][i >> 2][i & 3] = 0.f;
#pragma unroll
            for (int h = HALVES - 1; h >= 0; --h)   // the smallest parts first: a sum is cut at its size in every step
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < RT; ++r)
                            mma_16x8x16<kBf>(c[r][i], k[8 * b + 4 * i], k[8 * b + 4 * i + 1], k[8 * b + 4 * i + 2], k[8 * b + 4 * i + 3],
                                             q[r][b][4 * h + 2 * i], q[r][b][4 * h + 2 * i + 1]);
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[r][i] = c[r][0][i] + c[r][1][i];
        } else {
            uint32_t k0[NB * KP / 4], k1[NB * KP / 4], e0[(NB + 3) / 4], e1[(NB + 3) / 4];
            load_lane<NB * KP>(rec, lane, k0);
            load_lane<NB * KP>(rec + 32 * NB * KP, lane, k1);
            load_scales<NB>(rec + kv_key_scale_offset(FMT, NB) + g * kv_scale_stride(NB), e0);
            load_scales<NB>(rec + kv_key_scale_offset(FMT, NB) + (g + 8) * kv_scale_stride(NB), e1);
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                uint32_t f[4], h[4];   // elements 8 t .. + 7 of tokens g and g + 8
                if constexpr (FMT == kKvMx8) {
                    f16_of_e4m3x4(k0[2 * b], f[0], f[1]);
                    f16_of_e4m3x4(k0[2 * b + 1], f[2], f[3]);
                    f16_of_e4m3x4(k1[2 * b], h[0], h[1]);
                    f16_of_e4m3x4(k1[2 * b + 1], h[2], h[3]);
                } else {
                    f16_of_e2m1x8(k0[b], f[0], f[1], f[2], f[3]);
                    f16_of_e2m1x8(k1[b], h[0], h[1], h[2], h[3]);
                }
                const float2 sk = mul2(make_float2(scale_at(e0[b / 4], b & 3), scale_at(e1[b / 4], b & 3)), make_float2(ks, ks));
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = HALVES - 1; u >= 0; --u) {
                        mma_16x8x16<false>(c, f[0], h[0], f[1], h[1], q[r][b][4 * u], q[r][b][4 * u + 1]);
                        mma_16x8x16<false>(c, f[2], h[2], f[3], h[3], q[r][b][4 * u + 2], q[r][b][4 * u + 3]);
                    }
                    s[r][0] = fmaf(c[0], sk.x, s[r][0]), s[r][1] = fmaf(c[1], sk.x, s[r][1]);
                    s[r][2] = fmaf(c[2], sk.y, s[r][2]), s[r][3] = fmaf(c[3], sk.y, s[r][3]);
                }
            }
        }
    }

    // A record's value scales: every block's exponent relative to the largest of its token, as f16 pairs of the tokens 2t,
    // 2t + 1 and 2t + 8, 2t + 9 (zero for tokens outside [lo, hi)).
    template <bool EDGE>
    __device__ __forceinline__ void value_scales(const uint8_t* rec, int lo, int hi, uint32_t (&rel)[2][NB], int lane) const {
        const int t = lane & 3;
        uint32_t tops[2], live[2] = {0xffffffffu, 0xffffffffu}, odd = 0;
        if constexpr (EDGE) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int tok = 2 * t + 8 * p;
                live[p] = kv_live_bytes(tok >= lo && tok < hi, tok + 1 >= lo && tok + 1 < hi);
            }
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            uint32_t w[(NB + 1) / 2];
            load_pair_scales<NB>(rec + kv_value_scale_offset(FMT, NB) + (t + 4 * p) * 2 * kv_scale_stride(NB), w);
            tops[p] = *reinterpret_cast<const uint32_t*>(rec + kv_value_top_offset(FMT, NB) + 4 * (t + 4 * p)) & live[p];
            odd |= tops[p];
            const uint32_t both = __byte_perm(tops[p], 0, 0x1010);
#pragma unroll
            for (int b = 0; b < NB; ++b) rel[p][b] = __byte_perm(kv_relative_scales(w[b / 2] & live[p], both), 0, b & 1 ? 0x3424 : 0x1404);
        }
        if (__any_sync(0xffffffffu, (odd & 0xffff0000u) != 0u)) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                uint32_t w[(NB + 1) / 2];
                load_pair_scales<NB>(rec + kv_value_scale_offset(FMT, NB) + (t + 4 * p) * 2 * kv_scale_stride(NB), w);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int e = (int)(w[b / 2] >> (16 * (b & 1) + 8 * i) & 0xffu), top = (int)(tops[p] >> (8 * i) & 0xffu);
                        f[i] = e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)max(e - top + 127, 0) << 23);
                    }
                    rel[p][b] = f16x2_of(f[0], f[1]);   // zero below 2^-25
                }
            }
        }
        if constexpr (EDGE) {   // what lies in the places that do not count may be anything
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t keep = live_pair(t, p, lo, hi);
#pragma unroll
                for (int b = 0; b < NB; ++b) rel[p][b] &= keep;
            }
        }
    }
    // mask of the f16 pair of tokens 2t + 8 p and the next
    __device__ static __forceinline__ uint32_t live_pair(int t, int p, int lo, int hi) {
        const int tok = 2 * t + 8 * p;
        return (tok >= lo && tok < hi ? 0xffffu : 0u) | (tok + 1 >= lo && tok + 1 < hi ? 0xffff0000u : 0u);
    }

    // Adds a record's values; weights as pairs of the tokens 2t, 2t + 1 (0) and 2t + 8, 2t + 9 (1) of head g.
    template <bool EDGE>
    __device__ __forceinline__ void values(const uint8_t* rec, int lo, int hi, const Weights& weights, const uint32_t (&rel)[2][NB],
                                           int lane) {
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if constexpr (!kMx && EDGE) keep[0] = live_pair(lane & 3, 0, lo, hi), keep[1] = live_pair(lane & 3, 1, lo, hi);
        uint32_t v[NB * VP / 4];
        load_lane<NB * VP>(rec + kv_value_offset(FMT, NB), lane, v);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t f[4][2];   // [element][token pair]
            if constexpr (!kMx) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        f[e][p] = v[8 * b + 4 * (e >> 1) + 2 * p + (e & 1)];
                        if constexpr (EDGE) f[e][p] &= keep[p];
                    }
            } else if constexpr (FMT == kKvMx8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f16_of_e4m3x4(v[4 * b + e], f[e][0], f[e][1]);
            } else {
                f16_of_e2m1x8(v[2 * b], f[0][0], f[0][1], f[1][0], f[1][1]);
                f16_of_e2m1x8(v[2 * b + 1], f[2][0], f[2][1], f[3][0], f[3][1]);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                uint32_t w[kParts][2];
#pragma unroll
                for (int u = 0; u < kParts; ++u)
#pragma unroll
                    for (int p = 0; p < 2; ++p) w[u][p] = kMx ? mul_f16x2(weights[r][u][p], rel[p][b]) : weights[r][u][p];
#pragma unroll
                for (int u = 0; u < kParts; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        mma_16x8x16<kBf>(o[r][b][i], f[2 * i][0], f[2 * i + 1][0], f[2 * i][1], f[2 * i + 1][1], w[u][0], w[u][1]);
            }
        }
    }

    // the largest over all lanes that hold the same heads
    static __device__ __forceinline__ float max_over_tokens(float x) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
    }

    // Moves a lagging maximum (held negated) to 7 below the largest of p if that passes it by more than the lag; returns the
    // factor for what was summed relative to the old one, applies it to l, and moves the second maximum, which is relative.
    template <int N, typename F>
    static __device__ __forceinline__ float raise(const float2 (&p)[N][2], float& neg, float& neg_relative, float& l, F&& head) {
        float most = -INFINITY;
#pragma unroll
        for (int n = 0; n < N; ++n) most = fmaxf(most, fmaxf(head(p[n][0]), head(p[n][1])));
        most = max_over_tokens(most);
        const float to = most + neg > kKvLag ? kKvHead - ceilf(most) : neg, shift = to - neg;   // old - new
        neg = to;
        neg_relative -= shift;
        const float f = ex2(shift);
        l *= f;
        return f;
    }

    // N records; EDGE: of their 16 N tokens [lo, hi) count, else all.  Two at a time keep twice the independent work in
    // flight and share the tests for a new maximum and the work around the ring.
    template <int N, bool EDGE>
    __device__ __forceinline__ void records(const uint8_t* const (&rec)[N], int lo, int hi, int lane) {
        const int g = lane >> 2;
        float s[N][RT][4];
#pragma unroll
        for (int n = 0; n < N; ++n) scores(rec[n], s[n], lane);
        bool dead[N][2];   // tokens g, g + 8 that do not count
        float te[N][2];
        uint32_t rel[N][2][NB];
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int tok = n * kKvRecord + g + 8 * i;
                dead[n][i] = EDGE && (tok < lo || tok >= hi);
                // the token's top byte as a float, by way of the integers behind 2^23
                if constexpr (kMx)
                    te[n][i] = __uint_as_float(0x4b000000u | rec[n][kv_value_top_offset(FMT, NB) + 4 * (g >> 1) + (g & 1) + 16 * i]) - 8388735.f;
            }
            if constexpr (kMx) value_scales<EDGE>(rec[n], lo - n * kKvRecord, hi - n * kKvRecord, rel[n], lane);
        }
        // softmax
        Weights weights[N];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            // tokens g (0) and g + 8 (1): scores, and exponents of the weights.  A score is rounded before m is taken from it
            // (no fma): what m was made of and what it is compared with are the same number, however large
            float2 p[N][2], x[N][2];
            float over = -INFINITY;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    p[n][i] = mul2(make_float2(s[n][r][2 * i], s[n][r][2 * i + 1]), qs[r]);
                    if (dead[n][i]) p[n][i] = make_float2(-INFINITY, -INFINITY);
                    x[n][i] = add2(p[n][i], nm[r]);
                    over = fmaxf(over, fmaxf(x[n][i].x, x[n][i].y));
                }
            if (__any_sync(0xffffffffu, over > kKvLag)) {
                // from the scores: the first time, m is far below them and their differences are lost in x
                const float2 f = make_float2(raise(p, nm[r].x, nd[r].x, l[r][0], [](float2 v) { return v.x; }),
                                             raise(p, nm[r].y, nd[r].y, l[r][1], [](float2 v) { return v.y; }));
                if constexpr (!kMx) scale_rows(r, f);
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) x[n][i] = add2(p[n][i], nm[r]);
            }
            float w[N][4];
#pragma unroll
            for (int n = 0; n < N; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) w[n][2 * i] = ex2(x[n][i].x), w[n][2 * i + 1] = ex2(x[n][i].y);
                l[r][0] += w[n][0] + w[n][2];
                l[r][1] += w[n][1] + w[n][3];
            }
            if constexpr (kMx) {
                float2 y[N][2];
                float high = -INFINITY;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        y[n][i] = add2(x[n][i], add2(make_float2(te[n][i], te[n][i]), nd[r]));
                        high = fmaxf(high, fmaxf(y[n][i].x, y[n][i].y));
                    }
                if (__any_sync(0xffffffffu, high > kKvLag)) {
                    float2 sum[N][2];
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) sum[n][i] = add2(x[n][i], make_float2(te[n][i], te[n][i]));
                    float none = 0.f, nothing = 0.f;
                    scale_rows(r, make_float2(raise(sum, nd[r].x, none, nothing, [](float2 v) { return v.x; }),
                                              raise(sum, nd[r].y, none, nothing, [](float2 v) { return v.y; })));
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) y[n][i] = add2(x[n][i], add2(make_float2(te[n][i], te[n][i]), nd[r]));
                }
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) w[n][2 * i] = ex2(y[n][i].x), w[n][2 * i + 1] = ex2(y[n][i].y);
            }
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t part[kParts];
                    split_pair<kBf>(w[n][2 * i], w[n][2 * i + 1], part);
#pragma unroll
                    for (int u = 0; u < kParts; ++u) weights[n][r][u][i] = transpose8x8(part[u]);
                }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) values<EDGE>(rec[n], lo - n * kKvRecord, hi - n * kKvRecord, weights[n], rel[n], lane);
    }

    // the sum of weights of head 2t + c of tile r
    __device__ __forceinline__ float denominator(int r, int c) const {
        float s = l[r][c];
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        s += __shfl_xor_sync(0xffffffffu, s, 8);
        return s + __shfl_xor_sync(0xffffffffu, s, 16);
    }
    // its numerators 32 b + 4 g .. + 3
    __device__ __forceinline__ float4 numerators(int r, int c, int b) const {
        return make_float4(o[r][b][0][c], o[r][b][0][2 + c], o[r][b][1][c], o[r][b][1][2 + c]);
    }
    __device__ __forceinline__ float maximum(int r, int c) const { return -(c ? nm[r].y : nm[r].x); }
    __device__ __forceinline__ float relative(int r, int c) const { return kMx ? -(c ? nd[r].y : nd[r].x) : 0.f; }
    // Partial result of this warp's rows: denominators (times 2^m), numerators (times 2^(m + d)); m, d, denominators last.
    __device__ __forceinline__ void store_partial(float* o_rows, float* stats, int lane) const {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float s = denominator(r, c);
                const int row = 8 * r + 2 * t + c;
                if (g == 0) {
                    stats[3 * row] = maximum(r, c);
                    stats[3 * row + 1] = relative(r, c);
                    stats[3 * row + 2] = s;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) *reinterpret_cast<float4*>(o_rows + row * D + 32 * b + 4 * g) = numerators(r, c, b);
            }
    }
};

// The quotient of a numerator 2^(m + d) o and a denominator 2^m l.  The power of two is applied in two halves: the scales of
// the values span fp32's exponents, and their product with 1 / l alone could leave them.  Nothing attended to gives 0.
struct KvQuotient {
    float inv, p, q, lse;
    __device__ __forceinline__ KvQuotient(float l, float d, float m) {
        const int k = (int)fminf(fmaxf(d, -252.f), 252.f), half = k / 2;   // an integer
        inv = l == 0.f ? 0.f : __fdividef(1.f, l);   // (l stays below 2^126: 2^15 for each of fewer than 2^31 tokens)
        p = __uint_as_float((uint32_t)(half + 127) << 23);
        q = __uint_as_float((uint32_t)(k - half + 127) << 23);
        lse = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.693147180559945309f;
    }
    __device__ __forceinline__ float operator()(float o) const { return o * inv * p * q; }
};

// ------------------------------------------------------------------------------------------------
// Split of the work (its arithmetic: kv_split.cuh).  Units are (sequence, key head, chunk of query heads); the records of all
// units, one unit after the other, are cut into equal ranges, one for each CTA and within it for each warp, wherever the cuts
// fall: lengths may differ as they like.  (Where whole units make ranges that are hardly longer, the CTAs' cuts are between units: nothing is
// left to join across CTAs, which takes 3 to 4 us.  96 sequences of 32 to 64 records, one unit each: 35 -> 30 us; 128 units of 7
// to 44: 14.8 -> 11.9; 8 of 32, on 8 CTAs instead of 32: 11.2, the same.)  A warp writes what it holds of units that lie in
// its range altogether; at most its first and its last unit are partial.  Partial results are joined in shared memory by the
// CTA, and what is still partial then (at most two units a CTA) through the workspace by whichever of the unit's CTAs is done
// last.  All joins run in a fixed order: same bits every time.  (A second kernel for that join cost 4 to 7 us a call.)
// The counts behind "last" are never set back: they carry the number of the call, and a count that holds a smaller one is raised
// to it first.  So whatever calls that overlapped against the rules have left there, the next one finds its counts at zero.  The
// number: every CTA of a call reads how many CTAs have run before its own, over all calls, and then adds itself; divided by the CTAs
// of a call that is the same for all of them.  (0 to 0.3 us a call; counts zeroed by the CTA that is done with them last 0.6 to
// 1.2, calls numbered by what the additions return 0.3 to 1.3.)
// ------------------------------------------------------------------------------------------------

// Shape of a CTA.  Each warp (or team of warps that share records) has a ring of records in shared memory, filled by
// bulk copies: one copy a record, since a record is contiguous.  The partial result of a warp's last unit goes into its
// ring, which is empty by then; that of its first one, if it is another, to the workspace.
template <int FMT, int NB, int RT, int HALVES>
struct KvShape {
    // at most as many warps as registers allow: accumulators and query take 8 NB RT + 4 NB RT HALVES registers a thread of the
    // 65536 / (32 warps)
    static constexpr int kRegisters = 8 * NB * RT + 4 * NB * RT * HALVES;
    // (16 instead of 12 for mx8 and heads of 128: a batch of up to 4097 tokens 68 us instead of 63; 12 instead of 16 for mx4:
    // 96 instead of 90, whose spills cost less than the warps bring.)
    // Two records at a time where a record is much arithmetic for few bytes: mx8, 131071 tokens, 56.5 us instead of 61.3 one
    // at a time, mx4 89.6 instead of 96.8; 16-bit formats lose by it, heads of 64 under fp32 queries 38.4 instead of 32.8.
    static constexpr bool kPair = FMT >= kKvMx8 && NB * RT <= 4;
    static constexpr int kMaxWarps = kRegisters <= (FMT == kKvMx4 ? 48 : 32) ? 16 : kRegisters <= 80 ? 12 : 8;
    static constexpr int kMaxThreads = 32 * kMaxWarps;
    static constexpr int kRecord = kv_record_bytes(FMT, NB);
    static constexpr int kMaxStages = 16;                        // of a ring
    static constexpr int kSmemMax = 232448 - 12288;              // of a CTA, less the static part
    static constexpr int kRows = 8 * RT;
    static constexpr int kPartial = kRows * (32 * NB + 3);       // floats: numerators, then (m, d, l) of each row
    static_assert(kMaxWarps * kPartial <= kv_slot_floats(32 * NB) && kMaxWarps * kPartial * 4 <= kSmemMax && kSmemMax / 4 / kRecord >= 3 &&
                      kPartial * 4 % 32 == 0 && kRecord % 16 == 0, "rings, slots");
};

constexpr unsigned long long kKvCall = 1024;   // more than a call ever counts to

struct KvSplit {
    int chunks;                     // chunks of query heads per key head
    int row_warps;                  // warps that share a record, each with its own rows
    int per_seq, teams, stages;     // units of a sequence; warps of a CTA / row_warps; records of a team's ring
    int ring_bytes;                 // of a team: its records, and room for its warps' partial results
    KvDiv by_ctas, by_per_seq, by_teams, by_page, by_chunks;   // (by_page: records of a page)
    float* slots;                   // [ctas][kv_slot_floats]: partial results of the warps' first units
    float* partial;                 // [ctas][2][rows][dim + 3]: of the CTAs, numerators of all rows, then (m, d, l) of each
    unsigned long long* count;      // [ctas][2], [ctas]: parts of a group, groups of a unit that are done, under the call's number
                                    // times kKvCall; [1]: CTAs that have run
};

// positions of sequence b that are attended to: [lo, hi)
__device__ __forceinline__ bool kv_span(const KvPool& pool, const KvSeqs& s, int window, int b, int& lo, int& hi) {
    const int n = __ldg(s.lengths + b);
    const int64_t room = (int64_t)s.max_pages * pool.records_per_page * kKvRecord;
    hi = (int)min((int64_t)max(n, 0), room);
    lo = window > 0 ? max(hi - window, 0) : 0;
    return n >= 0 && n <= room;
}

// A walk over the records of a range, in order: the unit (b, hu) and the record r of its n.
struct KvWalk {
    int b, hu, r, n, lo, hi;

    // to the record `at` of all records; i0 / first: a sequence at or before its own, and the records before that
    __device__ __forceinline__ void seek(const KvPool& pool, const KvSeqs& s, int window, int per_seq, int64_t q, int64_t at, int i0,
                                         int64_t first) {
        for (b = i0;; ++b) {
            kv_span(pool, s, window, b, lo, hi);
            n = kv_records(lo, hi);
            if (first + n > q) break;
            first += n;
        }
        at -= first * per_seq;
        hu = per_seq > 1 ? (int)kv_div(at, n) : 0;
        r = (int)(at - (int64_t)hu * n);
    }
    // to the first record of the next unit (there is one)
    __device__ __forceinline__ void next_unit(const KvPool& pool, const KvSeqs& s, int window, int per_seq) {
        r = 0;
        if (++hu < per_seq) return;
        hu = 0;
        do {
            kv_span(pool, s, window, ++b, lo, hi);
            n = kv_records(lo, hi);
        } while (n == 0);
    }
};

// Where a team's copies are: the walk stands behind the records that are fetched or about to be from the current page.
struct KvAhead {
    KvWalk walk;
    int to_fetch, slot, in;   // records left behind them, slot of the page in the table, first record of the next page
};

// One bulk copy of a record into shared memory, its bytes counted on the mbarrier.  The records are read once: they make
// way in the L2 first, so that page tables, partial results and the program itself stay there (2 to 3 us of 60 to 180).
__device__ __forceinline__ void kv_copy_record(uint32_t dst, const uint8_t* src, uint32_t bytes, uint32_t bar, uint64_t policy) {
    mbar_arrive_expect_tx(bar, bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy)
                 : "memory");
}

// 16 bytes of a partial result, in shared memory or (other CTAs' too, so not from the L1) in global memory
__device__ __forceinline__ float4 load_part4(const float* p) {
    float4 v;
    asm volatile("ld.relaxed.gpu.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float load_part(const float* p) {
    float v;
    asm volatile("ld.relaxed.gpu.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}

template <int FMT, int NB, int RT, int HALVES>
__global__ void __launch_bounds__(KvShape<FMT, NB, RT, HALVES>::kMaxThreads, 1)
    kv_attend_kernel(KvPool pool, KvSeqs seqs, KvAttend a, KvSplit split, uint64_t* errors) {
    using Shape = KvShape<FMT, NB, RT, HALVES>;
    constexpr int D = 32 * NB, kRows = Shape::kRows, kMaxWarps = Shape::kMaxWarps, kMaxStages = Shape::kMaxStages;
    extern __shared__ __align__(128) uint8_t smem[];          // rings
    __shared__ int64_t s_before[32 * kMaxWarps];                  // records of the sequences before thread i's
    __shared__ int64_t s_warp[kMaxWarps];
    __shared__ int64_t s_unit[2 * kMaxWarps];
    __shared__ int s_ends[2 * kMaxWarps];                        // bit 0: the unit begins there, 1: it ends there, 2: in the ring
    __shared__ int64_t s_from[2 * kMaxWarps];                    // first record, among all, of the slot's unit, and
    __shared__ int s_long[2 * kMaxWarps];                        // its records
    __shared__ int s_turn[2];                                 // whether this CTA joins its first / last unit's parts
    __shared__ __align__(8) unsigned long long s_call;        // CTAs that have run before this one; the call's number times kKvCall
    __shared__ __align__(8) uint64_t s_full[kMaxWarps][kMaxStages], s_empty[kMaxWarps][kMaxStages];
    __shared__ uint8_t s_ok[kMaxWarps][kMaxStages];              // whether the record could be fetched
    __shared__ int s_abort, s_drain[kMaxWarps];
    __shared__ KvAhead s_ahead[kMaxWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int threads = blockDim.x, warps = threads >> 5;
    const int per_seq = split.per_seq;
    const int chunk_rows = kRows * split.row_warps;
    const int teams = split.teams, team = split.row_warps == 1 ? warp : warp / split.row_warps, rw = warp - team * split.row_warps;
    const int stages = split.stages;
    uint8_t* ring = smem + team * split.ring_bytes;
    // partial results: slot 0 (a unit that began before the warp's range), slot 1 (one that goes on behind it); `last`: of
    // the warp's last unit
    auto slot_rows = [&](int w, bool last) {
        const int of = split.row_warps == 1 ? w : w / split.row_warps;   // team
        return last ? reinterpret_cast<float*>(smem + of * split.ring_bytes) + (w - of * split.row_warps) * Shape::kPartial
                    : split.slots + (int64_t)blockIdx.x * kv_slot_floats(D) + w * Shape::kPartial;
    };

    const bool numbers = tid == threads - 1;   // the thread that sees to the call's number, waited for behind the records
    if (numbers)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(&s_call)), "l"(split.count + 3 * gridDim.x) : "memory");

    // ---- records of all sequences, scanned by the CTA
    const int per = (seqs.batch + threads - 1) / threads;
    int64_t mine = 0;
#pragma unroll 1
    for (int b = tid * per; b < min((tid + 1) * per, seqs.batch); ++b) {
        int lo, hi;
        if (!kv_span(pool, seqs, a.window, b, lo, hi) && blockIdx.x == 0) kv_report(errors, kStatusBadSequence);
        mine += kv_records(lo, hi);
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) s_warp[warp] = upto;
    if (tid < 2 * warps) s_unit[tid] = -1;
    if (tid == 0) s_abort = 0;
    if (rw == 0 && lane < stages) {
        mbar_init(smem_u32(&s_full[team][lane]), 1);
        mbar_init(smem_u32(&s_empty[team][lane]), split.row_warps);
    }
    mbar_fence_init();
    __syncthreads();
    int64_t base = 0, total = 0;
    for (int i = 0; i < warps; ++i) {
        if (i < warp) base += s_warp[i];
        total += s_warp[i];
    }
    s_before[tid] = base + upto - mine;
    total *= per_seq;
    const int64_t part = kv_part(split.by_ctas, total);
    // Whole units, as many for each CTA, where no range gets much longer by it
    const int64_t units = (int64_t)seqs.batch * per_seq, whole = split.by_ctas(units + gridDim.x - 1);
    const bool cut = __syncthreads_or(per > 1 || !kv_keep_whole(whole, mine, part));
    auto range_begin = [&](int64_t cta) -> int64_t {
        if (cut) return min(cta * part, total);
        const int64_t u = cta * whole;
        if (u >= units) return total;
        const int b = (int)split.by_per_seq(u);
        int lo, hi;
        kv_span(pool, seqs, a.window, b, lo, hi);
        return s_before[b] * per_seq + (u - (int64_t)b * per_seq) * kv_records(lo, hi);
    };
    const int64_t c0 = range_begin(blockIdx.x), c1 = range_begin((int64_t)blockIdx.x + 1);
    const KvRange range = kv_team_range(split.by_teams, c0, c1, team);
    const int64_t t0 = range.begin;
    int left = (int)min(range.end - t0, (int64_t)0x7fffffff);   // records of the team that are not yet done with
    if (range.part > 0x7fffffff && tid == 0) kv_report(errors, kStatusBadSequence);   // (2^31 records a warp: lengths gone wrong)

    if (left > 0) {
        KvWalk at;
        {
            const int64_t q = split.by_per_seq(t0);   // all units of a sequence have as many records
            int i = 31 - __clz(__ballot_sync(0xffffffffu, s_before[lane * warps] <= q));
            i = i * warps + 31 - __clz(__ballot_sync(0xffffffffu, lane < warps && s_before[min(i * warps + lane, threads - 1)] <= q));
            at.seek(pool, seqs, a.window, per_seq, q, t0, i * per, s_before[i]);
        }
        // The copies, by the team's first warp: the walk of the records to fetch runs a ring ahead of the one below.  What it
        // needs at the end of a page only waits in shared memory.
        const uint8_t* src = nullptr;   // the next record (null: a page id out of range)
        int run = 0;                    // records to fetch from there on the page
        int next_page = -1;             // page id of the next slot of the page table, asked for early
        KvAhead& ahead = s_ahead[warp];
        if (rw == 0) {
            const int rec = at.lo / kKvRecord + at.r, slot = (int)split.by_page(rec);
            next_page = __ldg(seqs.table + (int64_t)at.b * seqs.max_pages + slot);   // (kv_span cuts at max_pages)
            if (lane == 0) ahead = {at, left, slot - 1, rec - slot * pool.records_per_page};
            __syncwarp();
        }
        auto another_page = [&]() {     // false: nothing left to fetch
            KvWalk x = ahead.walk;
            int to_fetch = ahead.to_fetch, slot = ahead.slot + 1, in = ahead.in, page = next_page;
            if (to_fetch == 0) return false;
            if (x.r == x.n) {
                x.next_unit(pool, seqs, a.window, per_seq);
                slot = (int)split.by_page(x.lo / kKvRecord);
                in = x.lo / kKvRecord - slot * pool.records_per_page;
                page = __ldg(seqs.table + (int64_t)x.b * seqs.max_pages + slot);
            }
            run = min(min(pool.records_per_page - in, x.n - x.r), to_fetch);
            src = page < 0 || page >= pool.pages
                      ? nullptr
                      : pool.base + (((int64_t)page * pool.heads + (int)split.by_chunks(x.hu)) * pool.records_per_page + in) * Shape::kRecord;
            if (slot + 1 < seqs.max_pages) next_page = __ldg(seqs.table + (int64_t)x.b * seqs.max_pages + slot + 1);
            x.r += run;
            __syncwarp();
            if (lane == 0) ahead = {x, to_fetch - run, slot, 0};
            __syncwarp();
            return true;
        };
        const uint32_t ring_at = smem_u32(ring), full_at = smem_u32(&s_full[team][0]),
                       empty_at = smem_u32(&s_empty[team][0]);
        uint64_t policy;
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));

        KvWarp<FMT, NB, RT, HALVES> w;
        int stage = 0, fill = 0, empty = rw == 0 ? stages : 0;   // stage to read next; stage to fill next, stages to fill
        uint32_t phase = 0, fill_phase = 1;
        bool alive = true;   // no wait has run out (the same in all lanes)
#pragma unroll 1
        while (true) {
            int seg = min(at.n - at.r, left);   // records of the unit here
            const int h = (int)split.by_chunks(at.hu), row0 = (at.hu - h * split.chunks) * chunk_rows + rw * kRows;
            w.load_query(a, (int64_t)at.b * a.seq_stride + (int64_t)h * a.group * a.head_stride, row0, a.group, lane);
            // the unit's span relative to the next record's first token
            int lo = at.lo - (at.lo / kKvRecord + at.r) * kKvRecord, hi = lo + (at.hi - at.lo);
            const int row_warps = opaque(split.row_warps);
            const int batch = stages >> 1;
            int fresh = opaque(1);                       // the query is on its way
            const bool pair = opaque(stages) >= 4;   // (else two would leave nothing under way)
#pragma unroll 1
            for (int j = seg; j > 0;) {
#pragma unroll 1
                while (empty >= batch && alive) {   // half a ring at a time
                    if (run == 0 && !another_page()) {
                        empty = -0x40000000;   // never again
                        break;
                    }
                    // as many at once as there are in a row, one a lane
                    const int k = min(min(empty, run), stages - fill);
                    if (lane < k) {
                        const int st = fill + lane;
                        // every warp of the team is done with what the stage held (true at once the first time round)
                        if (row_warps > 1) alive = mbar_wait(empty_at + 8 * st, fill_phase, &s_abort);
                        if (alive) {
                            s_ok[team][st] = src != nullptr;
                            if (src != nullptr) {
                                kv_copy_record(ring_at + st * Shape::kRecord, src + lane * Shape::kRecord, Shape::kRecord, full_at + 8 * st, policy);
                            } else {
                                mbar_arrive(full_at + 8 * st);
                            }
                        }
                    }
                    if (src == nullptr && lane == 0) kv_report(errors, kStatusBadPage);
                    if (row_warps > 1) alive = __all_sync(0xffffffffu, alive);
                    if (src != nullptr) src += k * Shape::kRecord;
                    run -= k;
                    empty -= k;
                    fill += k;
                    if (fill == stages) fill = 0, fill_phase ^= 1u;
                }
                if (fresh) {   // (the first copies' latency and the query's pass together)
                    w.convert_query(a, lane);
                    w.reset();
                    fresh = opaque(0);
                }
                const int take = Shape::kPair && j > 1 && lo <= 0 && hi >= 2 * kKvRecord && pair ? 2 : 1;
                const int next = stage + 1 == stages ? 0 : stage + 1;
                alive = alive && mbar_wait_warp(full_at + 8 * stage, phase, Shape::kPair && take == 2, full_at + 8 * next,
                                                next == 0 ? phase ^ 1u : phase, &s_abort);
                const uint8_t* here = ring + stage * Shape::kRecord;
                const bool ok = alive && s_ok[team][stage];
                bool one = ok;
                if constexpr (Shape::kPair) {
                    if (take == 2) {   // (all tokens of both count)
                        const uint8_t* there = ring + next * Shape::kRecord;
                        const bool ok2 = alive && s_ok[team][next];
                        one = ok != ok2;   // a record that is missing is left out
                        if (ok && ok2) {
                            const uint8_t* const both[2] = {here, there};
                            w.template records<2, false>(both, 0, 2 * kKvRecord, lane);
                        } else if (ok2) {
                            here = there;
                        }
                    }
                }
                if (one) {
                    const uint8_t* const single[1] = {here};
                    if (!Shape::kPair && lo <= 0 && hi >= kKvRecord) w.template records<1, false>(single, 0, kKvRecord, lane);
                    else w.template records<1, true>(single, max(lo, 0), min(hi, kKvRecord), lane);
                }
                __syncwarp();
                if (row_warps > 1 && lane == 0) {
                    mbar_arrive(empty_at + 8 * stage);
                    if (take == 2) mbar_arrive(empty_at + 8 * next);
                }
                j -= take;
                if (rw == 0) empty += take;
                lo -= take * kKvRecord;
                hi -= take * kKvRecord;
                stage += take;
                if (stage >= stages) stage -= stages, phase ^= 1u;
            }
            const bool begins = at.r == 0, ends = at.r + seg == at.n;
            if (begins && ends) {
                const int g = lane >> 2, t = lane & 3;
                const int64_t out0 = (int64_t)at.b * a.q_heads + split.by_chunks(at.hu) * a.group;
#pragma unroll
                for (int k = 0; k < RT; ++k)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float l = w.denominator(k, c);
                        const int row = row0 + 8 * k + 2 * t + c;
                        if (row < a.group) {
                            const KvQuotient f(l, w.relative(k, c), w.maximum(k, c));
                            if (g == 0 && a.lse != nullptr) a.lse[out0 + row] = f.lse;
#pragma unroll
                            for (int blk = 0; blk < NB; ++blk) {
                                const float4 o = w.numerators(k, c, blk);
                                const float y[4] = {f(o.x), f(o.y), f(o.z), f(o.w)};
                                store_row(a.out, (out0 + row) * D + 32 * blk + 4 * g, a.type, y);
                            }
                        }
                    }
            } else {
                const int which = begins ? 1 : 0;
                const bool last = left == seg;
                if (last && row_warps > 1) named_bar_sync(1 + team, 32 * row_warps);   // the ring is free
                float* rows = slot_rows(warp, last);
                w.store_partial(rows, rows + kRows * D, lane);
                if (lane == 0) {
                    s_unit[2 * warp + which] = (int64_t)at.b << 32 | at.hu;
                    s_ends[2 * warp + which] = (begins ? 1 : 0) | (ends ? 2 : 0) | (last ? 4 : 0);
                    s_from[2 * warp + which] = range.end - left - at.r;
                    s_long[2 * warp + which] = at.n;
                }
            }
            left -= seg;
            if (left == 0) break;
            at.next_unit(pool, seqs, a.window, per_seq);
        }
        if (!alive && lane == 0) {
            kv_report(errors, kStatusPipelineTimeout);
            // the copies still under way must land before the CTA leaves: the last fill of every stage
            for (int i = 0; rw == 0 && i < stages; ++i) {
                s_drain[warp] = 0;
                mbar_wait_limit(full_at + 8 * i, i < fill ? fill_phase ^ 1u : fill_phase, &s_drain[warp], 100000000LL);
            }
        }
    }
    __syncthreads();

    // ---- Joins.  Phase 0: the partial results of the CTA's warps, runs of equal units among the teams' slots, in order (lane e
    // looks at slot e % 2 of team e / 2).  What is whole then is final.  Units that several CTAs hold parts of: of every 24
    // neighbours the one that is done last joins their parts (phase 1), and of these the last one joins the unit's groups
    // (phase 2).  What is joined, and in which order, is fixed.  One warp joins one row of a task.
    {
        auto slot_of = [&](int e, int k) { return 2 * ((e >> 1) * split.row_warps + k) + (e & 1); };   // entry e, row warp k
        const int mine_at = slot_of(min(lane, 2 * teams - 1), 0);
        const int64_t unit = lane < 2 * teams ? s_unit[mine_at] : -1;
        const uint32_t valid = __ballot_sync(0xffffffffu, unit >= 0), before = valid & ((1u << lane) - 1u);
        const int64_t last = __shfl_sync(0xffffffffu, unit, before ? 31 - __clz(before) : 0);
        const uint32_t starts = __ballot_sync(0xffffffffu, unit >= 0 && (before == 0 || last != unit));
        const uint32_t begun = __ballot_sync(0xffffffffu, unit >= 0 && (s_ends[mine_at] & 1)),
                       ended = __ballot_sync(0xffffffffu, unit >= 0 && (s_ends[mine_at] & 2));
        const int rows_used = min(chunk_rows, a.group);
        auto run_from = [&](int e0) {   // the slots of the run that starts at e0
            const uint32_t later = starts & ~((2u << e0) - 1u);
            return valid & ~((1u << e0) - 1u) & (later ? (later & -later) - 1u : 0xffffffffu);
        };
        // the CTA's partial result of a unit that began before it (0) or goes on behind it (1)
        auto partial_of = [&](int64_t cta, int which) { return split.partial + (2 * cta + which) * chunk_rows * (D + 3); };
        // the CTA's units that are not whole in it: the first run's, if it began before the CTA, and the last run's, if it goes on
        const int e_first = starts ? __ffs(starts) - 1 : 0, e_last = starts ? 31 - __clz(starts) : 0;
        const uint32_t m_first = starts ? run_from(e_first) : 0u, m_last = starts ? run_from(e_last) : 0u;
        const bool open_first = m_first && !(begun & m_first), open_last = m_last && (begun & m_last) && !(ended & m_last);
        const bool open = open_first || open_last;
        KvHolders holders[2] = {};      // the CTAs that hold parts of such a unit
        if (open) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at_slot = slot_of(i ? e_last : e_first, 0);
                holders[i] = kv_holders(s_from[at_slot], s_long[at_slot], part);
            }
        }
        bool turn[2];                   // whether this CTA joins them
        auto join_of = [&](int i, int phase_no) { return kv_join(holders[i], blockIdx.x, phase_no, gridDim.x); };
        if (numbers) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("red.relaxed.gpu.global.add.u64 [%0], 1;" ::"l"(split.count + 3 * gridDim.x) : "memory");
            if (open) {   // (the counts that this CTA may add to, raised while the warps' results are joined)
                s_call = (unsigned long long)split.by_ctas((int64_t)s_call) * kKvCall;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!(i ? open_last : open_first)) continue;
                    for (int n = 1; n <= (holders[i].parts > kKvGroup ? 2 : 1); ++n)
                        asm volatile("red.relaxed.gpu.global.max.u64 [%0], %1;" ::"l"(split.count + join_of(i, n).count), "l"(s_call) : "memory");
                }
            }
        }
#pragma unroll 1
        for (int phase_no = 0; phase_no < 3; ++phase_no) {
            if (phase_no == 1 && !open) break;
            if (phase_no > 0) {
                const bool first = phase_no == 1 ? open_first : turn[0] && holders[0].parts > kKvGroup,
                           second = phase_no == 1 ? open_last : turn[1] && holders[1].parts > kKvGroup;   // what there is to count
                __syncthreads();   // the CTA's parts are written
                if (tid < 64 && lane == 0) {   // warp 0 for the first unit, warp 1 for the last
                    const int i = tid >> 5;
                    const KvJoin join = join_of(i, phase_no);
                    bool mine_now = i ? second : first;
                    if (mine_now) {
                        unsigned long long done;
                        asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], 1;" : "=l"(done) : "l"(split.count + join.count) : "memory");
                        mine_now = done == s_call + join.n - 1;
                    }
                    s_turn[i] = mine_now;
                }
                __syncthreads();
                turn[0] = s_turn[0], turn[1] = s_turn[1];
                if (!turn[0] && !turn[1]) break;
            }
            const int tasks = phase_no == 0 ? __popc(starts) : 2;
#pragma unroll 1
            for (int item = warp; item < tasks * rows_used; item += warps) {
                const int task = item / rows_used, row = item - task * rows_used;
                // where the results to join lie, one a lane, and where the joined one goes
                const float *from, *from_stats;
                float* to;
                uint32_t members;
                int64_t u;
                bool final_row;
                if (phase_no == 0) {
                    const int k = row / kRows, in = row - k * kRows;
                    uint32_t rest = starts;
                    for (int i = 0; i < task; ++i) rest &= rest - 1;
                    const int e0 = __ffs(rest) - 1;
                    members = run_from(e0);
                    const int sl = slot_of(members >> lane & 1u ? lane : e0, k);
                    const float* rows = slot_rows(sl >> 1, s_ends[sl] & 4);
                    from = rows + in * D;
                    from_stats = rows + kRows * D + 3 * in;
                    u = __shfl_sync(0xffffffffu, unit, e0);
                    final_row = (begun & members) && (ended & members);
                    to = partial_of(blockIdx.x, begun & members ? 1 : 0);
                } else {
                    if (!(task ? turn[1] : turn[0])) continue;
                    const KvHolders held = task ? holders[1] : holders[0];
                    const KvJoin join = kv_join(held, blockIdx.x, phase_no, gridDim.x);
                    const int cta = join.lead + join.step * min(lane, join.n - 1);
                    const float* rows = partial_of(cta, cta == held.owner ? 1 : 0);
                    from = rows + row * D;
                    from_stats = rows + chunk_rows * D + 3 * row;
                    members = (1u << join.n) - 1u;
                    u = __shfl_sync(0xffffffffu, unit, task ? e_last : e_first);
                    final_row = phase_no == 2 || held.parts <= kKvGroup;
                    to = partial_of(join.lead, join.lead == held.owner ? 1 : 0);
                }
                constexpr int kQuads = (D + 127) / 128;   // lane: elements 4 lane + 128 i .. + 3
                const bool member = members >> lane & 1u;
                float s[3] = {kKvMaxInit, 0.f, 0.f};   // m, d, l
                if (member) {
#pragma unroll
                    for (int i = 0; i < 3; ++i) s[i] = load_part(from_stats + i);
                }
                float4 o[kQuads];
#pragma unroll
                for (int i = 0; i < kQuads; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                float m = 0.f, d = 0.f, l = 0.f, c = 0.f;
                const int any = __ffs(members) - 1;
                for (uint32_t rest = members, round = 0; rest; ++round) {
                    float4 y[4][kQuads];
                    int e[4];
                    bool real[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {   // four on their way at once; the first result again, times 0, at the end
                        real[x] = rest != 0;
                        e[x] = rest ? __ffs(rest) - 1 : any;
                        rest &= rest - 1;
                        const float* row_at = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(from), e[x]));
#pragma unroll
                        for (int i = 0; i < kQuads; ++i) y[x][i] = load_part4(row_at + min(4 * lane + 128 * i, D - 4));
                    }
                    if (round == 0) {   // (while the first rows are on their way)
                        m = warp_max(s[0]);
                        const float shift = s[0] - m, e = member ? s[1] + shift : kKvMaxInit;
                        if constexpr (FMT >= kKvMx8) d = warp_max(e);
                        l = warp_sum(s[2] * ex2(shift));
                        c = member ? ex2(e - d) : 0.f;
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float f = __shfl_sync(0xffffffffu, c, e[x]);
                        if (!real[x]) f = 0.f;
#pragma unroll
                        for (int i = 0; i < kQuads; ++i) {
                            o[i].x = fmaf(y[x][i].x, f, o[i].x), o[i].y = fmaf(y[x][i].y, f, o[i].y);
                            o[i].z = fmaf(y[x][i].z, f, o[i].z), o[i].w = fmaf(y[x][i].w, f, o[i].w);
                        }
                    }
                }
                if (final_row) {
                    const int hu = (int)u, h = (int)split.by_chunks(hu), at_row = (hu - h * split.chunks) * chunk_rows + row;
                    if (at_row >= a.group) continue;   // a row behind the key head's last query head
                    const int64_t out_row = (u >> 32) * a.q_heads + (int64_t)h * a.group + at_row;
                    const KvQuotient f(l, d, m);
#pragma unroll
                    for (int i = 0; i < kQuads; ++i) {
                        const float y[4] = {f(o[i].x), f(o[i].y), f(o[i].z), f(o[i].w)};
                        if (4 * lane + 128 * i < D) store_row(a.out, out_row * D + 4 * lane + 128 * i, a.type, y);
                    }
                    if (lane == 0 && a.lse != nullptr) a.lse[out_row] = f.lse;
                } else {
#pragma unroll
                    for (int i = 0; i < kQuads; ++i)
                        if (4 * lane + 128 * i < D) *reinterpret_cast<float4*>(to + row * D + 4 * lane + 128 * i) = o[i];
                    if (lane == 0) {
                        float* to_stats = to + chunk_rows * D + 3 * row;
                        to_stats[0] = m, to_stats[1] = d, to_stats[2] = l;
                    }
                }
            }
        }
    }

    // ---- sequences with nothing to attend to
#pragma unroll 1
    for (int64_t b = blockIdx.x; b < seqs.batch; b += gridDim.x) {
        int lo, hi;
        kv_span(pool, seqs, a.window, (int)b, lo, hi);
        if (hi > lo) continue;
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int i = tid; i < a.q_heads * (D / 4); i += threads)
            store_row(a.out, b * a.q_heads * D + 4 * i, a.type, zero);
        if (a.lse != nullptr)
#pragma unroll 1
            for (int i = tid; i < a.q_heads; i += threads) a.lse[b * a.q_heads + i] = -INFINITY;
    }
}

template <int FMT, int NB, int RT, int HALVES>
struct KvAttendInstance {
    using Shape = KvShape<FMT, NB, RT, HALVES>;
    static cudaError_t init() {
        return cudaFuncSetAttribute(kv_attend_kernel<FMT, NB, RT, HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmemMax);
    }
    static int launch(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, uint64_t* errors,
                      cudaStream_t stream) {
        KvSplit split{};
        // warps for the rows of a key head: as many as it takes to cover them, a power of two, at most 8 (64 or 128 rows)
        split.row_warps = 1;
        while (split.row_warps < 8 && split.row_warps * 8 * RT < a.group) split.row_warps *= 2;
        // as many warps as registers allow and rings of three records (of four where two records are taken at a time)
        int warps = Shape::kMaxWarps;
        for (;; warps -= 4) {
            split.teams = warps / split.row_warps;
            split.stages = std::min(Shape::kSmemMax / split.teams / Shape::kRecord, Shape::kMaxStages);
            if (warps % split.row_warps == 0 && (split.stages >= (Shape::kPair ? 4 : 3) || warps <= 8)) break;
        }
        if (split.stages < 3) {   // 16-bit records of 12 KB and more, one row warp
            warps = split.teams = 4;
            split.stages = Shape::kSmemMax / split.teams / Shape::kRecord;
        }
        split.ring_bytes = std::max(split.stages * Shape::kRecord, split.row_warps * Shape::kPartial * 4);
        const int chunk_rows = split.row_warps * 8 * RT;
        split.chunks = (a.group + chunk_rows - 1) / chunk_rows;
        split.per_seq = pool.heads * split.chunks;
        split.by_ctas = KvDiv(work.ctas);
        split.by_per_seq = KvDiv(split.per_seq);
        split.by_teams = KvDiv(split.teams);
        split.by_page = KvDiv(pool.records_per_page);
        split.by_chunks = KvDiv(split.chunks);
        split.count = reinterpret_cast<unsigned long long*>(work.count);
        split.slots = work.slots;
        split.partial = work.partial;
        kv_attend_kernel<FMT, NB, RT, HALVES><<<work.ctas, 32 * warps, split.teams * split.ring_bytes, stream>>>(pool, seqs, a, split, errors);
        return 1;
    }
};

// Two tiles (16 heads) a warp where a key head serves more than 8 query heads, codes are to be converted -- once for both --
// and accumulators and query leave enough of 255 registers.  16 sequences of 8000 to 16384 tokens, 4 key heads of 192 with
// 16 query heads each: mx8 92 us against 100 with two warps that share the records, mx4 89 against 95; f16, with nothing
// to convert, 113 against 108 (of 128: 82 against 80).
constexpr bool kv_two_tiles(int fmt, int nb, int halves) { return fmt >= kKvMx8 && nb * (16 + 8 * halves) <= 144; }
template <int FMT, int NB, int HALVES>
int kv_attend_tiles(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, uint64_t* errors, cudaStream_t stream) {
    if constexpr (kv_two_tiles(FMT, NB, HALVES))
        if (a.group > 8) return KvAttendInstance<FMT, NB, 2, HALVES>::launch(pool, seqs, a, work, errors, stream);
    return KvAttendInstance<FMT, NB, 1, HALVES>::launch(pool, seqs, a, work, errors, stream);
}
// The query is one operand where its type fits it exactly.
template <int FMT, int NB>
int kv_attend_rows(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, uint64_t* errors, cudaStream_t stream) {
    if (a.type == kTypeBf16 || (a.type == kTypeF16 && FMT != kKvBf16))
        return kv_attend_tiles<FMT, NB, 1>(pool, seqs, a, work, errors, stream);
    if constexpr (FMT == kKvBf16)
        if (a.type == kTypeF32) return kv_attend_tiles<FMT, NB, 3>(pool, seqs, a, work, errors, stream);
    return kv_attend_tiles<FMT, NB, 2>(pool, seqs, a, work, errors, stream);
}
template <int FMT, int NB, int HALVES>
cudaError_t kv_attend_tiles_init() {
    if constexpr (kv_two_tiles(FMT, NB, HALVES)) {
        const cudaError_t e = KvAttendInstance<FMT, NB, 2, HALVES>::init();
        if (e != cudaSuccess) return e;
    }
    return KvAttendInstance<FMT, NB, 1, HALVES>::init();
}
template <int FMT, int NB>
cudaError_t kv_attend_rows_init() {
    cudaError_t e = kv_attend_tiles_init<FMT, NB, 1>();
    if (e == cudaSuccess) e = kv_attend_tiles_init<FMT, NB, 2>();
    if constexpr (FMT == kKvBf16)
        if (e == cudaSuccess) e = kv_attend_tiles_init<FMT, NB, 3>();
    return e;
}

template <int FMT>
int kv_attend_format(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, uint64_t* errors, cudaStream_t stream) {
    switch (pool.blocks) {
        case 1: return kv_attend_rows<FMT, 1>(pool, seqs, a, work, errors, stream);
        case 2: return kv_attend_rows<FMT, 2>(pool, seqs, a, work, errors, stream);
        case 3: return kv_attend_rows<FMT, 3>(pool, seqs, a, work, errors, stream);
        case 4: return kv_attend_rows<FMT, 4>(pool, seqs, a, work, errors, stream);
        case 6: return kv_attend_rows<FMT, 6>(pool, seqs, a, work, errors, stream);
        default: return kv_attend_rows<FMT, 8>(pool, seqs, a, work, errors, stream);
    }
}
template <int FMT>
cudaError_t kv_attend_format_init(int blocks) {
    switch (blocks) {
        case 1: return kv_attend_rows_init<FMT, 1>();
        case 2: return kv_attend_rows_init<FMT, 2>();
        case 3: return kv_attend_rows_init<FMT, 3>();
        case 4: return kv_attend_rows_init<FMT, 4>();
        case 6: return kv_attend_rows_init<FMT, 6>();
        default: return kv_attend_rows_init<FMT, 8>();
    }
}

int kv_attend_f16(const KvPool&, const KvSeqs&, const KvAttend&, const KvWork&, uint64_t*, cudaStream_t);
int kv_attend_bf16(const KvPool&, const KvSeqs&, const KvAttend&, const KvWork&, uint64_t*, cudaStream_t);
int kv_attend_mx8(const KvPool&, const KvSeqs&, const KvAttend&, const KvWork&, uint64_t*, cudaStream_t);
int kv_attend_mx4(const KvPool&, const KvSeqs&, const KvAttend&, const KvWork&, uint64_t*, cudaStream_t);
cudaError_t kv_attend_f16_init(int blocks);
cudaError_t kv_attend_bf16_init(int blocks);
cudaError_t kv_attend_mx8_init(int blocks);
cudaError_t kv_attend_mx4_init(int blocks);

}  // namespace eosb

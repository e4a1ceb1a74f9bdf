// Paged key-value cache: host-side interface of its kernels (kv_cache.cu, kv_attend_*.cu) and the page layout (how work is cut: kv_split.cuh).
//
// A page holds page_size tokens of every head; the unit of the layout is the RECORD: the keys and values of 16
// consecutive tokens of one head, contiguous, 16-byte aligned,
//     key codes | value codes | key scales | value scales | value tops      (the last three in the block-scaled formats)
// page p, head h, record r of the page sit at ((p * heads + h) * (page_size / 16) + r) * record_bytes.
//
// Inside a record the codes are stored in the order in which the 32 lanes of a warp feed them to mma.sync m16n8k16, so
// that the attention kernel reads them with conflict-free 16-byte loads and no shuffle.  With lane = 4 g + t
// (g = 0..7, t = 0..3) and blocks b of 32 elements:
//     keys    lane (g, t) holds elements 32 b + 8 t .. + 7 of every block b of the tokens g and g + 8 (an mma sums over
//             elements, so any order of them serves as long as the query uses the same one): first all of token g, then
//             all of token g + 8 -- but in the 16-bit formats, whose words are operands as they are, the two tokens' words
//             in turn, so that the four operands of an mma are one 16-byte load
//     values  lane (g, t) holds tokens {2t, 2t+1, 2t+8, 2t+9}, elements 32 b + 4 g + {0..3}; the two tokens of one 32-bit
//             operand are neighbours.  mx: element by element; 16 bits: words of the pairs (2t, 2t+1) and (2t+8, 2t+9) in the
//             order of the operands, elements (0, 1) with the first pair, (0, 1) with the second, (2, 3) likewise
// A lane's bytes are cut into 16-byte pieces (then 8, then 4); piece i of all lanes is one contiguous plane.
// Scales are one byte per token and block (2^(byte - 127)), blocks rounded up to 1, 2, 4 or 8: keys [16 tokens][blocks],
// values [8 token pairs][blocks][2], the order in which the attention kernel makes f16 pairs of them.  For every token
// pair a 32-bit word says what the kernel would otherwise have to find out for each of its loads: the largest scale byte
// of each token's values (bits 0-7, 8-15) and whether the token is out of the ordinary (bits 16, 24): a block stored as
// NaN, or one more than 2^14 below the token's largest (a block of zeros too).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace eosb {

constexpr int kKvF16 = 0, kKvBf16 = 1, kKvMx8 = 2, kKvMx4 = 3;        // EOS_B200_KV_*
constexpr int kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2;              // EOS_B200_TYPE_*
constexpr int kKvRecord = 16;                                         // tokens of a record

// bytes of one lane and one 32-element block: keys (one token) and values (four)
__host__ __device__ constexpr int kv_key_piece(int format) { return format <= kKvBf16 ? 16 : format == kKvMx8 ? 8 : 4; }
__host__ __device__ constexpr int kv_value_piece(int format) { return 2 * kv_key_piece(format); }
__host__ __device__ constexpr int kv_scale_stride(int blocks) { return blocks <= 2 ? blocks : blocks <= 4 ? 4 : 8; }
__host__ __device__ constexpr int kv_scale_bytes(int format, int blocks) {
    return format <= kKvBf16 ? 0 : kKvRecord * kv_scale_stride(blocks);
}
__host__ __device__ constexpr int kv_value_offset(int format, int blocks) { return 64 * blocks * kv_key_piece(format); }
__host__ __device__ constexpr int kv_key_scale_offset(int format, int blocks) {
    return kv_value_offset(format, blocks) + 32 * blocks * kv_value_piece(format);
}
__host__ __device__ constexpr int kv_value_scale_offset(int format, int blocks) {
    return kv_key_scale_offset(format, blocks) + kv_scale_bytes(format, blocks);
}
__host__ __device__ constexpr int kv_value_top_offset(int format, int blocks) {
    return kv_value_scale_offset(format, blocks) + kv_scale_bytes(format, blocks);
}
__host__ __device__ constexpr int kv_record_bytes(int format, int blocks) {
    return kv_value_top_offset(format, blocks) + (format <= kKvBf16 ? 0 : 32);
}
constexpr int kKvNear = 14;   // exponents below a token's largest that the attention kernel's ordinary path covers
// Scale bytes of a token pair's values, two blocks of (first token, second token), relative to the tokens' largest (tops: twice
// the pair's): bytes 60 - 4 (top - e), with zeros below them the f16 numbers 2^(e - top) for top - e <= kKvNear.  Four
// subtractions in one, right as long as no byte leaves its place; a token that does not count may hold anything -- it may be
// written meanwhile, its top already and its scales not yet -- so its bytes are masked first.
__host__ __device__ inline uint32_t kv_relative_scales(uint32_t scales, uint32_t tops) { return scales * 4u + (0x3c3c3c3cu - tops * 4u); }
__host__ __device__ inline uint32_t kv_live_bytes(bool first, bool second) { return (first ? 0x00ff00ffu : 0u) | (second ? 0xff00ff00u : 0u); }
// offset of byte p of a lane's `bytes` bytes (planes of 16, then 8, then 4 bytes per lane)
__host__ __device__ constexpr int kv_lane_offset(int bytes, int lane, int p) {
    const int plane = p >> 4, in = p & 15, rest = bytes - (plane << 4);
    if (rest >= 16) return plane * 512 + lane * 16 + in;
    if (rest >= 8 && in < 8) return plane * 512 + lane * 8 + in;
    return plane * 512 + (rest >= 8 ? 256 + lane * 4 + in - 8 : lane * 4 + in);
}

// Records that the positions [lo, hi) of a sequence lie in, for any positions that an int holds.
__host__ __device__ inline int kv_records(int lo, int hi) { return hi > lo ? (hi - 1) / kKvRecord + 1 - lo / kKvRecord : 0; }

struct KvPool {
    uint8_t* base;
    int64_t pages;
    int heads, dim, blocks, format;
    int records_per_page, record_bytes;
};

// The sequences of a call: row b of table lists the pages of sequence b in order.
struct KvSeqs {
    const int32_t* table;   // [batch, max_pages]
    int max_pages, batch;
    const int32_t* starts;  // [batch] position of the first token of the call (append / read)
    const int32_t* cu;      // [batch + 1] first row of each sequence's tokens; null: one token each
    const int32_t* lengths; // [batch] cached tokens (attend)
};

struct KvRows {             // keys or values of a call, [tokens, heads, dim] with strides in elements
    void* p;
    int64_t token_stride, head_stride;
    int vec;                // accesses of 16 bytes (1), of 32 bytes (2) are aligned
};

void launch_kv_append(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type,
                      int64_t tokens, uint64_t* errors, cudaStream_t stream);
void launch_kv_read(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                    uint64_t* errors, cudaStream_t stream);

struct KvAttend {
    const void* query;      // [batch, q_heads, dim], strides in elements
    int64_t seq_stride, head_stride;
    int vec;                // 16-byte loads of the query are aligned
    int type;               // of query and out
    int q_heads, group;
    void* out;              // [batch, q_heads, dim], 16-byte aligned
    float* lse;             // [batch, q_heads] or null
    float scale_log2;       // score scale times log2(e)
    int window;             // 0: all positions
};

// Workspace of a cache's attention calls, of a fixed size: captured graphs keep its addresses.
struct KvWork {
    int ctas;               // one per SM
    float* slots;           // [ctas][kv_slot_floats(dim)]: partial results of the CTAs' warps
    float* partial;         // [ctas][2][kKvMaxRows][dim + 3]: of the CTAs
    uint64_t* count;        // [3 ctas], and how many CTAs have run (see kv_attend.cuh); zero at first, never set back
    uint64_t* errors;       // [kKvErrors] what append, read and attend met; the counts only grow, the host remembers what it has reported
};
constexpr int kKvErrors = 3;           // pipeline timeout, bad page, bad sequence: kStatusPipelineTimeout and the two codes behind it
constexpr int kKvMaxRows = 128;        // query heads of one unit, at most
// 128 rows, or (small heads, 16 warps) 256
__host__ __device__ constexpr int kv_slot_floats(int dim) { return kKvMaxRows * (dim + 3) + (dim <= 96 ? 128 * (dim + 3) : 0); }

// cudaSuccess once the kernels of this format and dim are ready on the current device
cudaError_t kv_init(int format, int blocks);
int launch_kv_attend(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, uint64_t* errors,
                     cudaStream_t stream);

}  // namespace eosb

// Paged key-value cache: the calls by format.  Kernels: kv_io.cuh (append, read), kv_attend.cuh (attention).
#include "kv_cache.cuh"

#include "kv_attend.cuh"
#include "kv_io.cuh"

namespace eosb {

void launch_kv_append(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type,
                      int64_t tokens, uint64_t* errors, cudaStream_t stream) {
    switch (pool.format) {
        case kKvF16: return kv_append_f16(pool, seqs, key, value, type, tokens, errors, stream);
        case kKvBf16: return kv_append_bf16(pool, seqs, key, value, type, tokens, errors, stream);
        case kKvMx8: return kv_append_mx8(pool, seqs, key, value, type, tokens, errors, stream);
        default: return kv_append_mx4(pool, seqs, key, value, type, tokens, errors, stream);
    }
}

void launch_kv_read(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                    uint64_t* errors, cudaStream_t stream) {
    switch (pool.format) {
        case kKvF16: return kv_read_f16(pool, seqs, key, value, type, tokens, errors, stream);
        case kKvBf16: return kv_read_bf16(pool, seqs, key, value, type, tokens, errors, stream);
        case kKvMx8: return kv_read_mx8(pool, seqs, key, value, type, tokens, errors, stream);
        default: return kv_read_mx4(pool, seqs, key, value, type, tokens, errors, stream);
    }
}

int launch_kv_attend(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, uint64_t* errors,
                     cudaStream_t stream) {
    switch (pool.format) {
        case kKvF16: return kv_attend_f16(pool, seqs, a, work, errors, stream);
        case kKvBf16: return kv_attend_bf16(pool, seqs, a, work, errors, stream);
        case kKvMx8: return kv_attend_mx8(pool, seqs, a, work, errors, stream);
        default: return kv_attend_mx4(pool, seqs, a, work, errors, stream);
    }
}

cudaError_t kv_init(int format, int blocks) {
    cudaError_t e;
    switch (format) {
        case kKvF16: e = kv_io_f16_init(blocks); return e == cudaSuccess ? kv_attend_f16_init(blocks) : e;
        case kKvBf16: e = kv_io_bf16_init(blocks); return e == cudaSuccess ? kv_attend_bf16_init(blocks) : e;
        case kKvMx8: e = kv_io_mx8_init(blocks); return e == cudaSuccess ? kv_attend_mx8_init(blocks) : e;
        default: e = kv_io_mx4_init(blocks); return e == cudaSuccess ? kv_attend_mx4_init(blocks) : e;
    }
}

}  // namespace eosb

// Writing to and reading from a paged cache: the kernels of the f16 format (kv_io.cuh).
#include "kv_io.cuh"

namespace eosb {

void kv_append_f16(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                  uint64_t* errors, cudaStream_t stream) {
    kv_io_format<false, kKvF16>(pool, seqs, key, value, type, tokens, errors, stream);
}
void kv_read_f16(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                uint64_t* errors, cudaStream_t stream) {
    kv_io_format<true, kKvF16>(pool, seqs, key, value, type, tokens, errors, stream);
}

cudaError_t kv_io_f16_init(int blocks) { return kv_io_format_init<kKvF16>(blocks); }

}  // namespace eosb

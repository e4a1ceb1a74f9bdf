// Writing to and reading from a paged cache: the kernels of the bf16 format (kv_io.cuh).
#include "kv_io.cuh"

namespace eosb {

void kv_append_bf16(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                  uint64_t* errors, cudaStream_t stream) {
    kv_io_format<false, kKvBf16>(pool, seqs, key, value, type, tokens, errors, stream);
}
void kv_read_bf16(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                uint64_t* errors, cudaStream_t stream) {
    kv_io_format<true, kKvBf16>(pool, seqs, key, value, type, tokens, errors, stream);
}

cudaError_t kv_io_bf16_init(int blocks) { return kv_io_format_init<kKvBf16>(blocks); }

}  // namespace eosb

// Writing to and reading from a paged cache: the kernels of the mx8 format (kv_io.cuh).
#include "kv_io.cuh"

namespace eosb {

void kv_append_mx8(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                  uint64_t* errors, cudaStream_t stream) {
    kv_io_format<false, kKvMx8>(pool, seqs, key, value, type, tokens, errors, stream);
}
void kv_read_mx8(const KvPool& pool, const KvSeqs& seqs, const KvRows& key, const KvRows& value, int type, int64_t tokens,
                uint64_t* errors, cudaStream_t stream) {
    kv_io_format<true, kKvMx8>(pool, seqs, key, value, type, tokens, errors, stream);
}

cudaError_t kv_io_mx8_init(int blocks) { return kv_io_format_init<kKvMx8>(blocks); }

}  // namespace eosb

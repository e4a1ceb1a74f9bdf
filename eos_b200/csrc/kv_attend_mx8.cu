// Attention over a paged cache: the kernels of the mx8 format (kv_attend.cuh).
#include "kv_attend.cuh"

namespace eosb {

int kv_attend_mx8(const KvPool& pool, const KvSeqs& seqs, const KvAttend& a, const KvWork& work, uint64_t* errors,
                 cudaStream_t stream) {
    return kv_attend_format<kKvMx8>(pool, seqs, a, work, errors, stream);
}
cudaError_t kv_attend_mx8_init(int blocks) { return kv_attend_format_init<kKvMx8>(blocks); }

}  // namespace eosb

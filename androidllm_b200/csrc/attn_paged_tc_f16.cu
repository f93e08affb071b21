// Paged attention on tcgen05 instantiated for f16 caches (attn_paged_tc_body.cuh).
#include "attn_paged_tc_body.cuh"

namespace alm {
cudaError_t launch_attn_paged_tc_f16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int nq, int* err,
                                    cudaStream_t st) {
  return launch_tc_t<half>(a, b, kv, nq, err, st);
}
cudaError_t attn_paged_tc_attrs_f16() { return tc_paged_attrs<half>(); }
bool attn_paged_tc_fits(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv) { return tc_paged_fits(a, b, kv); }
}  // namespace alm

// Paged attention instantiated for f16 caches (attn_paged_body.cuh).
#include "attn_paged_body.cuh"

namespace alm {
cudaError_t launch_attn_paged_f16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st) {
  return launch_paged_t<half>(a, b, kv, err, st);
}
cudaError_t attn_paged_attrs_f16() { return paged_attr_all<half>(); }
}  // namespace alm

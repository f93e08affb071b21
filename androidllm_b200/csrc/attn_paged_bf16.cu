// Paged attention instantiated for bf16 caches (attn_paged_body.cuh).
#include "attn_paged_body.cuh"

namespace alm {
cudaError_t launch_attn_paged_bf16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st) {
  return launch_paged_t<__nv_bfloat16>(a, b, kv, err, st);
}
cudaError_t attn_paged_attrs_bf16() { return paged_attr_all<__nv_bfloat16>(); }
}  // namespace alm

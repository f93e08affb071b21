// Paged attention on tcgen05 instantiated for bf16 caches (attn_paged_tc_body.cuh).
#include "attn_paged_tc_body.cuh"

namespace alm {
cudaError_t launch_attn_paged_tc_bf16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int nq, int* err,
                                    cudaStream_t st) {
  return launch_tc_t<__nv_bfloat16>(a, b, kv, nq, err, st);
}
cudaError_t attn_paged_tc_attrs_bf16() { return tc_paged_attrs<__nv_bfloat16>(); }
}  // namespace alm

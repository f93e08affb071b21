// Operators of a batched step on device data: argument structs and launchers
// shared by paged_api.cu (entry points and checks), rope_append.cu,
// attn_paged_body.cuh, attn_paged_tc_body.cuh and verify.cu.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace alm {

// One layer's pages, (n_pages, kv_heads, page_size, head_dim) each.
struct PagedKV {
  char* k;
  char* v;
  int n_pages, page_size, page_shift;   // page_shift: log2(page_size), or -1
  int kv_heads, head_dim;
};

// The pass's sequences (see alm_seq_batch).
struct SeqBatch {
  int n_seq, n_rows, max_rows;
  int table_rows, table_pages, page_stride;
  const int* row_start;
  const int* kv_len;
  const int* table;
  const int* slots;
};

// What a sequence's entries say, clamped to what exists: rows [row0, row0 +
// n_new), the last of n_kv positions (n_new > n_kv leaves rows at negative
// positions), its row of the page table (null: no such row).  A sequence longer
// than its row of the table has no position (fits is false): the places of its
// rows are not known.
struct Seq {
  int row0, n_new, n_kv;
  bool fits;
  const int* pages;
};

ALM_DEV Seq load_seq(const SeqBatch& b, const PagedKV& kv, int s) {
  Seq q;
  const int lo = max(0, min(__ldg(b.row_start + s), b.n_rows));
  const int hi = max(lo, min(__ldg(b.row_start + s + 1), b.n_rows));
  q.row0 = lo;
  q.n_new = hi - lo;
  // (256 below 2^31, so that the end of a tile behind the last position is a number)
  const long long cap = min(static_cast<long long>(b.table_pages) * kv.page_size, 0x7fffff00ll);
  const int len = max(0, __ldg(b.kv_len + s));
  q.fits = len <= cap;
  q.n_kv = q.fits ? len : 0;
  const int t = b.slots ? __ldg(b.slots + s) : s;
  q.pages = t >= 0 && t < b.table_rows ? b.table + static_cast<size_t>(t) * b.page_stride : nullptr;
  return q;
}

ALM_DEV int page_of(const PagedKV& kv, int pos) { return kv.page_shift >= 0 ? pos >> kv.page_shift : pos / kv.page_size; }

// Element offset of (page, head, position) inside K or V.
ALM_DEV size_t kv_offset(const PagedKV& kv, int page, int head, int in_page) {
  return ((static_cast<size_t>(page) * kv.kv_heads + head) * kv.page_size + in_page) * kv.head_dim;
}

// Pairs of fp32 in one 64-bit register: one instruction for both.
ALM_DEV uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
ALM_DEV void unpair(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
ALM_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
ALM_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
ALM_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Launch of an operator: its grid may be set up while the stream's last kernel
// ends (programmatic dependent launch); every kernel here calls
// grid_dep_wait() before it reads anything.
struct OpLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  OpLaunch(dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster = 0) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cluster > 0) {
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim.x = cluster;
      attr[1].val.clusterDim.y = 1;
      attr[1].val.clusterDim.z = 1;
      cfg.numAttrs = 2;
    }
  }
};

struct RopeAppend {
  const char *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // bytes
  char* q_out;
  int64_t qo_row, qo_head;                               // bytes
  int heads;
  const char *q_norm, *k_norm;
  float eps;
  const char* rope;
  int rope_rows, rot;
};

struct AttnPaged {
  const char* q;
  int64_t q_row, q_head;       // bytes
  char* out;
  int64_t out_row, out_head;   // bytes
  float* lse;
  int64_t lse_row;             // elements
  int heads, group, window;
  float scale_log2;            // scale * log2(e)
  char* work;                  // partial results
  void* records;               // 16 bytes a CTA
  unsigned* arrived;           // a counter a CTA, zero between calls; null: the join kernel follows
  int n_cta;                   // CTAs that share the tiles
};

struct Verify {
  int n_seq, n_rows, k_max, vocab;
  const int* row_start;
  const char* logits;
  int64_t logits_row;          // bytes
  int vec;                     // rows are 16-byte aligned
  const int* draft;
  const float* q;
  int64_t q_seq, q_step;
  const double* u;
  const float* temperature;
  const float* min_p;
  int* tokens;
  int* n_accepted;
  float* p_draft;
  int n_sms;
};

// dtype: ALM_F16 / ALM_BF16 / ALM_F32
cudaError_t launch_rope_append(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int dtype, int rope_dtype,
                               bool interleaved, int n_sms, int* err, cudaStream_t st);
cudaError_t launch_verify(const Verify& a, int dtype, cudaStream_t st);
size_t attn_paged_work_bytes(int n_sms, int head_dim);
cudaError_t paged_init_attrs();

}  // namespace alm

// Entry points of the operators of a batched step on device data
// (alm_kv_view, alm_rope_append, alm_attn_paged, alm_verify): argument checks
// on the host (arguments before the context), then one launch (attention of
// more than a few rows: two, the second joins partial results) on the context's
// stream.  Nothing here waits for the GPU or allocates, so the calls can be
// captured.
#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/androidllm_b200.h"
#include "paged.cuh"

int alm_internal_fail(int code, const char* msg);
int alm_internal_ctx_paged(alm_ctx* ctx, int* device, int* n_sms, cudaStream_t* stream, int** range_err);
int alm_internal_kv(alm_kv* kv, int layer, alm_paged_kv* view, const int32_t** table, int* rows, int* pages);

namespace alm {
cudaError_t launch_attn_paged_f16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st);
cudaError_t launch_attn_paged_bf16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st);
cudaError_t attn_paged_attrs_f16();
cudaError_t attn_paged_attrs_bf16();
bool attn_paged_tc_fits(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv);
cudaError_t launch_attn_paged_tc_f16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int nq, int* err,
                                     cudaStream_t st);
cudaError_t launch_attn_paged_tc_bf16(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int nq, int* err,
                                      cudaStream_t st);
cudaError_t attn_paged_tc_attrs_f16();
cudaError_t attn_paged_tc_attrs_bf16();
cudaError_t verify_init_attrs();

cudaError_t paged_init_attrs() {
  cudaError_t e = attn_paged_attrs_f16();
  if (e == cudaSuccess) e = attn_paged_attrs_bf16();
  if (e == cudaSuccess) e = attn_paged_tc_attrs_f16();
  if (e == cudaSuccess) e = attn_paged_tc_attrs_bf16();
  if (e == cudaSuccess) e = verify_init_attrs();
  return e;
}

// Sequences of more rows than this (tokens times the heads that share a K/V
// head) take the tcgen05 kernel.  Measured with 4 K/V heads of 128, mma.sync
// against tcgen05, us:
//   rows            16             32             40             64            128
//   8 x 4000    22.2 / 28.2    22.9 / 28.3    37.2 / 29.1    38.2 / 29.5    54.0 / 31.9
//   1 x 16000   16.9 / 24.6    17.8 / 24.7    25.8 / 25.2    26.4 / 25.4    34.8 / 26.1
//   64 x 1000   36.9 / 50.9    39.0 / 51.2    69.4 / 53.1    72.1 / 54.3   104.1 / 57.9
// (With its TMA producer at 64 rows too the mma.sync kernel takes as long as
// the tcgen05 kernel there, and 16% longer at 49 rows of 131 thousand
// positions.)  max_rows, the host's bound, picks one kernel for all sequences: a
// prompt chunk takes the single rows of its batch to the tcgen05 kernel too.
constexpr long long kTcMinRows = 32;

// Sequences of at most this many rows: the last of a unit's CTAs joins their
// results, a warp a row.  More rows, and few units of long sequences (many
// partials a row), are joined by a kernel of their own, which spreads them over
// more CTAs but costs a launch (4 us of the host's time).  Joined there against
// by the kernel, 8 rows a K/V head, 4 heads of 128: 3 x 100 7.4 / 9.1 us, 64 x
// 1000 36.3 / 36.8 us, 2 x 4000 14.0 / 13.5 us, 1 x 16000 20.0 / 17.0 us.  The
// host knows the table's width, not the lengths: few short sequences under a
// table of kLongTable positions or more pay for the second kernel.
constexpr long long kJoinHere = 8, kFewUnits = 8, kLongTable = 4096;

// The work area: a counter and a record a CTA, at the same place for every head
// dimension (the counters stay zero between calls), then two partial results a
// CTA, of the largest row block.
size_t attn_paged_head_bytes(int n_sms) { return (static_cast<size_t>(n_sms) * 20 + 255) / 256 * 256; }
size_t attn_paged_work_bytes(int n_sms, int head_dim) {
  return attn_paged_head_bytes(n_sms) + static_cast<size_t>(n_sms) * 2 * 256 * (head_dim + 2) * sizeof(float);
}
}  // namespace alm

using namespace alm;

namespace {

#define REQ(cond, msg)                                          \
  do {                                                          \
    if (!(cond)) return alm_internal_fail(ALM_ERR_ARG, msg);    \
  } while (0)
#define TRY(expr)                  \
  do {                             \
    const int rc_ = (expr);        \
    if (rc_ != ALM_OK) return rc_; \
  } while (0)

// The context's device for the call, the caller's afterwards.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int d) {
    if (cudaGetDevice(&before) != cudaSuccess) before = -1;
    if (before != d) cudaSetDevice(d);
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool vec8(int64_t stride) { return stride % 8 == 0; }

int cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return ALM_OK;
  return alm_internal_fail(ALM_ERR_CUDA, (std::string(what) + ": " + cudaGetErrorString(e)).c_str());
}

int check_kv(const alm_paged_kv* v, PagedKV* kv) {
  REQ(v && v->k_dev && v->v_dev, "null argument");
  REQ(v->dtype == ALM_F16 || v->dtype == ALM_BF16, "the cache's type must be fp16 or bf16");
  REQ(v->head_dim == 32 || v->head_dim == 64 || v->head_dim == 96 || v->head_dim == 128 || v->head_dim == 256,
      "head_dim must be 32, 64, 96, 128 or 256");
  REQ(v->kv_heads >= 1 && v->kv_heads <= 4096, "kv_heads must be in 1..4096");
  REQ(v->n_pages >= 1, "the pool must have a page");
  REQ(v->page_size >= 1 && v->page_size <= 65536, "page_size must be in 1..65536");
  REQ(aligned16(v->k_dev) && aligned16(v->v_dev), "K and V must be 16-byte aligned");
  kv->k = static_cast<char*>(v->k_dev);
  kv->v = static_cast<char*>(v->v_dev);
  kv->n_pages = v->n_pages;
  kv->page_size = v->page_size;
  kv->page_shift = (v->page_size & (v->page_size - 1)) == 0 ? __builtin_ctz(v->page_size) : -1;
  kv->kv_heads = v->kv_heads;
  kv->head_dim = v->head_dim;
  return ALM_OK;
}

int check_batch(const alm_seq_batch* v, SeqBatch* b) {
  REQ(v, "null argument");
  REQ(v->n_seq >= 0 && v->n_seq <= 4096, "n_seq must be in 0..4096");
  REQ(v->n_rows >= 0 && v->max_rows >= 0, "n_rows and max_rows must not be negative");
  REQ(v->n_seq == 0 || v->n_rows == 0 || (v->row_start_dev && v->kv_len_dev && v->page_table_dev), "null argument");
  REQ(aligned4(v->row_start_dev) && aligned4(v->kv_len_dev) && aligned4(v->page_table_dev) && aligned4(v->slots_dev),
      "the batch's arrays must be 4-byte aligned");
  REQ(v->table_rows >= (v->slots_dev ? 1 : v->n_seq), "the page table needs a row for every sequence");
  REQ(v->table_pages >= 0 && v->page_stride >= v->table_pages, "page_stride must be at least table_pages");
  b->n_seq = v->n_seq;
  b->n_rows = v->n_rows;
  b->max_rows = v->max_rows < 1 ? 1 : v->max_rows;
  b->table_rows = v->table_rows;
  b->table_pages = v->table_pages;
  b->page_stride = v->page_stride;
  b->row_start = v->row_start_dev;
  b->kv_len = v->kv_len_dev;
  b->table = v->page_table_dev;
  b->slots = v->slots_dev;
  return ALM_OK;
}

}  // namespace

extern "C" {

ALM_API int alm_kv_view(alm_kv* kv, int layer, alm_paged_kv* view, const int32_t** page_table_dev, int* table_rows,
                        int* table_pages) {
  return alm_internal_kv(kv, layer, view, page_table_dev, table_rows, table_pages);
}

ALM_API int alm_rope_append(alm_ctx* ctx, const alm_paged_kv* kv_, const alm_seq_batch* batch,
                            const alm_rope_append_args* v) {
  REQ(v, "null argument");
  PagedKV kv;
  SeqBatch b;
  TRY(check_kv(kv_, &kv));
  TRY(check_batch(batch, &b));
  REQ(v->heads >= 1 && v->heads <= 65536, "heads must be in 1..65536");
  const bool none = b.n_seq == 0 || b.n_rows == 0;   // nothing to do: the tensors may be empty
  REQ(none || (v->q_dev && v->k_dev && v->v_dev && v->q_out_dev && v->rope_dev), "null argument");
  REQ(aligned16(v->q_dev) && aligned16(v->k_dev) && aligned16(v->v_dev) && aligned16(v->q_out_dev) &&
          aligned16(v->rope_dev) && aligned16(v->q_norm_dev) && aligned16(v->k_norm_dev),
      "tensors must be 16-byte aligned");
  REQ(vec8(v->q_row) && vec8(v->q_head) && vec8(v->k_row) && vec8(v->k_head) && vec8(v->v_row) && vec8(v->v_head) &&
          vec8(v->qo_row) && vec8(v->qo_head),
      "row and head strides must be multiples of 8 elements");
  REQ(v->rope_dtype == ALM_F16 || v->rope_dtype == ALM_BF16 || v->rope_dtype == ALM_F32,
      "the rotation table's type must be fp16, bf16 or fp32");
  REQ(v->rope_rows >= 1, "the rotation table must have a row");
  REQ(v->rot_dim >= 16 && v->rot_dim <= kv.head_dim && v->rot_dim % 16 == 0,
      "rot_dim must be a multiple of 16, at most head_dim");
  REQ(v->eps >= 0.f && std::isfinite(v->eps), "eps must be finite and not negative");
  int device, n_sms, *err;
  cudaStream_t st;
  TRY(alm_internal_ctx_paged(ctx, &device, &n_sms, &st, &err));
  if (none) return ALM_OK;
  RopeAppend a;
  a.q = static_cast<const char*>(v->q_dev);
  a.k = static_cast<const char*>(v->k_dev);
  a.v = static_cast<const char*>(v->v_dev);
  a.q_row = v->q_row * 2, a.q_head = v->q_head * 2;
  a.k_row = v->k_row * 2, a.k_head = v->k_head * 2;
  a.v_row = v->v_row * 2, a.v_head = v->v_head * 2;
  a.q_out = static_cast<char*>(v->q_out_dev);
  a.qo_row = v->qo_row * 2, a.qo_head = v->qo_head * 2;
  a.heads = v->heads;
  a.q_norm = static_cast<const char*>(v->q_norm_dev);
  a.k_norm = static_cast<const char*>(v->k_norm_dev);
  a.eps = v->eps;
  a.rope = static_cast<const char*>(v->rope_dev);
  a.rope_rows = v->rope_rows;
  a.rot = v->rot_dim;
  OnDevice on(device);
  return cuda_status(launch_rope_append(a, b, kv, kv_->dtype, v->rope_dtype, v->interleaved != 0, n_sms, err, st),
                     "rope_append");
}

ALM_API int alm_attn_paged_work(alm_ctx* ctx, int heads, int kv_heads, int head_dim, size_t* bytes) {
  REQ(bytes, "null argument");
  REQ(kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  REQ(head_dim >= 1 && head_dim <= 256, "head_dim must be in 1..256");
  int device, n_sms, *err;
  cudaStream_t st;
  TRY(alm_internal_ctx_paged(ctx, &device, &n_sms, &st, &err));
  *bytes = attn_paged_work_bytes(n_sms, head_dim);
  return ALM_OK;
}

ALM_API int alm_attn_paged(alm_ctx* ctx, const alm_paged_kv* kv_, const alm_seq_batch* batch,
                           const alm_attn_paged_args* v) {
  REQ(v, "null argument");
  PagedKV kv;
  SeqBatch b;
  TRY(check_kv(kv_, &kv));
  TRY(check_batch(batch, &b));
  const bool none = b.n_seq == 0 || b.n_rows == 0;   // nothing to do: the tensors may be empty
  REQ(none || (v->q_dev && v->out_dev), "null argument");
  REQ(v->work_dev, "null argument");
  REQ(v->heads >= 1 && v->heads % kv.kv_heads == 0, "heads must be a multiple of kv_heads");
  REQ(v->heads / kv.kv_heads <= 128, "at most 128 query heads may share a K/V head");
  REQ(aligned16(v->q_dev) && aligned16(v->out_dev), "tensors must be 16-byte aligned");
  REQ(aligned4(v->lse_dev), "lse must be 4-byte aligned");
  REQ(vec8(v->q_row) && vec8(v->q_head) && vec8(v->out_row) && vec8(v->out_head),
      "row and head strides must be multiples of 8 elements");
  REQ(v->window >= 0, "window must not be negative");
  REQ(v->scale > 0.f && v->scale <= 1e30f, "scale must be positive and at most 1e30");
  REQ((reinterpret_cast<uintptr_t>(v->work_dev) & 255) == 0, "the work area must be 256-byte aligned");
  int device, n_sms, *err;
  cudaStream_t st;
  TRY(alm_internal_ctx_paged(ctx, &device, &n_sms, &st, &err));
  // (a row can be made again from its q, when its place in out has been written)
  REQ(none || v->q_dev != v->out_dev, "out_dev must not be q_dev");
  REQ(v->work_bytes >= attn_paged_work_bytes(n_sms, kv.head_dim), "the work area is too small (alm_attn_paged_work)");
  if (none) return ALM_OK;
  AttnPaged a;
  a.q = static_cast<const char*>(v->q_dev);
  a.q_row = v->q_row * 2, a.q_head = v->q_head * 2;
  a.out = static_cast<char*>(v->out_dev);
  a.out_row = v->out_row * 2, a.out_head = v->out_head * 2;
  a.lse = v->lse_dev;
  a.lse_row = v->lse_row;
  a.heads = v->heads;
  a.group = v->heads / kv.kv_heads;
  // a window as long as the table hides nothing (and the kernels' 32-bit
  // differences of a position and the window stay in range)
  const long long cap = std::min(static_cast<long long>(b.table_pages) * kv.page_size, 0x7fffff00ll);
  a.window = v->window >= cap ? 0 : v->window;
  a.scale_log2 = v->scale * 1.4426950408889634f;
  char* const work = static_cast<char*>(v->work_dev);
  a.records = work;
  a.work = work + attn_paged_head_bytes(n_sms);
  a.n_cta = n_sms;
  OnDevice on(device);
  const long long rows = static_cast<long long>(b.max_rows) * a.group;
  a.arrived = nullptr;
  const bool bf = kv_->dtype == ALM_BF16;
  if (rows > kTcMinRows && attn_paged_tc_fits(a, b, kv)) {
    const int nq = rows > 128 ? 2 : 1;
    return cuda_status(bf ? launch_attn_paged_tc_bf16(a, b, kv, nq, err, st)
                          : launch_attn_paged_tc_f16(a, b, kv, nq, err, st),
                       "attn_paged");
  }
  const bool few_long = b.n_seq * kv.kv_heads <= kFewUnits &&
                        static_cast<long long>(b.table_pages) * kv.page_size >= kLongTable;
  if (rows <= kJoinHere && kv.head_dim <= 128 && !few_long)   // (the 16-row kernel)
    a.arrived = reinterpret_cast<unsigned*>(work + static_cast<size_t>(n_sms) * 16);
  return cuda_status(bf ? launch_attn_paged_bf16(a, b, kv, err, st) : launch_attn_paged_f16(a, b, kv, err, st),
                     "attn_paged");
}

ALM_API int alm_verify(alm_ctx* ctx, const alm_verify_args* v) {
  REQ(v, "null argument");
  REQ(v->n_seq >= 0 && v->n_seq <= 65536, "n_seq must be in 0..65536");
  REQ(v->n_rows >= 0, "n_rows must not be negative");
  REQ(v->k_max >= 0 && v->k_max <= 31, "k_max must be in 0..31");
  REQ(v->vocab >= 1 && v->vocab <= (1 << 24), "vocab must be in 1..16777216");
  REQ(v->logits_dtype == ALM_F16 || v->logits_dtype == ALM_BF16 || v->logits_dtype == ALM_F32,
      "the logits' type must be fp16, bf16 or fp32");
  REQ(v->n_seq == 0 || (v->row_start_dev && v->uniforms_dev && v->temperature_dev && v->tokens_dev && v->n_accepted_dev),
      "null argument");
  REQ(v->n_rows == 0 || v->logits_dev, "null argument");
  REQ(v->n_seq == 0 || v->k_max == 0 || v->draft_tokens_dev, "null argument");
  REQ(v->logits_row >= v->vocab || v->n_rows <= 1, "logits_row must be at least vocab");
  const int item = v->logits_dtype == ALM_F32 ? 4 : 2;
  REQ((reinterpret_cast<uintptr_t>(v->logits_dev) % item) == 0, "logits must be aligned to their type");
  REQ(aligned4(v->row_start_dev) && aligned4(v->draft_tokens_dev) && aligned4(v->draft_probs_dev) &&
          aligned4(v->temperature_dev) && aligned4(v->min_p_dev) && aligned4(v->tokens_dev) &&
          aligned4(v->n_accepted_dev) && aligned4(v->p_draft_dev) && (reinterpret_cast<uintptr_t>(v->uniforms_dev) & 7) == 0,
      "arrays must be aligned to their type");
  int device, n_sms, *err;
  cudaStream_t st;
  TRY(alm_internal_ctx_paged(ctx, &device, &n_sms, &st, &err));
  if (v->n_seq == 0) return ALM_OK;
  Verify a;
  a.n_seq = v->n_seq, a.n_rows = v->n_rows, a.k_max = v->k_max, a.vocab = v->vocab;
  a.row_start = v->row_start_dev;
  a.logits = static_cast<const char*>(v->logits_dev);
  a.logits_row = v->logits_row * item;
  a.vec = aligned16(v->logits_dev) && (a.logits_row % 16 == 0);
  a.draft = v->draft_tokens_dev;
  a.q = v->draft_probs_dev;
  a.q_seq = v->q_seq, a.q_step = v->q_step;
  a.u = v->uniforms_dev;
  a.temperature = v->temperature_dev;
  a.min_p = v->min_p_dev;
  a.tokens = v->tokens_dev;
  a.n_accepted = v->n_accepted_dev;
  a.p_draft = v->p_draft_dev;
  a.n_sms = n_sms;
  OnDevice on(device);
  return cuda_status(launch_verify(a, v->logits_dtype, st), "verify");
}

}  // extern "C"

// Pages of K and V through TMA: the copies, bounded waits on their barriers and
// the tensor maps, for the paged attention kernels.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "tc.cuh"

namespace alm {

ALM_DEV void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
      : "memory");
}
ALM_DEV void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}
// One lane of a converged warp.  (With this instruction, unlike a test of the
// lane number, the compiler knows that one thread runs what follows.)
ALM_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
// Named barrier that also tells whether any thread's p holds.
ALM_DEV bool bar_or(int id, int n, bool p) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n bar.red.or.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"(id), "r"(n), "r"(p ? 1u : 0u) : "memory");
  return r != 0;
}
ALM_DEV void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }
ALM_DEV void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// What the waits of a CTA have in common.  dead: one ran out, and everybody
// leaves.  beat: counts the steps of work that no barrier shows (results with
// infinities made again); a wait's time starts anew with each.
struct Waits {
  int dead, beat;
};
// The rest of a wait whose first look failed: true when the phase completed.
ALM_DEV bool slow_wait(uint64_t* bar, uint32_t parity, volatile Waits* w, int* err) {
  unsigned long long t0 = global_ns();
  int beat = w->beat;
  for (unsigned i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait_suspend(bar, parity)) return true;
    if (w->dead) return false;
    if (w->beat != beat) {
      beat = w->beat;
      t0 = global_ns();
      i = 0;
    }
    if (global_ns() - t0 > kWaitLimitNs) break;
  }
  w->dead = 1;
  *err = 2;
  return false;
}

// One page piece of a K or V tile that a lane loads: pieces of box_rows rows and
// 64 columns.  The first row of its box in the pool's rows of head_dim
// elements, or a row behind the pool (which reads zeros) for a piece
// behind the sequence's end or of a page outside the pool (bad).
ALM_DEV int piece_row(const PagedKV& kv, const int* pages, int kv_head, int n_kv, int pos, bool on, bool& bad) {
  const bool in = on && pos < n_kv;
  const int pi = page_of(kv, pos);
  const int page = in && pages ? __ldg(pages + pi) : -1;
  const bool ok = page >= 0 && page < kv.n_pages;
  bad |= in && !ok;
  return ok ? (page * kv.kv_heads + kv_head) * kv.page_size + pos - pi * kv.page_size
            : kv.n_pages * kv.kv_heads * kv.page_size;
}

// ---- host --------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 cu_tensor_map_encoder();

// K or V as rows of head_dim elements, read as boxes of box_rows rows x 64 columns.
template <typename T>
bool encode_pages(CUtensorMap* map, const char* p, const PagedKV& kv, int box_rows) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = cu_tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(kv.head_dim),
                        static_cast<cuuint64_t>(kv.n_pages) * kv.kv_heads * kv.page_size};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(kv.head_dim) * sizeof(T)};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, std::is_same<T, half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
             const_cast<char*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of a TMA box: the largest power of two that divides the page, at most a tile.
inline int page_box_rows(const PagedKV& kv) { return std::min(kv.page_size & -kv.page_size, 128); }

// Pages that TMA reads: whole 8-row pieces (the swizzle's period), 64 or 128
// columns, and a row index that fits a TMA coordinate.
inline bool tma_pages(const PagedKV& kv) {
  return (kv.head_dim == 64 || kv.head_dim == 128) && kv.page_size % 8 == 0 &&
         static_cast<long long>(kv.n_pages) * kv.kv_heads * kv.page_size < (1ll << 31) - 256;
}

}  // namespace alm

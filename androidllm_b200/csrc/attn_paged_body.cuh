// Attention of a pass's new rows over the paged cache (alm_attn_paged): the
// mma.sync kernel for few rows a sequence, and the join of the partial results
// of units cut between CTAs (by the last of them, or by a kernel).
// Instantiated for fp16 and bf16 in attn_paged_f16.cu and attn_paged_bf16.cu.
//
//   o_i = sum_j exp(c (s_ij - m_i)) v_j / sum_j exp(c (s_ij - m_i)),  s = q.k,
//   c = scale, over the positions j that row i sees; m_i = max_j s_ij.
//
// One pass over K and V with a running maximum and sum (rescaled when the
// maximum grows).  A decode or verify pass reads far more K/V bytes than
// it computes on, so HBM bounds it: the CTAs share all tiles evenly
// (attn_sched.cuh), each streams its run of tiles through a ring of
// shared-memory stages filled across unit borders, and the rows
// of the query heads that share a K/V head are one matrix operand, so K and V
// are read once for all of them.
//
// CTA: 8 warps as WM x WK.  Warp (wm, wk) computes rows 16 wm .. 16 wm + 15
// on the wk-th slice of each tile, with its own running statistics;
// the WK slices are merged at a unit's end through the stage just consumed.
//
// 64 sequences of 1 .. 8191 positions, one token each (28 heads over 4 K/V
// heads of 128, 127 MB): 39 us, 3.2 TB/s; filled by cp.async from the computing
// warps it was 52 us.  The stream itself runs near HBM's rate; the start
// (lengths, shares, the first tile), the units' merges and the join take the
// rest.  One sequence of 700: 11 us, all of it these latencies.
#pragma once
#include <algorithm>

#include "attn_paged_tma.cuh"
#include "attn_sched.cuh"

namespace alm {

constexpr int kPagedThreads = 256;
constexpr int kJoinThreads = 128;
constexpr int kPagedWarps = kPagedThreads / kWarp;
// A weight is 2^(c s - round(c m)), one multiply-add a score.  What round()
// leaves scales a chunk's weights by up to 2^(2^-24 c m): by 2^-14 at this |c m|,
// an eighth of fp16's half step.  Beyond it (at 2^28 every weight would be 0 or
// infinite) m is taken off the scores first: c (s - m) is 0 at the maximum
// whatever c is.
constexpr float kFarScore = 1024.f;

template <typename T>
struct Elem;
template <>
struct Elem<half> {
  ALM_DEV static uint32_t pack(float a, float b) {
    half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  ALM_DEV static float up(half h) { return __half2float(h); }
  ALM_DEV static half down(float f) { return __float2half_rn(f); }
  ALM_DEV static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma16816(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <>
struct Elem<__nv_bfloat16> {
  ALM_DEV static uint32_t pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  ALM_DEV static float up(__nv_bfloat16 h) { return __bfloat162float(h); }
  ALM_DEV static __nv_bfloat16 down(float f) { return __float2bfloat16_rn(f); }
  ALM_DEV static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

ALM_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

ALM_DEV void ldmatrix_x4_trans(uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a) : "memory");
}
ALM_DEV void ldmatrix_x4_at(uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a) : "memory");
}
// 16 bytes, or zeros where `bytes` is 0
ALM_DEV void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
ALM_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
ALM_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// TMA: stages filled by a producer warp, each 128-byte column group of a tile
// swizzled as TMA does; else (other head dimensions, pages that are not whole
// 8-row pieces) by cp.async from all threads, with padded rows.
template <int HD, int WM, bool TMA>
struct PagedShape {
  static constexpr int kThreads = kPagedThreads + (TMA ? kWarp : 0);
  static constexpr int kTile = HD > 128 ? 64 : 128;        // positions a tile
  static constexpr int kWK = kPagedWarps / WM;
  static constexpr int kNP = kTile / kWK;                  // positions a warp and tile
  static constexpr int kChunk = kNP < 64 ? kNP : 64;       // ... and step
  static constexpr int kRows = 16 * WM;
  // rows padded by 16 bytes: an odd number of 16-byte units, so that the 8
  // rows of an ldmatrix matrix lie in 8 different bank groups
  static constexpr int kPitch = TMA ? HD * 2 : HD * 2 + 16;
  static constexpr int kTileBytes = kTile * kPitch;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = HD <= 64 ? 6 : HD <= 96 ? 4 : 3;
  // merge of the WK slices in one stage: 128 fp32 rows of HD / kPasses columns,
  // padded by 8, or groups of 8 columns exchanged by the row's number
  static constexpr int kPasses = HD > 128 ? 4 : 1;
  static constexpr int kMergePitch = TMA ? HD : HD / kPasses + 8;
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes + (TMA ? 1024 : 0);
  // byte offset of 16-byte unit c of row r in a tile
  ALM_DEV static uint32_t unit(int r, int c) {
    if constexpr (TMA) return (c / 8) * (kTile * 128) + r * 128 + ((c ^ r) & 7) * 16;
    else return r * kPitch + c * 16;
  }
  // element offset of column c of row r in the merge
  ALM_DEV static int merge(int r, int c) { return r * kMergePitch + (TMA ? c ^ (r & 7) * 8 : c); }
  static_assert(128 * kMergePitch * 4 <= kStageBytes, "merge fits a stage");
  static_assert(kNP >= 16, "a warp's slice holds a k16 step");
};

// Partial result of a CTA's first (which = 0) or last (1) unit: kRows rows of
// HD fp32 sums, then their maxima, then their sums of weights.
template <int HD>
ALM_DEV float* partial_at(char* work, int rows, int cta, int which) {
  return reinterpret_cast<float*>(work) + (static_cast<size_t>(cta) * 2 + which) * rows * (HD + 2);
}

// What a CTA leaves for the join: the unit that it began and did not finish as
// (number of partials, first packed row, tokens, K/V head); 0 partials: none.
ALM_DEV int4* join_record(const AttnPaged& a, int cta) { return reinterpret_cast<int4*>(a.records) + cta; }
ALM_DEV int4 record_of(const Unit& u, int cta, int n_cta, long long total) {
  // the CTA of the unit's last place p: the largest i with total i / n <= p
  const int last = static_cast<int>(((u.start + u.n_tile) * n_cta - 1) / total);
  return make_int4(last - cta + 1, u.row0, u.n_tok, u.h);
}

// x where it is infinite or NaN, else 0
ALM_DEV float not_finite(float x) { return fabsf(x) < __int_as_float(0x7f800000) ? 0.f : x; }

// V consecutive fp32 values behind L1 (another SM wrote them).
template <int V>
ALM_DEV void load_row(const float* p, float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(p + i));
      v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
  } else if constexpr (V == 2) {
    const float2 x = __ldcg(reinterpret_cast<const float2*>(p));
    v[0] = x.x, v[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __ldcg(p + i);
  }
}

// One row of the unit that CTA `cta` began, by a warp: the sum of its n partial
// results in CTA order, kDeep of them under way at a time (left to the compiler
// two or three were: 8 x 5 rows 14.4 us instead of 11.8).
template <int HD, int ROWS, int kDeep>
ALM_DEV void join_part(const AttnPaged& a, int cta, int n, int row, float& m, float& l, float (&o)[HD / 32]) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x % kWarp;
  auto part = [&](int i) { return partial_at<HD>(a.work, ROWS, cta + i, i == 0 ? 1 : 0); };
  m = kNegInf;
  for (int i = lane; i < n; i += kWarp) m = fmaxf(m, __ldcg(part(i) + ROWS * HD + row));
  m = warp_max(m);
  const float base = m == kNegInf ? 0.f : m;
  l = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.f;
  for (int i0 = 0; i0 < n; i0 += kWarp) {
    float w = 0.f, li = 0.f;
    if (i0 + lane < n) {
      const float* p = part(i0 + lane) + ROWS * HD;
      w = ex2((__ldcg(p + row) - base) * a.scale_log2);
      li = __ldcg(p + ROWS + row);
    }
    const int k = min(kWarp, n - i0);
    for (int i = 0; i < k; i += kDeep) {
      float v[kDeep][V];
#pragma unroll
      for (int q = 0; q < kDeep; ++q)
        if (i + q < k) load_row<V>(part(i0 + i + q) + row * HD + lane * V, v[q]);
#pragma unroll
      for (int q = 0; q < kDeep; ++q) {
        if (i + q >= k) break;
        const float f = __shfl_sync(0xffffffffu, w, i + q);
        l = fmaf(__shfl_sync(0xffffffffu, li, i + q), f, l);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = fmaf(v[q][j], f, o[j]);
      }
    }
  }
  // an infinite part stays one, however small its weight
  bool odd = false;
#pragma unroll
  for (int j = 0; j < V; ++j) odd |= o[j] != o[j];
  if (__any_sync(0xffffffffu, odd && l == l)) {
    float x[V] = {};
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      float v[V];
      load_row<V>(part(i) + row * HD + lane * V, v);
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] += not_finite(v[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = x[j] != 0.f ? x[j] : o[j];
  }
}
template <typename T, int HD>
ALM_DEV void join_store(const AttnPaged& a, int row, int head, float m, float l, const float (&o)[HD / 32]) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x % kWarp;
  const float inv = m == kNegInf && l == 0.f ? 0.f : 1.f / l;
  T* dst = reinterpret_cast<T*>(a.out + row * a.out_row + head * a.out_head) + lane * V;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      reinterpret_cast<uint32_t*>(dst)[j / 2] = Elem<T>::pack(o[j] * inv, o[j + 1] * inv);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) dst[j] = Elem<T>::down(o[j] * inv);
  }
  if (a.lse && lane == 0)
    a.lse[row * a.lse_row + head] =
        m == kNegInf ? kNegInf : (m * a.scale_log2 + log2f(l)) * 0.693147180559945309f;
}
// All rows of a unit by n_warps warps, a warp a row.  A unit's ROWS rows are
// blocks of BLK rows, whole tokens each.
template <typename T, int HD, int ROWS, int BLK, int kDeep>
ALM_DEV void join_unit(const AttnPaged& a, int cta, int4 rec, int warp, int n_warps) {
  const int tq = BLK / a.group;
  for (int row = warp; row < ROWS; row += n_warps) {
    const int tk = row % BLK / a.group, tok = row / BLK * tq + tk;
    if (tk >= tq || tok >= rec.z) continue;
    float m, l, o[HD / 32];
    join_part<HD, ROWS, kDeep>(a, cta, rec.x, row, m, l, o);
    join_store<T, HD>(a, rec.y + tok, rec.w * a.group + row % BLK - tk * a.group, m, l, o);
  }
}
// (out of line: the attention kernel needs its registers)
template <typename T, int HD, int ROWS>
__device__ __noinline__ void join_unit_here(const AttnPaged& a, int cta, int4 rec, int warp) {
  join_unit<T, HD, ROWS, ROWS, 4>(a, cta, rec, warp, kPagedWarps);
}

// ---- infinities and NaN in V ----------------------------------------------------
// A hidden position's weight is 0, and 0 times an infinity or NaN spoils its
// column of the matrix product for rows that do not see it.  So a row whose sums
// are not finite though its weights are is looked at again: a column of it in
// which it sees an infinity or NaN is their sum (their weights are positive,
// however small), and one in which it sees none is summed by the formula.  64
// decodes over 2000 to 7670 positions, one of them with an infinity: 529 us
// instead of 122.

// A lane's V consecutive columns of a K or V row.
template <typename T, int V>
struct Columns {
  static constexpr int kWords = V % 2 ? V : V / 2;
  alignas(V == 8 ? 16 : V == 4 ? 8 : 4) uint32_t w[kWords];
  ALM_DEV void load(const T* row) {
    const T* p = row + threadIdx.x % kWarp * V;
    if constexpr (V == 8) *reinterpret_cast<uint4*>(w) = __ldg(reinterpret_cast<const uint4*>(p));
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(w) = __ldg(reinterpret_cast<const uint2*>(p));
    else if constexpr (V == 2) w[0] = __ldg(reinterpret_cast<const unsigned*>(p));
    else
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __ldg(reinterpret_cast<const unsigned short*>(p) + i);
  }
  ALM_DEV float at(int i) const {
    const unsigned short h = static_cast<unsigned short>(V % 2 ? w[i] : i % 2 ? w[i / 2] >> 16 : w[i / 2]);
    return Elem<T>::up(*reinterpret_cast<const T*>(&h));
  }
  // some bit is set where a value's exponent is all ones (infinity or NaN)
  ALM_DEV uint32_t odd() const {
    constexpr uint32_t kExp = std::is_same<T, half>::value ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t kOne = std::is_same<T, half>::value ? 0x04000400u : 0x00800080u;
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) r |= (w[i] & kExp) + kOne;
    return r & 0x80008000u;
  }
};

// Byte offset of position p in K and V, -1 behind `end` and for pages outside the
// pool.  (A lane finds a position's, and a warp then takes them from its lanes.)
template <typename T>
ALM_DEV long long place_at(const PagedKV& kv, const int* pages, int kv_head, int p, int end) {
  if (p >= end || pages == nullptr) return -1;
  const int pi = page_of(kv, p), page = __ldg(pages + pi);
  if (page < 0 || page >= kv.n_pages) return -1;
  return static_cast<long long>(kv_offset(kv, page, kv_head, p - pi * kv.page_size) * sizeof(T));
}

// Adds the infinities and NaN of V at positions [p0, p1) to x.  By a warp.
template <typename T, int HD>
ALM_DEV void gather_not_finite(const PagedKV& kv, const int* pages, int kv_head, int p0, int p1, float (&x)[HD / 32],
                               volatile Waits* waits) {
  constexpr int V = HD / 32, kDeep = 16;
  const int lane = threadIdx.x % kWarp;
  long long next = place_at<T>(kv, pages, kv_head, p0 + lane, p1);
  for (int p = p0; p < p1; p += kWarp) {
    const long long mine = next;
    next = place_at<T>(kv, pages, kv_head, p + kWarp + lane, p1);
    for (int j = 0; j < kWarp && p + j < p1; j += kDeep) {
      // (the loads one after the other, so that all are under way together)
      long long at[kDeep];
      Columns<T, V> v[kDeep];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) at[d] = __shfl_sync(0xffffffffu, mine, j + d);
#pragma unroll
      for (int d = 0; d < kDeep; ++d) v[d].load(reinterpret_cast<const T*>(kv.v + max(at[d], 0ll)));
      uint32_t odd = 0;
#pragma unroll
      for (int d = 0; d < kDeep; ++d) odd |= at[d] < 0 ? 0 : v[d].odd();
      if (__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] += at[d] < 0 ? 0.f : not_finite(v[d].at(i));
      }
    }
    if (p % 4096 < kWarp) waits->beat = waits->beat + 1;
  }
}

// Adds 2^(c (s - m)) inv V, V's infinities and NaN left out, at positions [p0, p1)
// to o.  By a warp: the scores a position a lane, the sums V columns a lane.
template <typename T, int HD>
ALM_DEV void sum_by_formula(const AttnPaged& a, const PagedKV& kv, const int* pages, int kv_head, const T* q, int p0, int p1,
                            float m, float inv, float (&o)[HD / 32], volatile Waits* waits) {
  constexpr int V = HD / 32, kDeep = 8;
  const int lane = threadIdx.x % kWarp;
  for (int p = p0; p < p1; p += kWarp) {
    const long long mine = place_at<T>(kv, pages, kv_head, p + lane, p1);
    float w = 0.f;
    if (mine >= 0) {
      const uint4* k = reinterpret_cast<const uint4*>(kv.k + mine);
      float s = 0.f;
#pragma unroll 8
      for (int c = 0; c < HD / 8; ++c) {
        const uint4 x = __ldg(k + c), y = __ldg(reinterpret_cast<const uint4*>(q) + c);
        const T *xs = reinterpret_cast<const T*>(&x), *ys = reinterpret_cast<const T*>(&y);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(Elem<T>::up(xs[i]), Elem<T>::up(ys[i]), s);
      }
      w = ex2((s - m) * a.scale_log2) * inv;
    }
    for (int j = 0; j < kWarp && p + j < p1; j += kDeep) {
      long long at[kDeep];
      Columns<T, V> v[kDeep];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) at[d] = max(__shfl_sync(0xffffffffu, mine, j + d), 0ll);
#pragma unroll
      for (int d = 0; d < kDeep; ++d) v[d].load(reinterpret_cast<const T*>(kv.v + at[d]));
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const float f = __shfl_sync(0xffffffffu, w, j + d);   // 0 where there is no page
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float y = v[d].at(i);
          o[i] = fmaf(f, fabsf(y) < __int_as_float(0x7f800000) ? y : 0.f, o[i]);
        }
      }
    }
    if (p % 1024 < kWarp) waits->beat = waits->beat + 1;
  }
}

// Rows r0 + step i of a block (bits i of todo; first packed row row0, first
// position pos0), of which the CTA has summed positions [p0, p1) and which lie in
// `part` (or, if that is null, in the output): what is not finite in them
// is put right.  Lane i brings its row's m and inv (1 / l, or 1 in a partial
// result).  By a warp; what all the rows see is read once for them.
template <typename T, int HD>
__device__ __noinline__ void mend_rows(const AttnPaged& a_, const PagedKV& kv_, const int* pages, int kv_head, int row0, int pos0,
                                       int r0, int step, unsigned todo, float m, float inv, int p0, int p1, float* part,
                                       volatile Waits* waits) {
  constexpr int V = HD / 32;
  if (todo == 0) return;
  const AttnPaged a = a_;   // (in registers: the loops would load them from the arguments every time)
  const PagedKV kv = kv_;
  const int lane = threadIdx.x % kWarp;
  auto pos_of = [&](int i) { return pos0 + (r0 + step * i) / a.group; };
  auto from = [&](int pos) { return max(p0, a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0); };
  auto upto = [&](int pos) { return min(p1, pos + 1); };
  int c0 = from(pos_of(31 - __clz(todo))), c1 = upto(pos_of(__ffs(todo) - 1));   // seen by all of them
  if (c0 >= c1) c0 = c1 = p1;
  float all[V];
#pragma unroll
  for (int i = 0; i < V; ++i) all[i] = 0.f;
  gather_not_finite<T, HD>(kv, pages, kv_head, c0, c1, all, waits);
  for (; todo; todo &= todo - 1) {
    const int src = __ffs(todo) - 1, r = r0 + step * src, tok = r / a.group, pos = pos0 + tok;
    const int head = kv_head * a.group + r - tok * a.group, s0 = from(pos), s1 = upto(pos);
    float x[V], o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = all[i], o[i] = 0.f;
    gather_not_finite<T, HD>(kv, pages, kv_head, s0, min(s1, c0), x, waits);
    gather_not_finite<T, HD>(kv, pages, kv_head, max(s0, c1), s1, x, waits);
    T* dst = reinterpret_cast<T*>(a.out + (row0 + tok) * a.out_row + head * a.out_head) + lane * V;
    float* dst32 = part ? part + r * HD + lane * V : nullptr;
    bool open = false;
    unsigned bad = 0;   // columns that are not finite
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (not_finite(part ? dst32[i] : Elem<T>::up(dst[i])) != 0.f) {
        bad |= 1u << i;
        open |= x[i] == 0.f;
      }
    const float mr = __shfl_sync(0xffffffffu, m, src), ir = __shfl_sync(0xffffffffu, inv, src);
    if (__any_sync(0xffffffffu, open))
      sum_by_formula<T, HD>(a, kv, pages, kv_head, reinterpret_cast<const T*>(a.q + (row0 + tok) * a.q_row + head * a.q_head),
                            s0, s1, mr == kNegInf ? 0.f : mr, ir, o, waits);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = x[i] != 0.f ? x[i] : o[i];
      if (x[i] == 0.f && !(bad >> i & 1)) continue;
      if (part) dst32[i] = y;
      else dst[i] = Elem<T>::down(y);
    }
  }
}

// Two packed values, zero where they are not finite.  (attn_paged_tc_body.cuh)
template <typename T>
ALM_DEV uint32_t finite_only(uint32_t x) {
  constexpr uint32_t kExp = std::is_same<T, half>::value ? 0x7c00u : 0x7f80u;   // all ones: infinity or NaN
  if ((x & kExp) == kExp) x &= 0xffff0000u;
  if ((x >> 16 & kExp) == kExp) x &= 0xffffu;
  return x;
}

template <typename T, int HD, int WM, bool TMA>
__global__ void __launch_bounds__(PagedShape<HD, WM, TMA>::kThreads, 1)
attn_paged_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                  const __grid_constant__ AttnPaged a, const __grid_constant__ SeqBatch b,
                  const __grid_constant__ PagedKV kv, int box_rows, int* err) {
  using S = PagedShape<HD, WM, TMA>;
  constexpr int kTile = S::kTile, kWK = S::kWK, kNP = S::kNP, kChunk = S::kChunk, kRows = S::kRows;
  extern __shared__ __align__(128) char smem_raw[];
  char* const smem = TMA ? smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023) : smem_raw;
  __shared__ SchedShared sched;
  __shared__ uint64_t full[S::kStages], empty[S::kStages];
  __shared__ Waits waits_;
  __shared__ float st_m[kWK][kRows], st_l[kWK][kRows];
  __shared__ float row_m[kRows], row_l[kRows];
  __shared__ int row_bad[kRows];
  __shared__ int joins;

  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int wm = warp % WM, wk = warp / WM, g = lane / 4, t4 = lane % 4;
  const int tpu = kRows / a.group;
  const int cta = blockIdx.x;
  // barrier of the eight computing warps
  auto sync = [] {
    if constexpr (TMA) bar_sync(1, kPagedThreads);
    else __syncthreads();
  };
  if (tid == 0) waits_.dead = waits_.beat = 0;
  if (TMA && tid == kPagedThreads) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], kPagedWarps);
    fence_mbar_init();
  }
  if (!TMA || warp < kPagedWarps)
    sched_init<kTile>(
        b, kv, tpu, a.window, sched, err,
        [&](long long total) {
          const int n = static_cast<int>(min(static_cast<long long>(a.n_cta), total));
          return cta < n ? share(total, cta, n) : -1ll;
        },
        sync);
  if (TMA) __syncthreads();
  const long long total = sched.total;
  const int n_cta = static_cast<int>(min(static_cast<long long>(a.n_cta), total));
  if (tid == 0) *join_record(a, cta) = make_int4(0, 0, 0, 0);
  if (cta >= n_cta) return;
  const long long x0 = share(total, cta, n_cta), x1 = share(total, cta + 1, n_cta);

  Unit u = unit_at<kTile>(b, kv, tpu, a.window, sched.found_seq, sched.found_at, x0);
  int t = u.from(x0), tb = u.upto(x1);   // this CTA's tiles of the unit: [t, tb)
  if (t >= tb) return;                   // only places without a tile
  // the loader's walk, kStages - 1 tiles ahead of the computation's
  Unit lu = u;
  int lt = t, ltb = tb;
  const uint32_t smem0 = smem_addr(smem);
  volatile Waits* waits = &waits_;
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {   // the same answer for the whole warp
    const bool ok = mbar_try_wait(bar, parity & 1) || slow_wait(bar, parity & 1, waits, err);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  if (TMA && warp == kPagedWarps) {
    // the producer: a page piece of K and of V a lane (128 / 8 pieces of 2 column groups at most)
    constexpr int kGroups = HD < 64 ? 1 : HD / 64;   // 128-byte column groups
    const int n_box = kTile / box_rows * kGroups, box = lane / kGroups, c = lane % kGroups;
    bool bad = false, quit = false;
    for (uint32_t n = 0; !quit; ++n) {
      const int y = piece_row(kv, lu.pages, lu.h, lu.n_kv, (lu.t0 + lt) * kTile + box * box_rows, lane < n_box, bad);
      const uint32_t st = n % S::kStages;
      if (!wait_warp(&empty[st], n / S::kStages + 1)) {
        quit = true;
        break;
      }
      if (lane == 0) mbar_expect_tx(&full[st], S::kStageBytes);
      __syncwarp();
      if (lane < n_box) {
        const uint32_t dst = smem0 + st * S::kStageBytes + c * (kTile * 128) + box * box_rows * 128;
        tma_2d(dst, &k_map, c * 64, y, &full[st]);
        tma_2d(dst + S::kTileBytes, &v_map, c * 64, y, &full[st]);
      }
      __syncwarp();
      if (++lt == ltb) {
        if (!lu.more(x1)) break;
        next_unit<kTile>(b, kv, tpu, a.window, lu);
        lt = 0;
        ltb = lu.upto(x1);
      }
    }
    if (bad) *err = 1;
    if (quit)   // no copy is in flight when the CTA leaves
      for (int i = 0; i < S::kStages; ++i) mbar_wait(&full[i], 0), mbar_wait(&full[i], 1);
    return;
  }
  constexpr int kUnits16 = HD / 8;   // 16-byte units of a K or V row
  bool bad_page = false;

  auto load_tile = [&](int stage) {
    if (lt < ltb) {
      const uint32_t dst = smem0 + stage * S::kStageBytes;
      const int base = (lu.t0 + lt) * kTile;
      constexpr int kIter = kTile * kUnits16 / kPagedThreads;
      // the page numbers first, all in flight together
      int page[kIter];
#pragma unroll
      for (int i = 0; i < kIter; ++i) {
        const int pos = base + (tid + i * kPagedThreads) / kUnits16;
        page[i] = pos < lu.n_kv && lu.pages ? __ldg(lu.pages + page_of(kv, pos)) : -1;
      }
#pragma unroll
      for (int i = 0; i < kIter; ++i) {
        const int idx = tid + i * kPagedThreads;
        const int r = idx / kUnits16, c = idx % kUnits16;
        const int pos = base + r;
        const bool ok = page[i] >= 0 && page[i] < kv.n_pages;
        bad_page |= !ok && pos < lu.n_kv;
        const size_t off =
            (ok ? kv_offset(kv, page[i], lu.h, pos - page_of(kv, pos) * kv.page_size) + c * 8 : 0) * sizeof(T);
        cp_async16(dst + S::unit(r, c), kv.k + off, ok ? 16 : 0);
        cp_async16(dst + S::kTileBytes + S::unit(r, c), kv.v + off, ok ? 16 : 0);
      }
      if (++lt == ltb && lu.more(x1)) {
        next_unit<kTile>(b, kv, tpu, a.window, lu);
        lt = 0;
        ltb = lu.upto(x1);
      }
    }
    cp_async_commit();
  };
  if (!TMA) {
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) load_tile(i);
  }

  int t_first = t;   // first tile of the unit computed here
  uint32_t qf[HD / 16][4];
  float o[HD / 8][4];
  float m[2], l[2];
  int hi[2];
  auto begin_unit = [&] {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = wm * 16 + g + 8 * j;
      const int tok = row / a.group, hh = row - tok * a.group;
      const bool live = tok < u.n_tok;
      hi[j] = live ? max(u.pos0 + tok, -1) : -1;
      const char* q = a.q + (u.row0 + tok) * a.q_row + (u.h * a.group + hh) * a.q_head;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        qf[k][j] = live ? __ldg(reinterpret_cast<const unsigned*>(q + (16 * k + 2 * t4) * 2)) : 0u;
        qf[k][j + 2] = live ? __ldg(reinterpret_cast<const unsigned*>(q + (16 * k + 8 + 2 * t4) * 2)) : 0u;
      }
      m[j] = kNegInf;
      l[j] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[n][j] = 0.f;
  };
  begin_unit();

  int stage = 0;
  uint32_t round = 0;
  auto next_stage = [&] {
    if (++stage == S::kStages) stage = 0, round ^= 1;
  };
  for (;;) {
    if constexpr (TMA) {
      wait_warp(&full[stage], round);
    } else {
      cp_async_wait<S::kStages - 2>();
      __syncthreads();
      load_tile(stage == 0 ? S::kStages - 1 : stage - 1);
    }
    const uint32_t kb = smem0 + stage * S::kStageBytes, vb = kb + S::kTileBytes;
    if constexpr (TMA) {
      // The sequence ends in this tile, and its last page piece goes on behind
      // it: those rows hold anything, and a zero weight times NaN is NaN.  Each
      // warp clears what it reads.
      const int end = u.n_kv - (u.t0 + t) * kTile;   // rows of the tile that exist
      if (end < (wk + 1) * kNP) {
        const int z0 = max(end, wk * kNP);
        for (int i = lane; i < ((wk + 1) * kNP - z0) * kUnits16; i += kWarp)
          *reinterpret_cast<uint4*>(smem + stage * S::kStageBytes + S::kTileBytes +
                                    S::unit(z0 + i / kUnits16, i % kUnits16)) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();   // before the stage is filled again
        __syncwarp();
      }
    }
#pragma unroll 1
    for (int c0 = 0; c0 < kNP; c0 += kChunk) {
      const int r0 = wk * kNP + c0;                    // first row of the chunk in the stage
      const int p0 = (u.t0 + t) * kTile + r0;          // ... and its position
      float s[kChunk / 8][4];
#pragma unroll
      for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int n = 0; n < kChunk / 8; n += 2) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4_at(b0, b1, b2, b3,
                         kb + S::unit(r0 + n * 8 + (lane & 7) + ((lane >> 4) & 1) * 8, 2 * k + ((lane >> 3) & 1)));
          Elem<T>::mma(s[n], qf[k], b0, b1);
          Elem<T>::mma(s[n + 1], qf[k], b2, b3);
        }
      // positions that some row of the block does not see
      if (p0 + kChunk - 1 > u.pos0 || (a.window > 0 && p0 <= max(u.pos0 + u.n_tok - 1, -1) - a.window)) {
#pragma unroll
        for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int p = p0 + n * 8 + 2 * t4 + (j & 1);
            const bool seen = p <= hi[j >> 1] && (a.window == 0 || p > hi[j >> 1] - a.window);
            s[n][j] = seen ? s[n][j] : kNegInf;
          }
      }
      float mc[2], base[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x_ = m[j];
#pragma unroll
        for (int n = 0; n < kChunk / 8; ++n) x_ = fmaxf(x_, fmaxf(s[n][2 * j], s[n][2 * j + 1]));
        x_ = fmaxf(x_, __shfl_xor_sync(0xffffffffu, x_, 1));
        x_ = fmaxf(x_, __shfl_xor_sync(0xffffffffu, x_, 2));
        base[j] = x_ == kNegInf ? 0.f : x_;   // nothing seen yet: every weight is exp(-inf)
        const float f = ex2((m[j] - base[j]) * a.scale_log2);
        m[j] = x_;
        mc[j] = base[j] * a.scale_log2;
        l[j] *= f;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          o[n][2 * j] *= f;
          o[n][2 * j + 1] *= f;
        }
      }
      if (__any_sync(0xffffffffu, fmaxf(fabsf(mc[0]), fabsf(mc[1])) > kFarScore)) {
#pragma unroll
        for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][j] -= base[j >> 1];
        mc[0] = mc[1] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[n][j] = ex2(fmaf(s[n][j], a.scale_log2, -mc[j >> 1]));
          l[j >> 1] += s[n][j];
        }
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k) {
        // weights in [0, 1] rounded to the cache's type for the tensor core:
        // half a step each, as the output's own rounding, averaged over the row
        const uint32_t p[4] = {Elem<T>::pack(s[2 * k][0], s[2 * k][1]), Elem<T>::pack(s[2 * k][2], s[2 * k][3]),
                               Elem<T>::pack(s[2 * k + 1][0], s[2 * k + 1][1]),
                               Elem<T>::pack(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
        for (int n = 0; n < HD / 8; n += 2) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4_trans(b0, b1, b2, b3,
                            vb + S::unit(r0 + k * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, n + (lane >> 4)));
          Elem<T>::mma(o[n], p, b0, b1);
          Elem<T>::mma(o[n + 1], p, b2, b3);
        }
      }
    }
    if (t + 1 < tb) {
      ++t;
      if constexpr (TMA) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
      next_stage();
      continue;
    }

    // the unit's end here: merge the WK slices through this stage
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
      l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
      if (t4 == 0) {
        st_m[wk][wm * 16 + g + 8 * j] = m[j];
        st_l[wk][wm * 16 + g + 8 * j] = l[j];
      }
    }
    if (tid < kRows) row_bad[tid] = 0;
    sync();
    if (tid < kRows) {
      float mm = kNegInf, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWK; ++w) mm = fmaxf(mm, st_m[w][tid]);
      const float base = mm == kNegInf ? 0.f : mm;
#pragma unroll
      for (int w = 0; w < kWK; ++w) ll += st_l[w][tid] * ex2((st_m[w][tid] - base) * a.scale_log2);
      row_m[tid] = mm;
      row_l[tid] = ll;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float mm = kNegInf;
#pragma unroll
      for (int w = 0; w < kWK; ++w) mm = fmaxf(mm, st_m[w][wm * 16 + g + 8 * j]);
      const float f = ex2((m[j] - (mm == kNegInf ? 0.f : mm)) * a.scale_log2);
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        o[n][2 * j] *= f;
        o[n][2 * j + 1] *= f;
      }
    }
    float* buf = reinterpret_cast<float*>(smem + stage * S::kStageBytes);
    const bool whole = t_first == 0 && tb == u.n_tile;
    float* part = partial_at<HD>(a.work, kRows, cta, t_first == 0 ? 1 : 0);
    if (tid == 0 && !whole && t_first == 0) *join_record(a, cta) = record_of(u, cta, n_cta, total);
    constexpr int kCols = HD / S::kPasses;
    bool any_bad = false;
#pragma unroll
    for (int ps = 0; ps < S::kPasses; ++ps) {
#pragma unroll
      for (int n = 0; n < kCols / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float2*>(buf + S::merge(wk * kRows + wm * 16 + g + 8 * j, n * 8 + 2 * t4)) =
              make_float2(o[ps * (kCols / 8) + n][2 * j], o[ps * (kCols / 8) + n][2 * j + 1]);
      sync();
      for (int i = tid; i < kRows * (kCols / 4); i += kPagedThreads) {
        const int row = i / (kCols / 4), c = (i % (kCols / 4)) * 4;
        const int tok = row / a.group, hh = row - tok * a.group;
        if (tok >= u.n_tok) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWK; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(buf + S::merge(w * kRows + row, c));
          v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
        }
        const bool bad = !(fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) < __int_as_float(0x7f800000)) ;
        if (bad) {
          row_bad[row] = 1;
          any_bad = true;
        }
        const int col = ps * kCols + c;
        if (whole) {
          // no position seen: the sums are zero, and so is the row
          const float inv = row_m[row] == kNegInf && row_l[row] == 0.f ? 0.f : 1.f / row_l[row];
          uint2 w2 = make_uint2(Elem<T>::pack(v.x * inv, v.y * inv), Elem<T>::pack(v.z * inv, v.w * inv));
          char* dst = a.out + (u.row0 + tok) * a.out_row + (u.h * a.group + hh) * a.out_head;
          *reinterpret_cast<uint2*>(dst + col * 2) = w2;
          if (a.lse && col == 0)
            a.lse[(u.row0 + tok) * a.lse_row + u.h * a.group + hh] =
                row_m[row] == kNegInf ? kNegInf
                                      : (row_m[row] * a.scale_log2 + log2f(row_l[row])) * 0.693147180559945309f;
        } else {
          *reinterpret_cast<float4*>(part + row * HD + col) = v;
          if (col == 0) {
            part[kRows * HD + row] = row_m[row];
            part[kRows * HD + kRows + row] = row_l[row];
          }
        }
      }
      if (ps + 1 < S::kPasses) sync();
    }
    bool some_bad;
    if constexpr (TMA) some_bad = bar_or(1, kPagedThreads, any_bad);
    else some_bad = __syncthreads_or(any_bad) != 0;
    if constexpr (TMA) {
      // the merge wrote the stage: its next fill comes after that
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }
    if (some_bad) {
      // rows warp, warp + 8, .., one a lane (a NaN score that it sees spoils the whole row)
      const int row = warp + lane * kPagedWarps;
      const float l_row = row < kRows && row_bad[row] ? row_l[row] : __int_as_float(0x7fffffff);
      const bool odd = l_row == l_row;
      const unsigned todo = __ballot_sync(0xffffffffu, odd);
      if (todo)
        mend_rows<T, HD>(a, kv, u.pages, u.h, u.row0, u.pos0, warp, kPagedWarps, todo, odd ? row_m[row] : 0.f,
                         odd && whole ? 1.f / l_row : 1.f, (u.t0 + t_first) * kTile, (u.t0 + t + 1) * kTile,
                         whole ? nullptr : part, waits);
      // every warp has read its rows' marks before the next unit's end clears
      // them (a TMA ring lets a warp run whole units ahead of another)
      sync();
    }
    if constexpr (WM == 1) {
      if (!whole && a.arrived) {
        // the last of the unit's CTAs to come here joins their results
        const int first = t_first == 0 ? cta : static_cast<int>(((u.start + 1) * n_cta - 1) / total);
        const int4 rec = record_of(u, first, n_cta, total);
        sync();
        if (tid == 0) {   // (releases what the barrier has gathered, and acquires for it)
          unsigned before;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.arrived + first) : "memory");
          joins = before + 1 == static_cast<unsigned>(rec.x);
          if (joins) a.arrived[first] = 0;
        }
        sync();
        if (joins) join_unit_here<T, HD, kRows>(a, first, rec, warp);
      }
    }
    if (!u.more(x1)) break;
    next_unit<kTile>(b, kv, tpu, a.window, u);
    t = t_first = 0;
    tb = u.upto(x1);
    begin_unit();
    next_stage();
  }
  if (!TMA) cp_async_wait<0>();
  if (bad_page) *err = 1;
}

// Joins the partial results of the unit that CTA blockIdx.x began and did not
// finish, as its record says.
template <typename T, int HD, int ROWS, int BLK>
__global__ void __launch_bounds__(kJoinThreads) attn_paged_join_kernel(const __grid_constant__ AttnPaged a) {
  constexpr int kWarps = kJoinThreads / kWarp;
  grid_dep_wait();
  const int4 rec = __ldcg(join_record(a, blockIdx.x));
  if (rec.x == 0) return;
  join_unit<T, HD, ROWS, BLK, 8>(a, blockIdx.x, rec, blockIdx.y * kWarps + threadIdx.x / kWarp, gridDim.y * kWarps);
}

template <typename T, int HD, int WM, bool TMA = false>
cudaError_t paged_attr() {
  return cudaFuncSetAttribute(attn_paged_kernel<T, HD, WM, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(PagedShape<HD, WM, TMA>::kSmem));
}
template <typename T, int HD>
cudaError_t paged_attr_hd() {
  cudaError_t e = paged_attr<T, HD, 2>();
  if constexpr (HD <= 128) {
    if (e == cudaSuccess) e = paged_attr<T, HD, 1>();
  }
  if constexpr (HD == 64 || HD == 128) {
    if (e == cudaSuccess) e = paged_attr<T, HD, 1, true>();
    if (e == cudaSuccess) e = paged_attr<T, HD, 2, true>();
  }
  if (e == cudaSuccess) e = paged_attr<T, HD, 4>();
  if (e == cudaSuccess) e = paged_attr<T, HD, 8>();
  return e;
}
template <typename T>
cudaError_t paged_attr_all() {
  cudaError_t e = paged_attr_hd<T, 32>();
  if (e == cudaSuccess) e = paged_attr_hd<T, 64>();
  if (e == cudaSuccess) e = paged_attr_hd<T, 96>();
  if (e == cudaSuccess) e = paged_attr_hd<T, 128>();
  if (e == cudaSuccess) e = paged_attr_hd<T, 256>();
  return e;
}

template <typename T, int HD, int ROWS, int BLK>
cudaError_t launch_join(const AttnPaged& a, cudaStream_t st) {
  // 16 blocks an owner at most: all of them are resident at once
  OpLaunch l(dim3(a.n_cta, std::min(ROWS / (kJoinThreads / kWarp), 16), 1), kJoinThreads, 0, st);
  return cudaLaunchKernelEx(&l.cfg, attn_paged_join_kernel<T, HD, ROWS, BLK>, a);
}

template <typename T, int HD, int WM, bool TMA = false>
cudaError_t launch_paged(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st) {
  using S = PagedShape<HD, WM, TMA>;
  CUtensorMap km = {}, vm = {};
  const int box = TMA ? page_box_rows(kv) : 0;
  if (TMA && (!encode_pages<T>(&km, kv.k, kv, box) || !encode_pages<T>(&vm, kv.v, kv, box))) return cudaErrorInvalidValue;
  OpLaunch l(dim3(a.n_cta, 1, 1), S::kThreads, S::kSmem, st);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, attn_paged_kernel<T, HD, WM, TMA>, km, vm, a, b, kv, box, err);
  return e != cudaSuccess || a.arrived ? e : launch_join<T, HD, S::kRows, S::kRows>(a, st);
}

// The smallest row block that holds the longest sequence's rows: K and V are
// read once per block of rows, and padding rows cost tensor work only.
template <typename T, int HD>
cudaError_t launch_paged_hd(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st) {
  const long long rows = static_cast<long long>(b.max_rows) * a.group;
  if constexpr (HD == 64 || HD == 128) {
    if (rows <= 32 && tma_pages(kv))
      return rows <= 16 ? launch_paged<T, HD, 1, true>(a, b, kv, err, st) : launch_paged<T, HD, 2, true>(a, b, kv, err, st);
  }
  if constexpr (HD <= 128) {
    if (rows <= 16) return launch_paged<T, HD, 1>(a, b, kv, err, st);
  }
  if (rows <= 32) return launch_paged<T, HD, 2>(a, b, kv, err, st);
  if (rows <= 64) return launch_paged<T, HD, 4>(a, b, kv, err, st);
  return launch_paged<T, HD, 8>(a, b, kv, err, st);
}
template <typename T>
cudaError_t launch_paged_t(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st) {
  switch (kv.head_dim) {
    case 32: return launch_paged_hd<T, 32>(a, b, kv, err, st);
    case 64: return launch_paged_hd<T, 64>(a, b, kv, err, st);
    case 96: return launch_paged_hd<T, 96>(a, b, kv, err, st);
    case 128: return launch_paged_hd<T, 128>(a, b, kv, err, st);
    default: return launch_paged_hd<T, 256>(a, b, kv, err, st);
  }
}

}  // namespace alm

// Acceptance of drafted tokens for a ragged batch (alm_verify): one
// thread-block cluster a sequence, one launch, no scratch in global memory.
//
//   e_j = exp((l_j - M) / T), M = max l;  e_j = 0 where e_j < min_p
//   p_j = e_j / Z, Z = sum e;  accept token i iff u_i q_i(x_i) < p_i(x_i)
//   at the first refusal: draw from r_j = max(0, p_j - q_j), R = sum r:
//   the first j whose running sum of r exceeds u R
//
// Answers are whole numbers, so values next to a border decide them: every
// comparison is made in 64 bits.  Z of every row is first summed from 32-bit
// exponentials (relative error below 1e-5: at most 6e-8 of |x| <= 104 from the
// product and the instruction's 2^-22 per term), which decides all but the
// comparisons within kNear of equality; those, and the row the token is drawn
// from, sum Z again in 64 bits, with a table-driven exponential (below).
//
// HBM bounds large batches (every row's logits once; the drawn row again from
// L2), latency small ones: the CTAs of a cluster own consecutive slices of
// the vocabulary and exchange maxima and sums through distributed shared
// memory.  A lane takes 8 consecutive entries at a time, a warp 256, so that
// a draw is found by one scan over the warps' sums and one over a warp's lanes.
#include <cooperative_groups.h>

#include <type_traits>

#include "../../include/androidllm_b200.h"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace alm {
namespace {

constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / kWarp;
constexpr int kVerRows = 32;        // k_max + 1 at most
constexpr int kVerBlock = 8 * kWarp;   // entries a warp takes at a time
constexpr double kNear = 1e-4;

struct VerShared {
  double table[64];     // 2^(i / 64)
  float wm[kVerRows][kVerWarps];
  double ws[kVerRows][kVerWarps];
  int wi[kVerRows][kVerWarps];
  // this CTA's slice of every row, read by the whole cluster
  float cta_m[kVerRows];
  double cta_s[kVerRows];
  int cta_i[kVerRows];
  // rows of the whole vocabulary
  float row_m[kVerRows];
  double row_z[kVerRows];
  int row_i[kVerRows];
  double dsum[kVerWarps];
  double cta_d[2];      // two slots in turn: one is read while the next is written
  double cta_r[2][kVerWarps];   // the residual's sums by warp, in index order (by attempt)
  int cta_last[2];              // last index with a positive residual, or -1
};

ALM_DEV float ex2f_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp((l - top) / T) in 64 bits, c = 64 log2(e) / T: with t = (l - top) c =
// n + g, n whole and |g| <= 1/2, it is 2^(n div 64) 2^((n mod 64) / 64)
// 2^(g / 64); the middle factor comes from a table, the last from its Taylor
// series to degree 5, whose remainder is below (ln 2 / 128)^6 / 720 = 4e-17
// (Tang's table-driven method).  12 instructions of the 64-bit pipe, about a
// third of the library function's.  NaN counts as -inf, +inf logits (l == top)
// share the mass; below 2^-1000 the result is 0.
ALM_DEV double exp64(double t, const double* table) {   // 2^(t / 64)
  constexpr double kMagic = 6755399441055744.0;   // 1.5 * 2^52: adding it rounds to a whole number
  constexpr double a1 = 0.693147180559945309417 / 64, a2 = a1 * a1 / 2, a3 = a2 * a1 / 3, a4 = a3 * a1 / 4,
                   a5 = a4 * a1 / 5;
  // no branch: eight of these run side by side, and the 64-bit pipe's latency is long
  const bool some = t > -64000.0;
  const double tt = some ? t : 0.0;
  const double r = tt + kMagic;
  const int n = __double2loint(r);
  const double g = tt - (r - kMagic);
  double p = fma(g, a5, a4);
  p = fma(g, p, a3);
  p = fma(g, p, a2);
  p = fma(g, p, a1);
  p = fma(g, p, 1.0);
  const double e = p * table[n & 63];
  const double w = __hiloint2double(__double2hiint(e) + ((n >> 6) << 20), __double2loint(e));
  return some ? w : 0.0;
}
ALM_DEV double weight64(float l, float top, double c, const double* table) {
  const double e = exp64((static_cast<double>(l) - static_cast<double>(top)) * c, table);
  return l == top && l > kNegInf ? 1.0 : e;
}

// 16-bit logits have few leading parts: l = h + r with h the value without its
// low bits and r what they add, so exp((l - top) / T) = exp((h - top) / T)
// exp(r / T), two table entries and one product in 64 bits instead of the 25
// instructions above.  h has one entry per sign, exponent and leading
// mantissa bits, r one per sign, exponent and low bits.
template <typename T>
struct Split {   // fp32: no tables
  static constexpr int kHi = 0, kLo = 0;
  ALM_DEV static int hi(uint32_t) { return 0; }
  ALM_DEV static int lo(uint32_t) { return 0; }
  ALM_DEV static void parts(int, float&, bool&) {}
  ALM_DEV static double rest(int) { return 0.0; }
};
template <>
struct Split<half> {   // 5 + 5 bits of the mantissa
  static constexpr int kHi = 2048, kLo = 2048;
  ALM_DEV static int hi(uint32_t b) { return b >> 5; }
  ALM_DEV static int lo(uint32_t b) { return (b >> 10) << 5 | (b & 31); }
  ALM_DEV static float value(uint32_t b) { return __half2float(__ushort_as_half(static_cast<unsigned short>(b))); }
  ALM_DEV static void parts(int i, float& v, bool& finite) {
    v = value(i << 5);
    finite = (i >> 5 & 31) != 31;
  }
  ALM_DEV static double rest(int i) {
    const uint32_t se = i >> 5;
    if ((se & 31) == 31) return 0.0;
    return static_cast<double>(value(se << 10 | (i & 31))) - static_cast<double>(value(se << 10));
  }
};
template <>
struct Split<__nv_bfloat16> {   // 3 + 4 bits of the mantissa; r for exponents 2^-63 .. 2^32
  static constexpr int kHi = 4096, kLo = 2 * 96 * 16;
  ALM_DEV static int hi(uint32_t b) { return b >> 4; }
  ALM_DEV static int lo(uint32_t b) {
    const int e = min(max(static_cast<int>(b >> 7 & 255) - 64, 0), 95);
    return ((b >> 15) * 96 + e) << 4 | (b & 15);
  }
  ALM_DEV static float value(uint32_t b) { return __uint_as_float(b << 16); }
  ALM_DEV static void parts(int i, float& v, bool& finite) {
    v = value(i << 4);
    finite = (i >> 3 & 255) != 255;
  }
  ALM_DEV static double rest(int i) {
    const int se = i >> 4, sign = se / 96;
    const uint32_t base = static_cast<uint32_t>(sign << 15 | (se % 96 + 64) << 7);
    return static_cast<double>(value(base | (i & 15))) - static_cast<double>(value(base));
  }
};
// Where the tables hold: both factors far from overflow, and no low bits
// that matter outside the exponents above.  (Weights below e^-630 of the
// largest may count as zero.)
ALM_DEV bool tables_hold(float top, float temp) {
  return fabsf(top) <= 2000.f * temp && temp >= 2.5e-4f && temp <= 1e4f;
}

// The bits of entries j .. j + 7 of a row; those of -inf behind the slice's end.
template <typename T>
ALM_DEV void load8(const T* l, int j, int end, bool vec, uint32_t (&v)[8]) {
  constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, half>::value ? 0xfc00u : 0xff80u;
  if (vec && j + 8 <= end) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(l + j));
    if constexpr (sizeof(T) == 4) {
      const uint4 y = __ldg(reinterpret_cast<const uint4*>(l + j) + 1);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = w[i] & 0xffffu, v[2 * i + 1] = w[i] >> 16;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = j + i < end ? __ldg(reinterpret_cast<const unsigned*>(l) + j + i) : kNone;
      else v[i] = j + i < end ? __ldg(reinterpret_cast<const unsigned short*>(l) + j + i) : kNone;
    }
  }
}
template <typename T>
ALM_DEV float value_of(uint32_t b) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(b);
  else return Split<T>::value(b);
}
ALM_DEV void load8f(const float* l, int j, int end, bool vec, float (&v)[8]) {
  uint32_t b[8];
  load8(l, j, end, vec, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(b[i]);
}

ALM_DEV double warp_sum64(double z) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  return z;
}
// A sum of 2^((v - m) k) for the maximum `top` instead of m.
ALM_DEV float scaled(float z, float m, float top, float k) { return m == top ? z : z * ex2f_((m - top) * k); }
// first place of the maximum
ALM_DEV void join_first(float& m, int& at, float om, int oi) {
  at = m > om ? at : om > m ? oi : min(at, oi);
  m = fmaxf(m, om);
}

template <typename T>
__global__ void __launch_bounds__(kVerThreads, 2) verify_kernel(const Verify a) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ VerShared sh;
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int n_cta = static_cast<int>(cl.num_blocks()), cta = static_cast<int>(cl.block_rank());
  const int s = blockIdx.x / n_cta;
  const int row0 = max(0, min(__ldg(a.row_start + s), a.n_rows));
  const int n_row = min(max(0, min(__ldg(a.row_start + s + 1), a.n_rows) - row0), a.k_max + 1);
  const int k = n_row - 1;
  const float temp = __ldg(a.temperature + s);
  const bool greedy = !(temp > 0.f);
  // an infinite temperature still leaves -inf (and the rest of a row with +inf) out
  const double inv_t = greedy ? 1.0 : fmax(1.0 / static_cast<double>(temp), 1e-37);
  const double c64 = 64 * 1.4426950408889634074 * inv_t;
  const double min_p = !greedy && a.min_p ? static_cast<double>(__ldg(a.min_p + s)) : 0.0;
  int* tokens = a.tokens + static_cast<size_t>(s) * (a.k_max + 1);
  if (n_row == 0) {   // the same for the whole cluster
    if (cta == 0 && tid <= a.k_max) tokens[tid] = -1;
    if (cta == 0 && tid == 0) a.n_accepted[s] = 0;
    if (cta == 0 && a.p_draft && tid < a.k_max) a.p_draft[static_cast<size_t>(s) * a.k_max + tid] = 0.f;
    return;
  }
  // this CTA's slice of the vocabulary, a multiple of 8 wide
  const int width = ((a.vocab + n_cta - 1) / n_cta + 7) / 8 * 8;
  const int v0 = min(a.vocab, cta * width), v1 = min(a.vocab, v0 + width);
  const float k_log2 = static_cast<float>(1.4426950408889634 * inv_t);
  const bool vec = a.vec != 0;
  if (tid < 64) sh.table[tid] = exp2(tid / 64.0);

  auto row_ptr = [&](int i) { return reinterpret_cast<const T*>(a.logits + (row0 + i) * a.logits_row); };

  // Maximum and 32-bit sum (greedy: first place of the maximum) of every row's
  // slice.  The rows' blocks of 256 entries form one line that the warps share.
  for (int i = tid; i < n_row * kVerWarps; i += kVerThreads) {
    sh.wm[i / kVerWarps][i % kVerWarps] = kNegInf;
    sh.ws[i / kVerWarps][i % kVerWarps] = 0.0;
    sh.wi[i / kVerWarps][i % kVerWarps] = 0x7fffffff;
  }
  __syncthreads();
  {
    const int n_blk = (v1 - v0 + kVerBlock - 1) / kVerBlock;
    const int b1 = n_row * n_blk * (warp + 1) / kVerWarps;
    constexpr int kDeep = sizeof(T) == 4 ? 2 : 4;   // blocks in flight
    for (int blk = n_row * n_blk * warp / kVerWarps; blk < b1;) {
      const int i = blk / n_blk;
      const int row_end = min(b1, (i + 1) * n_blk);
      const T* l = row_ptr(i);
      float m = kNegInf, z = 0.f;
      int at = 0x7fffffff;
      while (blk < row_end) {
        uint32_t v[kDeep][8];
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
          load8(l, v0 + (blk + d - i * n_blk) * kVerBlock + lane * 8, blk + d < row_end ? v1 : 0, vec, v[d]);
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
          float f[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) f[q] = value_of<T>(v[d][q]);
          float top = f[0];
#pragma unroll
          for (int q = 1; q < 8; ++q) top = fmaxf(top, f[q]);   // a NaN is passed over
          if (greedy) {
            if (top > m) {
              m = top;
#pragma unroll
              for (int q = 7; q >= 0; --q)
                if (f[q] == top) at = v0 + (blk + d - i * n_blk) * kVerBlock + lane * 8 + q;
            }
            continue;
          }
          if (top > m) {
            z *= ex2f_((m - top) * k_log2);
            m = top;
          }
          // the difference first: it is small where the weight is not
          const uint64_t m2 = pair(-m, -m), k2 = pair(k_log2, k_log2);
          float sum = 0.f;
#pragma unroll
          for (int q = 0; q < 8; q += 2) {
            float x, y;
            unpair(mul2(add2(pair(f[q], f[q + 1]), m2), k2), x, y);
            sum += ex2f_(x) + ex2f_(y);
          }
          if (!(sum < 16.f)) {   // NaN: a NaN logit, or infinities less infinities
            sum = 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              sum += !(f[q] > kNegInf) ? 0.f : f[q] == m ? 1.f : ex2f_((f[q] - m) * k_log2);
          }
          z += sum;
        }
        blk += kDeep;
      }
      blk = row_end;
      if (greedy) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          join_first(m, at, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, at, o));
      }
      const float top = warp_max(m);
      const double zd = warp_sum(scaled(z, m, top, k_log2));
      m = top;
      if (lane == 0) sh.wm[i][warp] = m, sh.ws[i][warp] = zd, sh.wi[i][warp] = at;
    }
  }
  __syncthreads();
  // a warp a row: the CTA's warps, then the cluster's CTAs, a lane each
  auto join_lanes = [&](float& m, double& z, int& at) {
    if (greedy) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1)
        join_first(m, at, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, at, o));
      return;
    }
    const float top = warp_max(m);
    z = warp_sum64(z * static_cast<double>(scaled(1.f, m, top, k_log2)));
    m = top;
  };
  for (int i = warp; i < n_row; i += kVerWarps) {
    float m = sh.wm[i][lane % kVerWarps];
    double z = lane < kVerWarps ? sh.ws[i][lane] : 0.0;
    int at = sh.wi[i][lane % kVerWarps];
    join_lanes(m, z, at);
    if (lane == 0) sh.cta_m[i] = m, sh.cta_s[i] = z, sh.cta_i[i] = at;
  }
  cl.sync();
  for (int i = warp; i < n_row; i += kVerWarps) {
    const VerShared* o = cl.map_shared_rank(&sh, min(lane % 16, n_cta - 1));
    const bool on = lane < n_cta;
    float m = on ? o->cta_m[i] : kNegInf;
    double z = on ? o->cta_s[i] : 0.0;
    int at = on ? o->cta_i[i] : 0x7fffffff;
    join_lanes(m, z, at);
    if (lane == 0) sh.row_m[i] = m, sh.row_z[i] = z, sh.row_i[i] = at;
  }
  __syncthreads();

  // 64-bit weights of row i: through the tables where they hold
  extern __shared__ __align__(16) double tables[];
  double *const t_hi = tables, *const t_lo = tables + Split<T>::kHi;
  int tab_row = -1;          // the row the tables are made for
  bool tab = false;          // ... and whether they are used
  auto make_tables = [&](int i) {   // by the whole CTA
    tab_row = i;
    const float top = sh.row_m[i];
    tab = Split<T>::kHi > 0 && tables_hold(top, temp);
    if (!tab) return;
    __syncthreads();         // the last row's are no longer read
    for (int j = tid; j < Split<T>::kHi; j += kVerThreads) {
      float v = 0.f;
      bool finite = false;
      Split<T>::parts(j, v, finite);
      // (entries above the maximum are not read)
      t_hi[j] = finite && v <= top + fabsf(top) ? exp64((static_cast<double>(v) - static_cast<double>(top)) * c64, sh.table) : 0.0;
    }
    for (int j = tid; j < Split<T>::kLo; j += kVerThreads) t_lo[j] = exp64(Split<T>::rest(j) * c64, sh.table);
    __syncthreads();
  };
  auto wt = [&](uint32_t bits, float top) {   // of row tab_row
    double e;
    if (tab) e = t_hi[Split<T>::hi(bits)] * t_lo[Split<T>::lo(bits)];
    else e = weight64(value_of<T>(bits), top, c64, sh.table);
    return e < min_p ? 0.0 : e;
  };
  auto bits_at = [&](int i, int j) -> uint32_t {
    if constexpr (sizeof(T) == 4) return __ldg(reinterpret_cast<const unsigned*>(row_ptr(i)) + j);
    else return __ldg(reinterpret_cast<const unsigned short*>(row_ptr(i)) + j);
  };

  // Sum of f over the vocabulary, 8 entries a lane; every CTA of the cluster
  // calls it together and gets the same value (the same additions).
  int turn = 0;
  auto cluster_sum = [&](auto&& f, const T* l) {
    double z = 0.0;
    for (int j = v0 + tid * 8; j < v1; j += kVerThreads * 8) {
      uint32_t v[8];
      load8(l, j, v1, vec, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) z += f(v[q]);
    }
    z = warp_sum64(z);
    if (lane == 0) sh.dsum[warp] = z;
    __syncthreads();
    if (warp == 0) {
      const double t = warp_sum64(lane < kVerWarps ? sh.dsum[lane] : 0.0);
      if (lane == 0) sh.cta_d[turn] = t;
    }
    cl.sync();
    // a lane a CTA: the remote reads are in flight together
    const double part = lane < n_cta ? cl.map_shared_rank(&sh, lane)->cta_d[turn] : 0.0;
    turn ^= 1;
    return warp_sum64(part);
  };
  auto exact_sum = [&](int i) {
    const float top = sh.row_m[i];
    if (tab_row != i) make_tables(i);
    return cluster_sum([&](uint32_t v) { return wt(v, top); }, row_ptr(i));
  };
  // Min-p: the 32-bit sums again without the entries below it, now that the
  // maxima are known.  row_i tells whether an entry lies too near the border.
  if (min_p > 0.0) {
    const float cut = static_cast<float>(min_p), lo = cut * (1.f - 1e-4f), hi = cut * (1.f + 1e-4f);
    const int n_blk = (v1 - v0 + kVerBlock - 1) / kVerBlock;
    const int b1 = n_row * n_blk * (warp + 1) / kVerWarps;
    for (int i = tid; i < n_row * kVerWarps; i += kVerThreads) {
      sh.ws[i / kVerWarps][i % kVerWarps] = 0.0;
      sh.wi[i / kVerWarps][i % kVerWarps] = 0;
    }
    __syncthreads();
    for (int blk = n_row * n_blk * warp / kVerWarps; blk < b1;) {
      const int i = blk / n_blk, row_end = min(b1, (i + 1) * n_blk);
      const T* l = row_ptr(i);
      const float top = sh.row_m[i];
      float z = 0.f;
      bool near = false;
#pragma unroll 4
      for (; blk < row_end; ++blk) {
        uint32_t v[8];
        load8(l, v0 + (blk - i * n_blk) * kVerBlock + lane * 8, v1, vec, v);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float f = value_of<T>(v[q]);
          const float e = !(f > kNegInf) ? 0.f : f == top ? 1.f : ex2f_((f - top) * k_log2);
          near |= e >= lo && e <= hi;
          z += e < cut ? 0.f : e;
        }
      }
      const double zd = warp_sum64(z);
      near = __any_sync(0xffffffffu, near);
      if (lane == 0) sh.ws[i][warp] = zd, sh.wi[i][warp] = near;
    }
    cl.sync();       // (the CTA's barrier too; the first sums have been read)
    for (int i = warp; i < n_row; i += kVerWarps) {
      const double z = warp_sum64(lane < kVerWarps ? sh.ws[i][lane] : 0.0);
      const int near = __any_sync(0xffffffffu, sh.wi[i][lane % kVerWarps] != 0);
      if (lane == 0) sh.cta_s[i] = z, sh.cta_i[i] = near;
    }
    cl.sync();
    for (int i = warp; i < n_row; i += kVerWarps) {
      const VerShared* o = cl.map_shared_rank(&sh, min(lane, n_cta - 1));
      const double z = warp_sum64(lane < n_cta ? o->cta_s[i] : 0.0);
      const int near = __any_sync(0xffffffffu, o->cta_i[i] != 0);
      if (lane == 0) sh.row_z[i] = z, sh.row_i[i] = near;
    }
    __syncthreads();
  }

  // Acceptance: lane i weighs token i (every warp alike), then the tokens are
  // gone through in order; what the 32-bit sums leave open is summed in 64 bits.
  const int* x = a.draft + static_cast<size_t>(s) * a.k_max;
  int acc = 0;
  double z_stop = 0.0;
  bool have_z = false;
  {
    double p = 0.0, uq = 0.0, z = 0.0;
    int xi = -1;
    bool in = false, open = false;   // open: not decided by the 32-bit sum
    if (lane < k) {
      xi = __ldg(x + lane);
      in = xi >= 0 && xi < a.vocab;
      const float top = sh.row_m[lane];
      if (greedy) {
        p = in && top > kNegInf && xi == sh.row_i[lane] ? 1.0 : 0.0;
      } else {
        double e = in ? weight64(value_of<T>(bits_at(lane, xi)), top, c64, sh.table) : 0.0;
        if (e < min_p) e = 0.0;
        const double q =
            !a.q ? 1.0 : in ? static_cast<double>(__ldg(a.q + s * a.q_seq + lane * a.q_step + xi)) : 0.0;
        uq = __ldg(a.u + static_cast<size_t>(s) * (a.k_max + 1) + lane) * q;
        z = sh.row_z[lane];
        p = e > 0.0 ? e / z : 0.0;
        open = fabs(uq - p) <= kNear * p || (min_p > 0.0 && sh.row_i[lane] != 0);
      }
    }
    unsigned yes = __ballot_sync(0xffffffffu, lane < k && uq < p);
    unsigned unsure = __ballot_sync(0xffffffffu, open);
    for (acc = 0; acc < k; ++acc) {
      if (unsure >> acc & 1) {
        const double zx = exact_sum(acc);
        bool ok = false;
        if (lane == acc) {
          const double e = in ? wt(bits_at(acc, xi), sh.row_m[acc]) : 0.0;   // by the sum's own weights
          z = zx;
          p = e > 0.0 ? e / zx : 0.0;
          ok = uq < p;
        }
        yes = (yes & ~(1u << acc)) | __ballot_sync(0xffffffffu, ok);
        if (!(yes >> acc & 1)) z_stop = zx, have_z = true;
      }
      if (!(yes >> acc & 1)) break;
    }
    // (behind the first refusal p is reported from the 32-bit sums, but for
    // entries at the min-p border, which only the 64-bit weights tell apart)
    for (int i = acc + 1; i < k; ++i)
      if (min_p > 0.0 && sh.row_i[i] != 0 && !greedy) {
        const double zx = exact_sum(i);
        if (lane == i) {
          const double e = in ? wt(bits_at(i, xi), sh.row_m[i]) : 0.0;
          p = e > 0.0 ? e / zx : 0.0;
        }
      }
    if (cta == 0 && warp == 0 && a.p_draft && lane < k)
      a.p_draft[static_cast<size_t>(s) * a.k_max + lane] = static_cast<float>(p);
  }
  if (cta == 0) {
    if (a.p_draft)
      for (int i = k + tid; i < a.k_max; i += kVerThreads) a.p_draft[static_cast<size_t>(s) * a.k_max + i] = 0.f;
    if (tid <= a.k_max && tid != acc) tokens[tid] = tid < acc ? __ldg(x + tid) : -1;
    if (tid == 0) a.n_accepted[s] = acc;
  }

  // the drawn token
  const float top = sh.row_m[acc];
  if (greedy || !(top > kNegInf)) {
    if (cta == 0 && tid == 0) tokens[acc] = top > kNegInf ? sh.row_i[acc] : -1;
  } else {
    const double z = have_z ? z_stop : exact_sum(acc);
    if (tab_row != acc) make_tables(acc);
    const double inv_z = 1.0 / z;
    const T* l = row_ptr(acc);
    const float* q = a.q && acc < k ? a.q + s * a.q_seq + acc * a.q_step : nullptr;
    const bool q_vec = q && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    const int drop = !a.q && acc < k ? __ldg(x + acc) : -1;   // a certain draft: its whole mass goes
    const double u = __ldg(a.u + static_cast<size_t>(s) * (a.k_max + 1) + k);
    // a warp owns a run of entries; the runs of all warps and CTAs are in index order
    const int run = ((width + kVerWarps - 1) / kVerWarps + kVerBlock - 1) / kVerBlock * kVerBlock;
    const int j0 = min(v1, v0 + warp * run), j1 = min(v1, j0 + run);
    for (int use_q = 1; use_q >= 0; --use_q) {
      // what a lane's 8 entries leave after the draft's share
      auto rest8 = [&](int j, double (&r)[8]) {
        uint32_t v[8];
        float w[8];
        load8(l, j, j1, vec, v);
        if (use_q && q) load8f(q, j, j1, q_vec, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          double e = wt(v[i], top) * inv_z;
          if (use_q && q) {
            // (a NaN or infinite share leaves nothing)
            e = fmax(e - static_cast<double>(w[i]), 0.0);
            if (j + i >= j1) e = 0.0;
          } else if (use_q && j + i == drop) {
            e = 0.0;
          }
          r[i] = e;
        }
      };
      double sum = 0.0;
      int last = -1;
      for (int j = j0 + lane * 8; j < j1; j += kVerBlock) {
        double r[8];
        rest8(j, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum += r[i];
          if (r[i] > 0.0) last = j + i;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
      }
      if (tid == 0) sh.cta_last[use_q] = -1;
      __syncthreads();
      if (lane == 0) {
        sh.dsum[warp] = sum;
        if (last >= 0) atomicMax(&sh.cta_last[use_q], last);
      }
      __syncthreads();
      // running sums in index order, each the last one plus a part that is not
      // negative, so they never decrease: the warps' inside the CTA, then the CTAs'
      if (tid == 0) {
        double t = 0.0;
        for (int w = 0; w < kVerWarps; ++w) sh.cta_r[use_q][w] = t += sh.dsum[w];
      }
      cl.sync();
      const VerShared* o = cl.map_shared_rank(&sh, min(lane, n_cta - 1));
      const double cta_sum = o->cta_r[use_q][kVerWarps - 1];
      int row_last = o->cta_last[use_q];
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) row_last = max(row_last, __shfl_xor_sync(0xffffffffu, row_last, w));
      double total = 0.0, base = 0.0;
      for (int c = 0; c < n_cta; ++c) {
        if (c == cta) base = total;
        total += __shfl_sync(0xffffffffu, cta_sum, c);
      }
      const double before = warp > 0 ? base + sh.cta_r[use_q][warp - 1] : base;
      const double end = base + sh.cta_r[use_q][warp];
      if (total > 0.0 || use_q == 0) {
        // the one warp whose run the goal lies in
        const double goal = u * total;
        if (before <= goal && end > goal) {
          double at = before;
          int found = -1;
          for (int b = j0; b < j1 && found < 0; b += kVerBlock) {
            double r[8];
            rest8(b + lane * 8, r);
            double mine = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) mine += r[i];
            double scan = mine;
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, scan, o);
              if (lane >= o) scan += y;
            }
            double run_sum = at + (scan - mine);
            int hit = -1;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              run_sum += r[i];
              if (hit < 0 && r[i] > 0.0 && run_sum > goal) hit = b + lane * 8 + i;
            }
            const unsigned any = __ballot_sync(0xffffffffu, hit >= 0);
            if (any) found = __shfl_sync(0xffffffffu, hit, __ffs(any) - 1);
            at += __shfl_sync(0xffffffffu, scan, kWarp - 1);
          }
          // rounding can leave the walk's end just short of the run's sum
          if (lane == 0) tokens[acc] = found >= 0 ? found : last;
        }
        // a draw of 1, or rounding at the row's end: the last entry with mass
        if (!(total > goal) && cta == 0 && tid == 0) tokens[acc] = row_last;
        break;
      }
    }
  }
  cl.sync();   // no CTA leaves while another reads its shared memory
}

template <typename T>
constexpr int table_bytes() {
  return (Split<T>::kHi + Split<T>::kLo) * static_cast<int>(sizeof(double));
}

template <typename T>
cudaError_t launch_t(const Verify& a, cudaStream_t st) {
  // few sequences: 16 CTAs each, so that a row's slices stay short; many: 8
  // (the portable size, which more GPCs can place)
  const int ctas = a.n_seq <= 8 ? 16 : 8;
  OpLaunch l(dim3(a.n_seq * ctas, 1, 1), kVerThreads, table_bytes<T>(), st, ctas);
  return cudaLaunchKernelEx(&l.cfg, verify_kernel<T>, a);
}

}  // namespace

template <typename T>
static cudaError_t verify_attrs_t() {
  cudaError_t e = cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, table_bytes<T>());
  return e;
}
cudaError_t verify_init_attrs() {
  cudaError_t e = verify_attrs_t<half>();
  if (e == cudaSuccess) e = verify_attrs_t<__nv_bfloat16>();
  if (e == cudaSuccess) e = verify_attrs_t<float>();
  return e;
}

cudaError_t launch_verify(const Verify& a, int dtype, cudaStream_t st) {
  return dtype == ALM_F16 ? launch_t<half>(a, st) : dtype == ALM_BF16 ? launch_t<__nv_bfloat16>(a, st) : launch_t<float>(a, st);
}

}  // namespace alm

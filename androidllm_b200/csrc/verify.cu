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
// exponentials, which decides all but the comparisons within kNear + kNearBlock n
// of equality, n the blocks of 8 entries that a lane adds up at most; those, and
// the row the token is drawn from, sum Z again with 64-bit weights.  The sums'
// relative error is below 1e-5 (at most 6e-8 of |x| <= 104 from the product and
// the instruction's 2^-22 per term) and, for each block, 2^-24 for its addition
// and 3e-7 for the factor when the maximum grows, or 8 additions of 2^-24 (min-p):
// 5e-7.  n is 75 at 151,936 tokens, 8192 at the largest vocabulary.
//
// The CTAs of a cluster own consecutive slices of the vocabulary and exchange
// maxima and sums through distributed shared memory.  A lane takes 8
// consecutive entries at a time, a warp 256, so that a draw is found by one
// scan over the warps' sums and one over blocks of 256.
//
// Every row's logits come from HBM once, the drawn row's again from L2; at 64 x
// 0-4 drafts of 151936 tokens that would be 12 us.  It takes 72 us (1 TB/s):
// the serial steps inside a cluster (50 us: a pass over 1 to 5 rows, 3-9 us;
// their join, 2 us; min-p again over all rows, 2-9 us; the 64-bit pass, 9 us;
// the draw, 5 us) run on 36 clusters at a time, in two waves.  One session's
// 4 drafts take 22 us, five barriers across the cluster and the passes' latency.
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
constexpr double kNear = 1e-4, kNearBlock = 5e-7;

struct VerShared {
  double table[256 * 16];   // 2^(i / 256), 16 copies side by side
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
  int row_i[kVerRows];   // greedy: the maximum's place; min-p: an entry at the border
  double dsum[kVerWarps];
  double cta_d[2];      // two slots in turn: one is read while the next is written
  double cta_r[2][kVerWarps];   // the residual's sums by warp, in index order (by attempt)
  int cta_last[2];              // last index with a positive residual, or -1
  int warp_last[kVerWarps];
  int cta_over;                 // a lane has more than one entry at the draft's border
  int found;
};

ALM_DEV float ex2f_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp((l - top) / T) in 64 bits, c = 256 log2(e) / T: with t = (l - top) c =
// n + g, n whole and |g| <= 0.56 (n comes from 32 bits), it is 2^(n div 256)
// 2^((n mod 256) / 256) 2^(g / 256); the middle factor comes from a table, the
// last from its Taylor series to degree 4, whose remainder is below
// (0.56 ln 2 / 256)^5 / 120 = 7e-17 (Tang's table-driven method).  8
// instructions of the 64-bit pipe and a conversion.  The table has a copy for
// each lane of a half-warp, in banks of its own: random entries of one copy
// cost 6 turns of the shared memory instead of 2, which bound these passes.
// NaN counts as -inf, +inf logits (l == top) share the mass.  An entry below
// `least` (min-p, 2^-999 if there is none) weighs 0.
//
// kPlain: the maximum and `low`, the logit that weighs 2^-1000, are finite
// numbers: -inf and NaN are raised to `low`, which takes 9 instructions fewer
// than telling them apart (the 64-bit passes are bound by the issue of their
// instructions).  The two forms agree in every bit.
constexpr int kExpTable = 256, kExpCopies = 16;
template <bool kPlain>
struct Exp64 {
  const double* table;   // this lane's copy
  double top_d, c, least;
  float top, c_f, low;
  ALM_DEV double operator()(float l) const {
    constexpr double a1 = 0.693147180559945309417 / kExpTable, a2 = a1 * a1 / 2, a3 = a2 * a1 / 3, a4 = a3 * a1 / 4;
    // no branch: eight of these run side by side, and the 64-bit pipe's latency is long
    bool some = true;
    if (kPlain) {
      l = fmaxf(l, low);
    } else {
      some = (l - top) * c_f > -1000.f * kExpTable;
      if (l == top) some = l > kNegInf;
    }
    float x = l - top;
    if (!kPlain && (!some || l == top)) x = 0.f;
    const int n = __float_as_int(fmaf(x, c_f, 12582912.f));   // 1.5 2^23, whose last bit is 1: n + 0x4b400000
    const double n_d = __hiloint2double(0x43300000, n + 0x34c00000) - 4503601774854144.0;   // 2^52 + 2^31
    double d = static_cast<double>(l) - top_d;
    if (!kPlain && l == top) d = 0.0;
    const double g = fma(d, c, -n_d);
    double p = fma(g, a4, a3);
    p = fma(g, p, a2);
    p = fma(g, p, a1);
    p = fma(g, p, 1.0);
    const double e = p * table[(n & (kExpTable - 1)) * kExpCopies];
    const double w = __hiloint2double(__double2hiint(e) + ((n & 0xfff00) << 12), __double2loint(e));
    return !(w >= least) || !some ? 0.0 : w;
  }
};

template <typename T>
ALM_DEV float value_of(uint32_t b) {
  if constexpr (std::is_same<T, half>::value) return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
  else return __uint_as_float(sizeof(T) == 4 ? b : b << 16);
}

// Entries j .. j + 7 of a row as they lie in memory; -inf (`fill`) behind the slice's end.
template <typename T>
struct Raw8 {
  uint4 x[sizeof(T) / 2];
  ALM_DEV uint32_t word(int i) const {
    const uint4& u = x[i / 4];
    return i % 4 == 0 ? u.x : i % 4 == 1 ? u.y : i % 4 == 2 ? u.z : u.w;
  }
  ALM_DEV uint32_t bits(int i) const {
    if constexpr (sizeof(T) == 4) return word(i);
    else return i % 2 ? word(i / 2) >> 16 : word(i / 2) & 0xffffu;
  }
};
template <typename T>
constexpr uint32_t neg_inf() { return sizeof(T) == 4 ? 0xff800000u : std::is_same<T, half>::value ? 0xfc00u : 0xff80u; }
template <typename T>
ALM_DEV Raw8<T> load8(const T* l, int j, int end, bool vec, uint32_t fill = neg_inf<T>()) {
  Raw8<T> r;
  if (vec && j + 8 <= end) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) r.x[i] = __ldg(reinterpret_cast<const uint4*>(l + j) + i);
  } else {
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = j + i < end ? __ldg(reinterpret_cast<const unsigned*>(l) + j + i) : fill;
      else v[i] = j + i < end ? __ldg(reinterpret_cast<const unsigned short*>(l) + j + i) : fill;
    }
    if constexpr (sizeof(T) == 4) {
      r.x[0] = make_uint4(v[0], v[1], v[2], v[3]);
      r.x[1] = make_uint4(v[4], v[5], v[6], v[7]);
    } else {
      r.x[0] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
  }
  return r;
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

// kPerSm: CTAs an SM holds at once.  Two hide latency where there are more CTAs
// than SMs (64 sequences: 74 us against 98 us with one); one leaves a thread
// 128 registers, which serves fewer CTAs better (1 x 4: 21.9 against 23.2 us,
// 13 x 1-7: 17.0 against 17.6 us).
template <typename T, int kPerSm>
__global__ void __launch_bounds__(kVerThreads, kPerSm) verify_kernel(const Verify a) {
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
  const double c64 = kExpTable * 1.4426950408889634074 * inv_t;
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
  if (!greedy && tid < kExpTable) {
    const double e = exp2(tid / static_cast<double>(kExpTable));
    for (int i = 0; i < kExpCopies; ++i) sh.table[tid * kExpCopies + (i + tid) % kExpCopies] = e;
  }

  auto row_ptr = [&](int i) { return reinterpret_cast<const T*>(a.logits + (row0 + i) * a.logits_row); };

  // the drafted tokens, one a lane; their draft probabilities are fetched meanwhile
  const int* x = a.draft + static_cast<size_t>(s) * a.k_max;
  const int xi = lane < k ? __ldg(x + lane) : -1;
  auto qx = [&] { return a.q + s * a.q_seq + lane * a.q_step + xi; };
  if (a.q && xi >= 0 && xi < a.vocab && warp == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(qx()));

  // Goes through this CTA's slice of every row: the rows' blocks of 256 entries
  // form one line that the warps share evenly, and a warp's next blocks are
  // under way while it computes on the last ones.
  const int n_blk = (v1 - v0 + kVerBlock - 1) / kVerBlock;
  auto all_rows = [&](auto&& block, auto&& row_done) {
    constexpr int kDeep = sizeof(T) == 4 ? 2 : 4;   // blocks in flight
    const int b1 = n_row * n_blk * (warp + 1) / kVerWarps;
    int blk = n_row * n_blk * warp / kVerWarps;
    if (blk >= b1) return;
    Raw8<T> now[kDeep], next[kDeep];
    auto fetch = [&](Raw8<T> (&r)[kDeep], int blk, int i, int row_end) {
#pragma unroll
      for (int d = 0; d < kDeep; ++d)
        if (blk + d < row_end) r[d] = load8(row_ptr(i), v0 + (blk + d - i * n_blk) * kVerBlock + lane * 8, v1, vec);
    };
    int i = blk / n_blk, row_end = min(b1, (i + 1) * n_blk);
    fetch(now, blk, i, row_end);
    while (blk < b1) {
      const bool ends = blk + kDeep >= row_end;
      const int nb = ends ? row_end : blk + kDeep;
      const int ni = ends ? i + 1 : i, nend = ends ? min(b1, row_end + n_blk) : row_end;
      if (nb < b1) fetch(next, nb, ni, nend);
#pragma unroll
      for (int d = 0; d < kDeep; ++d)
        if (blk + d < row_end) block(i, v0 + (blk + d - i * n_blk) * kVerBlock + lane * 8, now[d]);
      if (ends) row_done(i);
      blk = nb, i = ni, row_end = nend;
#pragma unroll
      for (int d = 0; d < kDeep; ++d) now[d] = next[d];
    }
  };

  // Maximum and 32-bit sum (greedy: first place of the maximum) of every row.
  for (int i = tid; i < n_row * kVerWarps; i += kVerThreads) {
    sh.wm[i / kVerWarps][i % kVerWarps] = kNegInf;
    sh.ws[i / kVerWarps][i % kVerWarps] = 0.0;
    sh.wi[i / kVerWarps][i % kVerWarps] = 0x7fffffff;
  }
  __syncthreads();
  {
    float m = kNegInf, z = 0.f;
    int at = 0x7fffffff;
    all_rows(
        [&](int, int j, const Raw8<T>& v) {
          float f[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) f[q] = value_of<T>(v.bits(q));
          float top = f[0];
#pragma unroll
          for (int q = 1; q < 8; ++q) top = fmaxf(top, f[q]);   // a NaN is passed over
          if (greedy) {
            if (top > m) {
              m = top;
#pragma unroll
              for (int q = 7; q >= 0; --q)
                if (f[q] == top) at = j + q;
            }
            return;
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
        },
        [&](int i) {
          if (greedy) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
              join_first(m, at, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, at, o));
          }
          const float top = warp_max(m);
          const double zd = warp_sum(scaled(z, m, top, k_log2));
          if (lane == 0) sh.wm[i][warp] = top, sh.ws[i][warp] = zd, sh.wi[i][warp] = at;
          m = kNegInf, z = 0.f, at = 0x7fffffff;
        });
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

  // 64-bit weights of row i, and f called with them in the form that holds
  const float c_f = fminf(static_cast<float>(c64), 1e38f);
  const double least = fmax(min_p, 0x1p-999);
  auto weights = [&](int i, auto plain) {
    const float top = sh.row_m[i];
    return Exp64<decltype(plain)::value>{sh.table + lane % kExpCopies, top, c64, least, top, c_f,
                                         top - 1000.f * kExpTable / c_f};
  };
  auto with_weights = [&](int i, auto&& f) {
    if (fabsf(sh.row_m[i]) + 1000.f * kExpTable / c_f < 1e38f && c_f < 1e30f) f(weights(i, std::true_type()));
    else f(weights(i, std::false_type()));
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
      const Raw8<T> v = load8(l, j, v1, vec);
#pragma unroll
      for (int q = 0; q < 8; ++q) z += f(v.bits(q));
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
    double z = 0.0;
    with_weights(i, [&](const auto& w) {
      z = cluster_sum([&](uint32_t v) { return w(value_of<T>(v)); }, row_ptr(i));
    });
    return z;
  };
  // Min-p: the 32-bit sums again without the entries below it, now that the
  // maxima are known.  row_i then tells whether an entry lies too near the border.
  if (min_p > 0.0) {
    // the 32-bit weights' error at the border, threefold: 1.3e-7 a unit of log2, and 3e-7
    const float cut = static_cast<float>(min_p), band = cut * 1e-6f * (1.f + fabsf(log2f(cut)));
    for (int i = tid; i < n_row * kVerWarps; i += kVerThreads) {
      sh.ws[i / kVerWarps][i % kVerWarps] = 0.0;
      sh.wi[i / kVerWarps][i % kVerWarps] = 0;
    }
    __syncthreads();
    float z = 0.f;
    bool near = false;
    all_rows(
        [&](int i, int, const Raw8<T>& v) {
          const float top = sh.row_m[i];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float f = value_of<T>(v.bits(q));
            // (0 times an infinite 1 / T, and inf - inf, are NaN; a NaN logit is below every bound)
            const float e = f == top ? 1.f : ex2f_((f - top) * k_log2);
            near |= fabsf(e - cut) <= band;
            z += e >= cut ? e : 0.f;
          }
        },
        [&](int i) {
          const double zd = warp_sum(z);
          near = __any_sync(0xffffffffu, near);
          if (lane == 0) sh.ws[i][warp] = zd, sh.wi[i][warp] = near;
          z = 0.f, near = false;
        });
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
  int acc = 0;
  double z_stop = 0.0;
  bool have_z = false;
  // (from the slices' width, not this CTA's slice: the cluster decides alike)
  const double near_p = kNear + kNearBlock * ((width + kVerBlock - 1) / kVerBlock);
  {
    double p = 0.0, uq = 0.0, z = 0.0;
    const bool in = xi >= 0 && xi < a.vocab;
    bool open = false;   // not decided by the 32-bit sum
    if (lane < k) {
      const float top = sh.row_m[lane];
      if (greedy) {
        p = in && top > kNegInf && xi == sh.row_i[lane] ? 1.0 : 0.0;
      } else {
        const double e = in && top > kNegInf ? weights(lane, std::false_type())(value_of<T>(bits_at(lane, xi))) : 0.0;
        const double q =
            !a.q ? 1.0 : in ? static_cast<double>(__ldg(qx())) : 0.0;
        uq = __ldg(a.u + static_cast<size_t>(s) * (a.k_max + 1) + lane) * q;
        z = sh.row_z[lane];
        p = e > 0.0 ? e / z : 0.0;
        open = fabs(uq - p) <= near_p * p || (min_p > 0.0 && sh.row_i[lane] != 0);
      }
    }
    unsigned yes = __ballot_sync(0xffffffffu, lane < k && uq < p);
    unsigned unsure = __ballot_sync(0xffffffffu, open);
    for (acc = 0; acc < k; ++acc) {
      if (unsure >> acc & 1) {
        const double zx = exact_sum(acc);
        bool ok = false;
        if (lane == acc) {
          const double e = in ? weights(acc, std::false_type())(value_of<T>(bits_at(acc, xi))) : 0.0;
          z = zx;
          p = e > 0.0 ? e / zx : 0.0;
          ok = uq < p;
        }
        yes = (yes & ~(1u << acc)) | __ballot_sync(0xffffffffu, ok);
        if (!(yes >> acc & 1)) z_stop = zx, have_z = true;
      }
      if (!(yes >> acc & 1)) break;
    }
    // (p is reported from the 32-bit sums where they decided and behind the first
    // refusal, but for rows with entries at the min-p border, which only the
    // 64-bit weights tell apart)
    for (int i = acc + 1; i < k; ++i)
      if (min_p > 0.0 && sh.row_i[i] != 0 && !greedy) {
        const double zx = exact_sum(i);
        if (lane == i) {
          const double e = in ? weights(i, std::false_type())(value_of<T>(bits_at(i, xi))) : 0.0;
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
    with_weights(acc, [&](const auto& weight) {
    const T* l = row_ptr(acc);
    const float* q = a.q && acc < k ? a.q + s * a.q_seq + acc * a.q_step : nullptr;
    const bool q_vec = q && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    const int drop = !a.q && acc < k ? __ldg(x + acc) : -1;   // a certain draft: its whole mass goes
    const double u = __ldg(a.u + static_cast<size_t>(s) * (a.k_max + 1) + k);
    // a warp owns a run of entries; the runs of all warps and CTAs are in index order
    const int run = ((width + kVerWarps - 1) / kVerWarps + kVerBlock - 1) / kVerBlock * kVerBlock;
    const int j0 = min(v1, v0 + warp * run), j1 = min(v1, j0 + run);
    // One pass finds Z and the residual sums: with z the 32-bit sum and P the
    // entries with e > q z,
    //   sum over P of (e / Z - q) = (D - (Z - z) B) / Z,  D = sum of e - q z, B = sum of q,
    // since no entry changes sides between z and Z but those within 2^-15 e of
    // the border; a lane keeps one of these for afterwards.  A lane with two, or
    // a z further from Z than that allows, and the sums are made again from Z.
    double z = z_stop, rest = 0.0;
    int rest_last = -1;
    bool fused = false;
    if (!have_z) {
      if (q)   // its first use: all of the warp's lines at once
        for (int j = j0 + lane * 32; j < j1; j += kWarp * 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + j));
      const double zs = sh.row_z[acc];
      double zl = 0.0, part = 0.0;
      int border = -1;
      bool over = false;
      for (int j = j0 + lane * 8; j < j1; j += kVerBlock) {
        const Raw8<T> v = load8(l, j, j1, vec);
        Raw8<float> w;
        if (q) w = load8(q, j, j1, q_vec, 0u);
        unsigned close = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double e = weight(value_of<T>(v.bits(i)));
          zl += e;
          if (q) {
            const double wd = static_cast<double>(value_of<float>(w.bits(i))), d = fma(-wd, zs, e);
            const bool near = (__double2hiint(d) & 0x7fffffff) < __double2hiint(e) - (15 << 20);
            if (near) close |= 1u << i;
            if (!near && d > 0.0) {
              rest += d;
              part += wd;
              rest_last = j + i;
            }
          } else if (e > 0.0 && j + i != drop) {
            rest += e;
            rest_last = j + i;
          }
        }
        if (close) {
          over |= border >= 0 || (close & (close - 1));
          border = j + __ffs(close) - 1;
        }
      }
      double t = warp_sum64(zl);
      if (tid == 0) sh.cta_over = 0;
      __syncthreads();
      if (lane == 0) sh.dsum[warp] = t;
      if (over) sh.cta_over = 1;
      __syncthreads();
      if (warp == 0) {
        t = warp_sum64(lane < kVerWarps ? sh.dsum[lane] : 0.0);
        if (lane == 0) sh.cta_d[turn] = t;
      }
      cl.sync();
      const VerShared* o = cl.map_shared_rank(&sh, min(lane, n_cta - 1));
      z = warp_sum64(lane < n_cta ? o->cta_d[turn] : 0.0);
      fused = !__any_sync(0xffffffffu, o->cta_over) && fabs(z - zs) <= 1e-5 * z;
      turn ^= 1;
      rest = fmax(rest - (z - zs) * part, 0.0) / z;
      if (border >= 0) {
        const double r = weight(value_of<T>(bits_at(acc, border))) / z - static_cast<double>(__ldg(q + border));
        if (r > 0.0) {
          rest += r;
          rest_last = max(rest_last, border);
        }
      }
    }
    const double inv_z = 1.0 / z;
    for (int use_q = 1; use_q >= 0; --use_q) {
      // what entries j .. j + 7, of those below end, leave after the draft's share
      auto rest8 = [&](int j, int end, double (&r)[8]) {
        const Raw8<T> v = load8(l, j, end, vec);
        Raw8<float> w;
        if (use_q && q) w = load8(q, j, end, q_vec, 0u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          double e = weight(value_of<T>(v.bits(i))) * inv_z;
          if (use_q && q) {
            // (a NaN or infinite share leaves nothing)
            e = fmax(e - static_cast<double>(value_of<float>(w.bits(i))), 0.0);
          } else if (use_q && j + i == drop) {
            e = 0.0;
          }
          r[i] = e;
        }
      };
      const bool done = use_q && fused;
      double sum = done ? rest : 0.0;
      int last = done ? rest_last : -1;
      for (int j = done ? j1 : j0 + lane * 8; j < j1; j += kVerBlock) {
        double r[8];
        rest8(j, j1, r);
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
        sh.warp_last[warp] = last;
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
      if (total > 0.0 || use_q == 0) {
        const double goal = u * total;
        const double* run_end = sh.cta_r[use_q];
        if (base <= goal && base + run_end[kVerWarps - 1] > goal) {   // in this CTA's slice: all its warps look for it
          int of = 0;   // the warp whose run the goal lies in
          while (!(base + run_end[of] > goal)) ++of;
          double at = of > 0 ? base + run_end[of - 1] : base;
          const int a0 = min(v1, v0 + of * run), a1 = min(v1, a0 + run);
          if (tid == 0) sh.found = 0x7fffffff;
          bool found = false;
          for (int b = a0; b < a1 && !found; b += kVerBlock * kVerWarps) {
            double r[8];
            const int j = b + warp * kVerBlock + lane * 8;
            rest8(j, a1, r);
            double mine = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) mine += r[i];
            double scan = mine;
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, scan, o);
              if (lane >= o) scan += y;
            }
            __syncthreads();   // the last round's sums have been read
            if (lane == kWarp - 1) sh.dsum[warp] = scan;
            __syncthreads();
            double run_sum = at;
            for (int w = 0; w < kVerWarps; ++w) {
              if (w == warp) run_sum = at + (scan - mine);
              at += sh.dsum[w];
            }
            int hit = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              run_sum += r[i];
              if (hit == 0x7fffffff && r[i] > 0.0 && run_sum > goal) hit = j + i;
            }
            hit = __reduce_min_sync(0xffffffffu, hit);
            if (lane == 0 && hit != 0x7fffffff) atomicMin(&sh.found, hit);
            __syncthreads();
            found = sh.found != 0x7fffffff;
          }
          // rounding can leave the walk's end just short of the run's sum
          if (tid == 0) tokens[acc] = found ? sh.found : sh.warp_last[of];
        }
        // a draw of 1, or rounding at the row's end: the last entry with mass
        if (!(total > goal) && cta == 0 && tid == 0) tokens[acc] = row_last;
        break;
      }
    }
    });
  }
  cl.sync();   // no CTA leaves while another reads its shared memory
}

template <typename T>
cudaError_t launch_t(const Verify& a, cudaStream_t st) {
  // few sequences: 16 CTAs each, so that a row's slices stay short; many: 8
  // (the portable size, which more GPCs can place; 64 sequences: 74 us, with 4
  // 78 us)
  const int ctas = a.n_seq <= 8 ? 16 : 8;
  OpLaunch l(dim3(a.n_seq * ctas, 1, 1), kVerThreads, 0, st, ctas);
  return a.n_seq * ctas <= a.n_sms ? cudaLaunchKernelEx(&l.cfg, verify_kernel<T, 1>, a)
                                   : cudaLaunchKernelEx(&l.cfg, verify_kernel<T, 2>, a);
}

}  // namespace

template <typename T>
static cudaError_t verify_attrs_t() {
  const cudaError_t e = cudaFuncSetAttribute(verify_kernel<T, 1>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e != cudaSuccess
             ? e : cudaFuncSetAttribute(verify_kernel<T, 2>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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

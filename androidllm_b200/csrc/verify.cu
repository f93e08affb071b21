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

template <typename T>
struct Logit;
template <>
struct Logit<half> {
  ALM_DEV static float up(half v) { return __half2float(v); }
};
template <>
struct Logit<__nv_bfloat16> {
  ALM_DEV static float up(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <>
struct Logit<float> {
  ALM_DEV static float up(float v) { return v; }
};

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
  int near_min;         // an entry next to the min-p border
  double dsum[kVerWarps];
  double cta_d[2];      // two slots in turn: one is read while the next is written
  int cta_near[2];
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
ALM_DEV double weight64(float l, float top, double c, const double* table) {
  constexpr double kMagic = 6755399441055744.0;   // 1.5 * 2^52: adding it rounds to a whole number
  constexpr double a1 = 0.693147180559945309417 / 64, a2 = a1 * a1 / 2, a3 = a2 * a1 / 3, a4 = a3 * a1 / 4,
                   a5 = a4 * a1 / 5;
  if (l == top) return l > kNegInf ? 1.0 : 0.0;
  const double t = (static_cast<double>(l) - static_cast<double>(top)) * c;
  if (!(t > -64000.0)) return 0.0;
  const double r = t + kMagic;
  const int n = __double2loint(r);
  const double g = t - (r - kMagic);
  double p = fma(g, a5, a4);
  p = fma(g, p, a3);
  p = fma(g, p, a2);
  p = fma(g, p, a1);
  p = fma(g, p, 1.0);
  const double e = p * table[n & 63];
  return __hiloint2double(__double2hiint(e) + ((n >> 6) << 20), __double2loint(e));
}

// Entries j .. j + 7 of a row; -inf behind the slice's end.
template <typename T>
ALM_DEV void load8(const T* l, int j, int end, bool vec, float (&v)[8]) {
  if (vec && j + 8 <= end) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(l + j)), y = __ldg(reinterpret_cast<const float4*>(l + j) + 1);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(l + j));
      const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = Logit<T>::up(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = j + i < end ? Logit<T>::up(l[j + i]) : kNegInf;
  }
}

// (maximum, sum of 2^((v - maximum) k)) of two parts
ALM_DEV void join(float& m, double& z, float om, double oz, float k) {
  const float nm = fmaxf(m, om);
  const double fa = m == nm ? 1.0 : static_cast<double>(ex2f_((m - nm) * k));
  const double fb = om == nm ? 1.0 : static_cast<double>(ex2f_((om - nm) * k));
  z = z * fa + oz * fb;
  m = nm;
}
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

  // maximum and 32-bit sum (greedy: first place of the maximum) of every row's slice
  for (int i = 0; i < n_row; ++i) {
    const T* l = row_ptr(i);
    float m = kNegInf;
    if (greedy) {
      int at = 0x7fffffff;
#pragma unroll 2
      for (int j = v0 + tid * 8; j < v1; j += kVerThreads * 8) {
        float v[8];
        load8(l, j, v1, vec, v);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (v[q] > m) m = v[q], at = j + q;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        join_first(m, at, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, at, o));
      if (lane == 0) sh.wm[i][warp] = m, sh.wi[i][warp] = at;
    } else {
      float z = 0.f;
#pragma unroll 4
      for (int j = v0 + tid * 8; j < v1; j += kVerThreads * 8) {
        float v[8];
        load8(l, j, v1, vec, v);
        float top = v[0];
#pragma unroll
        for (int q = 1; q < 8; ++q) top = fmaxf(top, v[q]);   // a NaN is passed over
        if (top > m) {
          z *= ex2f_((m - top) * k_log2);
          m = top;
        }
        // the difference first: it is small where the weight is not
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) sum += ex2f_((v[q] - m) * k_log2);
        if (!(sum < 16.f)) {   // NaN: a NaN logit, or infinities less infinities
          sum = 0.f;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            sum += !(v[q] > kNegInf) ? 0.f : v[q] == m ? 1.f : ex2f_((v[q] - m) * k_log2);
        }
        z += sum;
      }
      double zd = z;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        join(m, zd, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, zd, o), k_log2);
      if (lane == 0) sh.wm[i][warp] = m, sh.ws[i][warp] = zd;
    }
  }
  __syncthreads();
  if (tid < n_row) {
    float m = sh.wm[tid][0];
    if (greedy) {
      int at = sh.wi[tid][0];
      for (int w = 1; w < kVerWarps; ++w) join_first(m, at, sh.wm[tid][w], sh.wi[tid][w]);
      sh.cta_i[tid] = at;
    } else {
      double z = sh.ws[tid][0];
      for (int w = 1; w < kVerWarps; ++w) join(m, z, sh.wm[tid][w], sh.ws[tid][w], k_log2);
      sh.cta_s[tid] = z;
    }
    sh.cta_m[tid] = m;
  }
  cl.sync();
  if (tid < n_row) {
    const VerShared* r = cl.map_shared_rank(&sh, 0);
    float m = r->cta_m[tid];
    if (greedy) {
      int at = r->cta_i[tid];
      for (int c = 1; c < n_cta; ++c) {
        const VerShared* q = cl.map_shared_rank(&sh, c);
        join_first(m, at, q->cta_m[tid], q->cta_i[tid]);
      }
      sh.row_i[tid] = at;
    } else {
      double z = r->cta_s[tid];
      for (int c = 1; c < n_cta; ++c) {
        const VerShared* q = cl.map_shared_rank(&sh, c);
        join(m, z, q->cta_m[tid], q->cta_s[tid], k_log2);
      }
      sh.row_z[tid] = z;
    }
    sh.row_m[tid] = m;
  }
  __syncthreads();

  // Sum of f over the vocabulary, 8 entries a lane; every CTA of the cluster
  // calls it together.  near: whether any CTA's f raised sh.near_min.
  int turn = 0;
  auto cluster_sum = [&](auto&& f, const T* l, bool& near) {
    double z = 0.0;
    for (int j = v0 + tid * 8; j < v1; j += kVerThreads * 8) {
      float v[8];
      load8(l, j, v1, vec, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) z += f(v[q]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) sh.dsum[warp] = z;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int w = 0; w < kVerWarps; ++w) t += sh.dsum[w];
      sh.cta_d[turn] = t;
      sh.cta_near[turn] = sh.near_min;
    }
    cl.sync();
    double t = 0.0;
    near = false;
    for (int c = 0; c < n_cta; ++c) {
      t += cl.map_shared_rank(&sh, c)->cta_d[turn];
      near |= cl.map_shared_rank(&sh, c)->cta_near[turn] != 0;
    }
    turn ^= 1;
    return t;
  };
  auto exact_sum = [&](int i) {
    const float top = sh.row_m[i];
    bool near;
    return cluster_sum(
        [&](float v) {
          const double e = weight64(v, top, c64, sh.table);
          return e < min_p ? 0.0 : e;
        },
        row_ptr(i), near);
  };
  // The 32-bit sum without the entries below min-p; the 64-bit one where an
  // entry is too near the border to tell.
  auto min_p_sum = [&](int i, bool& exact) {
    const float top = sh.row_m[i];
    const float cut = static_cast<float>(min_p), lo = cut * (1.f - 1e-4f), hi = cut * (1.f + 1e-4f);
    if (tid == 0) sh.near_min = 0;
    __syncthreads();
    const double z = cluster_sum(
        [&](float v) {
          const float e = !(v > kNegInf) ? 0.f : v == top ? 1.f : ex2f_((v - top) * k_log2);
          if (e >= lo && e <= hi) sh.near_min = 1;
          return static_cast<double>(e < cut ? 0.f : e);
        },
        row_ptr(i), exact);
    return exact ? exact_sum(i) : z;
  };

  const int* x = a.draft + static_cast<size_t>(s) * a.k_max;
  int acc = 0;
  double z_stop = 0.0;
  bool have_z = false, open = true;
  for (int i = 0; i < k; ++i) {
    const int xi = __ldg(x + i);
    const bool in = xi >= 0 && xi < a.vocab;
    const float top = sh.row_m[i];
    double p = 0.0;
    if (greedy) {
      const bool same = in && top > kNegInf && xi == sh.row_i[i];
      p = same ? 1.0 : 0.0;
      if (open) {
        if (same) ++acc;
        else open = false;
      }
    } else {
      double e = in ? weight64(Logit<T>::up(row_ptr(i)[xi]), top, c64, sh.table) : 0.0;
      if (e < min_p) e = 0.0;
      bool exact = false;
      double z = sh.row_z[i];
      if (min_p > 0.0 && top > kNegInf) z = min_p_sum(i, exact);
      p = e > 0.0 ? e / z : 0.0;
      if (open) {
        const double q =
            !a.q ? 1.0 : in ? static_cast<double>(__ldg(a.q + s * a.q_seq + i * a.q_step + xi)) : 0.0;
        const double uq = __ldg(a.u + static_cast<size_t>(s) * (a.k_max + 1) + i) * q;
        if (!exact && fabs(uq - p) <= kNear * p) {
          z = exact_sum(i);
          exact = true;
          p = e > 0.0 ? e / z : 0.0;
        }
        if (uq < p) {
          ++acc;
        } else {
          open = false;
          z_stop = z;
          have_z = exact;
        }
      }
    }
    if (cta == 0 && tid == 0 && a.p_draft) a.p_draft[static_cast<size_t>(s) * a.k_max + i] = static_cast<float>(p);
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
        float v[8], w[8];
        load8(l, j, j1, vec, v);
        if (use_q && q) load8(q, j, j1, q_vec, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          double e = weight64(v[i], top, c64, sh.table);
          e = e < min_p ? 0.0 : e * inv_z;
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
cudaError_t launch_t(const Verify& a, cudaStream_t st) {
  // few sequences: 16 CTAs each, so that a row's slices stay short; many: 8
  // (the portable size, which more GPCs can place)
  const int ctas = a.n_seq <= 8 ? 16 : 8;
  OpLaunch l(dim3(a.n_seq * ctas, 1, 1), kVerThreads, 0, st, ctas);
  return cudaLaunchKernelEx(&l.cfg, verify_kernel<T>, a);
}

}  // namespace

cudaError_t verify_init_attrs() {
  cudaError_t e = cudaFuncSetAttribute(verify_kernel<half>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(verify_kernel<__nv_bfloat16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(verify_kernel<float>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

cudaError_t launch_verify(const Verify& a, int dtype, cudaStream_t st) {
  return dtype == ALM_F16 ? launch_t<half>(a, st) : dtype == ALM_BF16 ? launch_t<__nv_bfloat16>(a, st) : launch_t<float>(a, st);
}

}  // namespace alm

// Acceptance of drafted tokens for a ragged batch (alm_verify): one
// thread-block cluster a sequence, one launch, no scratch in global memory.
//
//   e_j = exp((l_j - M) / T), M = max l;  e_j = 0 where e_j < min_p
//   p_j = e_j / Z, Z = sum e;  accept token i iff u_i q_i(x_i) < p_i(x_i)
//   at the first refusal: draw from r_j = max(0, p_j - q_j), R = sum r:
//   the first j whose running sum of r exceeds u R
//
// Answers are whole numbers, so values next to a border decide them: every
// comparison is made in 64 bits.  Exponentials in 64 bits cost about 40
// instructions, so Z of every row is first summed from 32-bit exponentials
// (relative error below 1e-5: at most 6e-8 of |x| <= 104 from the product and
// the instruction's 2^-22 per term), which decides all but the comparisons
// within kNear of equality; those, and the row the token is drawn from, sum
// Z again in 64 bits.
//
// HBM bounds large batches (every row's logits once; the drawn row again from
// L2), latency small ones: the CTAs of a cluster own consecutive slices of
// the vocabulary and exchange maxima and sums through distributed shared
// memory.
#include <cooperative_groups.h>

#include "../../include/androidllm_b200.h"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace alm {
namespace {

constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / kWarp;
constexpr int kVerRows = 32;        // k_max + 1 at most
constexpr int kVerMaxCtas = 16;
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
  // 64-bit sums of one row: per warp here, per CTA for the cluster
  double dsum[kVerWarps];
  double cta_d[2];       // two slots in turn, so that a slot is read before it is written again
  double cta_r[kVerWarps];   // the residual's sums by warp, in index order
  int cta_last;              // last index with a positive residual, or -1
  int pick;
};

ALM_DEV double exact_weight(float l, float top, double inv_t, float min_p) {
  // +inf logits share the mass; NaN counts as -inf
  if (!(l > kNegInf)) return 0.0;
  const double e = l == top ? 1.0 : exp((static_cast<double>(l) - static_cast<double>(top)) * inv_t);
  return e < static_cast<double>(min_p) ? 0.0 : e;
}

template <typename T>
__global__ void __launch_bounds__(kVerThreads) verify_kernel(const Verify a) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ VerShared sh;
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
  const float min_p = !greedy && a.min_p ? __ldg(a.min_p + s) : 0.f;
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
  constexpr int kVec = 16 / sizeof(T);

  auto row_ptr = [&](int i) { return reinterpret_cast<const T*>(a.logits + (row0 + i) * a.logits_row); };

  // maximum, first place of it and 32-bit sum of every row's slice
  for (int i = 0; i < n_row; ++i) {
    const T* l = row_ptr(i);
    float m = kNegInf, z = 0.f;
    int at = 0x7fffffff;
    auto take = [&](float v, int j) {
      if (v > m) {
        z = m == kNegInf ? 0.f : z * exp2f((m - v) * k_log2);
        m = v;
        at = j;
        z += 1.f;
      } else if (v > kNegInf) {
        z += v == m ? 1.f : exp2f((v - m) * k_log2);
      }
    };
    if (a.vec) {
      const int n_vec = (v1 - v0) / kVec;
      for (int j = tid; j < n_vec; j += kVerThreads) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(l + v0) + j);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int q = 0; q < kVec; ++q) take(Logit<T>::up(e[q]), v0 + j * kVec + q);
      }
      for (int j = v0 + n_vec * kVec + tid; j < v1; j += kVerThreads) take(Logit<T>::up(l[j]), j);
    } else {
      for (int j = v0 + tid; j < v1; j += kVerThreads) take(Logit<T>::up(l[j]), j);
    }
    double zd = z;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, o);
      const double oz = __shfl_xor_sync(0xffffffffu, zd, o);
      const int oi = __shfl_xor_sync(0xffffffffu, at, o);
      const float nm = fmaxf(m, om);
      const double fa = m == nm ? 1.0 : static_cast<double>(exp2f((m - nm) * k_log2));
      const double fb = om == nm ? 1.0 : static_cast<double>(exp2f((om - nm) * k_log2));
      at = m > om ? at : om > m ? oi : min(at, oi);
      zd = zd * fa + oz * fb;
      m = nm;
    }
    if (lane == 0) sh.wm[i][warp] = m, sh.ws[i][warp] = zd, sh.wi[i][warp] = at;
  }
  __syncthreads();
  auto join = [&](float& m, double& z, int& at, float om, double oz, int oi) {
    const float nm = fmaxf(m, om);
    const double fa = m == nm ? 1.0 : static_cast<double>(exp2f((m - nm) * k_log2));
    const double fb = om == nm ? 1.0 : static_cast<double>(exp2f((om - nm) * k_log2));
    at = m > om ? at : om > m ? oi : min(at, oi);
    z = z * fa + oz * fb;
    m = nm;
  };
  if (tid < n_row) {
    float m = sh.wm[tid][0];
    double z = sh.ws[tid][0];
    int at = sh.wi[tid][0];
    for (int w = 1; w < kVerWarps; ++w) join(m, z, at, sh.wm[tid][w], sh.ws[tid][w], sh.wi[tid][w]);
    sh.cta_m[tid] = m, sh.cta_s[tid] = z, sh.cta_i[tid] = at;
  }
  cl.sync();
  if (tid < n_row) {
    const VerShared* r = cl.map_shared_rank(&sh, 0);
    float m = r->cta_m[tid];
    double z = r->cta_s[tid];
    int at = r->cta_i[tid];
    for (int c = 1; c < n_cta; ++c) {
      const VerShared* q = cl.map_shared_rank(&sh, c);
      join(m, z, at, q->cta_m[tid], q->cta_s[tid], q->cta_i[tid]);
    }
    sh.row_m[tid] = m, sh.row_z[tid] = z, sh.row_i[tid] = at;
  }
  __syncthreads();

  // sum over the vocabulary in 64 bits; every CTA of the cluster calls it together
  int turn = 0;
  auto exact_sum = [&](int i) {
    const T* l = row_ptr(i);
    const float top = sh.row_m[i];
    double z = 0.0;
    for (int j = v0 + tid; j < v1; j += kVerThreads) z += exact_weight(Logit<T>::up(l[j]), top, inv_t, min_p);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) sh.dsum[warp] = z;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int w = 0; w < kVerWarps; ++w) t += sh.dsum[w];
      sh.cta_d[turn] = t;
    }
    cl.sync();
    double t = 0.0;
    for (int c = 0; c < n_cta; ++c) t += cl.map_shared_rank(&sh, c)->cta_d[turn];
    turn ^= 1;
    return t;
  };

  // min-p leaves entries out of the sum: every row needs the filtered one
  const int* x = a.draft + static_cast<size_t>(s) * a.k_max;
  int acc = 0;
  double z_stop = 0.0;
  bool have_z = false;
  bool open = true;
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
      const double e = in && top > kNegInf ? exact_weight(Logit<T>::up(row_ptr(i)[xi]), top, inv_t, min_p) : 0.0;
      double z = sh.row_z[i];
      bool exact = false;
      if (min_p > 0.f) z = exact_sum(i), exact = true;
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
  if (cta == 0 && a.p_draft)
    for (int i = max(k, 0) + tid; i < a.k_max; i += kVerThreads) a.p_draft[static_cast<size_t>(s) * a.k_max + i] = 0.f;

  // the drawn token
  int pick = -1;
  const float top = sh.row_m[acc];
  if (greedy) {
    if (top > kNegInf) pick = sh.row_i[acc];
  } else if (top > kNegInf) {
    const double z = have_z ? z_stop : exact_sum(acc);
    const T* l = row_ptr(acc);
    const float* q = a.q && acc < k ? a.q + s * a.q_seq + acc * a.q_step : nullptr;
    const int drop = !a.q && acc < k ? __ldg(x + acc) : -1;   // a certain draft: its whole mass goes
    const double u = __ldg(a.u + static_cast<size_t>(s) * (a.k_max + 1) + k);
    // a warp owns a run of indices; the runs of all warps and CTAs are in index order
    const int run = (width / kVerWarps + kWarp) / kWarp * kWarp;
    const int j0 = min(v1, v0 + warp * run), j1 = min(v1, j0 + run);
    for (int use_q = 1; use_q >= 0; --use_q) {
      auto rest = [&](int j) {
        const double p = exact_weight(Logit<T>::up(l[j]), top, inv_t, min_p) / z;
        if (!use_q) return p;
        if (drop >= 0) return j == drop ? 0.0 : p;
        return q ? fmax(p - static_cast<double>(__ldg(q + j)), 0.0) : p;
      };
      double r = 0.0;
      int last = -1;
      for (int j = j0 + lane; j < j1; j += kWarp) {
        const double v = rest(j);
        r += v;
        if (v > 0.0) last = j;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        r += __shfl_xor_sync(0xffffffffu, r, o);
        last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
      }
      if (tid == 0) sh.cta_last = -1;
      __syncthreads();
      if (lane == 0) {
        sh.cta_r[warp] = r;
        if (last >= 0) atomicMax(&sh.cta_last, last);
      }
      if (tid == 0) sh.pick = 0x7fffffff;
      cl.sync();
      double total = 0.0, before = 0.0;
      int row_last = -1;
      for (int c = 0; c < n_cta; ++c) {
        const VerShared* o = cl.map_shared_rank(&sh, c);
        row_last = max(row_last, o->cta_last);
        for (int w = 0; w < kVerWarps; ++w) {
          if (c == cta && w == warp) before = total;
          total += o->cta_r[w];
        }
      }
      if (total > 0.0 || use_q == 0) {
        // the warp whose run holds the draw walks it in order
        const double goal = u * total;
        if (r > 0.0 && before <= goal && before + r > goal) {
          double sum = before;
          int found = -1;
          for (int b = j0; b < j1 && found < 0; b += kWarp) {
            const int j = b + lane;
            const double v = j < j1 ? rest(j) : 0.0;
            double sc = v;
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, sc, o);
              if (lane >= o) sc += y;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, v > 0.0 && sum + sc > goal);
            if (hit) found = b + __ffs(hit) - 1;
            sum += __shfl_sync(0xffffffffu, sc, kWarp - 1);
          }
          // rounding can leave the walk's end just short of the run's sum
          if (found < 0) found = last;
          if (lane == 0) atomicMin(&cl.map_shared_rank(&sh, 0)->pick, found);
        }
        cl.sync();
        pick = cl.map_shared_rank(&sh, 0)->pick;
        if (pick == 0x7fffffff) pick = row_last;   // a draw of 1, or rounding at the row's end
        break;
      }
      cl.sync();   // before the sums are written again
    }
  }
  if (cta == 0) {
    if (tid <= a.k_max) tokens[tid] = tid < acc ? __ldg(x + tid) : tid == acc ? pick : -1;
    if (tid == 0) a.n_accepted[s] = acc;
  }
  cl.sync();   // no CTA leaves while another reads its shared memory
}

template <typename T>
cudaError_t launch_t(const Verify& a, cudaStream_t st) {
  // few sequences: 16 CTAs each, so that a row's slices stay short; many: 8
  // (the portable size, which more GPCs can place)
  const int ctas = a.n_seq <= 8 ? 16 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.n_seq * ctas, 1, 1);
  cfg.blockDim = dim3(kVerThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, verify_kernel<T>, a);
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

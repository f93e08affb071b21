// Head norms, position rotation and the paged cache write of a pass's new
// rows in one launch (alm_rope_append).
//
//   y = x / sqrt(mean(x^2) + eps) * w        (per head, optional)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)
//
// q goes to q_out, K to its page, V to its page unchanged.  Every value is
// read once and written once, so HBM bounds long passes and the launch with
// one dependent chain of loads (row -> sequence -> page) short ones.
//
// A thread owns two 8-value chunks of a head that hold whole rotation pairs:
// chunks t and t + rot/16 when halves are paired, two neighbours when
// adjacent values are (and behind the rotated part).  The rotation then needs
// no exchange, and the norm one sum over the head's lanes.
#include "../../include/androidllm_b200.h"
#include "paged.cuh"

namespace alm {
namespace {

template <typename T>
struct Pack;
template <>
struct Pack<half> {
  ALM_DEV static float2 up(uint32_t u) { return __half22float2(*reinterpret_cast<half2*>(&u)); }
  ALM_DEV static uint32_t down(float a, float b) {
    half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct Pack<__nv_bfloat16> {
  ALM_DEV static float2 up(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u)); }
  ALM_DEV static uint32_t down(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

template <typename T>
ALM_DEV void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Pack<T>::up(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T>
ALM_DEV uint4 pack8(const float (&f)[8]) {
  return make_uint4(Pack<T>::down(f[0], f[1]), Pack<T>::down(f[2], f[3]), Pack<T>::down(f[4], f[5]),
                    Pack<T>::down(f[6], f[7]));
}

// 8 / 4 consecutive table entries as fp32.
template <typename R>
ALM_DEV void table8(const char* row, int i, float (&f)[8]) {
  if constexpr (sizeof(R) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(row) + i / 4);
    const float4 b = __ldg(reinterpret_cast<const float4*>(row) + i / 4 + 1);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack8<R>(__ldg(reinterpret_cast<const uint4*>(row + static_cast<size_t>(i) * 2)), f);
  }
}

// The sequence of row r: the last s with row_start[s] <= r (row_start does
// not decrease), found by the whole warp 32 entries at a time; -1 if the
// row lies before the first or behind the last sequence.
ALM_DEV int seq_of_row(const SeqBatch& b, int r) {
  const int lane = threadIdx.x % kWarp;
  int lo = 0, n = b.n_seq + 1;   // the answer's index lies in [lo - 1, lo + n - 1)
  while (n > 0) {
    const int step = (n + kWarp - 1) / kWarp;
    const int i = lo + lane * step;
    const bool below = i < lo + n && __ldg(b.row_start + i) <= r;
    const int c = __popc(__ballot_sync(0xffffffffu, below));   // entries lo, lo + step, .. that are <= r
    if (c == 0) return lo - 1;
    const int end = lo + n;
    lo = lo + (c - 1) * step + 1;
    n = min(step - 1, end - lo);
  }
  return lo - 1;
}

// One block a row.  HL: lanes that share a head (a power of two >= head_dim / 16).
template <typename T, typename R, bool INTER, int HL>
__global__ void __launch_bounds__(1024) rope_append_kernel(const RopeAppend a, const SeqBatch b, const PagedKV kv, int* err) {
  grid_dep_wait();
  grid_dep_launch();
  const int r = blockIdx.x;
  const int d = kv.head_dim, per_head = d / 16;
  const int n_heads = a.heads + 2 * kv.kv_heads;
  const int t = threadIdx.x % HL;
  const int half_chunks = a.rot / 16;
  // the thread's two 8-value chunks of a head
  const bool turns = t < half_chunks;
  const int ca = (INTER || !turns) ? 2 * t : t;
  const int cb = (INTER || !turns) ? 2 * t + 1 : t + half_chunks;

  const int s = seq_of_row(b, r);
  if (s < 0 || s >= b.n_seq) return;
  const Seq q = load_seq(b, kv, s);
  const int pos = q.n_kv - q.n_new + (r - q.row0);
  const int page_i = pos >= 0 ? page_of(kv, pos) : 0;
  const bool in_table = pos >= 0 && pos < a.rope_rows && q.pages != nullptr && __ldg(b.kv_len + s) == q.n_kv;
  const int page = in_table ? __ldg(q.pages + page_i) : -1;
  const bool ok = page >= 0 && page < kv.n_pages;
  if (!ok) {
    if (threadIdx.x == 0) *err = 1;
    return;
  }
  const size_t base = kv_offset(kv, page, 0, pos - page_i * kv.page_size);
  const size_t head_stride = static_cast<size_t>(kv.page_size) * d;
  const char* cs = a.rope + static_cast<size_t>(pos) * a.rot * sizeof(R);

  float cf[8], sf[8];   // the angles of the thread's pairs
  if (turns) {
    if constexpr (INTER) {
      // pairs 8t .. 8t + 7 are the angles of chunks 2t and 2t + 1
      table8<R>(cs, 8 * t, cf);
      table8<R>(cs, a.rot / 2 + 8 * t, sf);
    } else {
      table8<R>(cs, 8 * t, cf);
      table8<R>(cs, a.rot / 2 + 8 * t, sf);
    }
  }

  const bool any_norm = a.q_norm != nullptr || a.k_norm != nullptr;
  // whole warps run every round: the norm's sum exchanges values inside a head's lanes
  const int n_item = (n_heads * HL + kWarp - 1) / kWarp * kWarp;
  for (int i = threadIdx.x; i < n_item; i += blockDim.x) {
    const int h = i / HL;
    const bool live = h < n_heads && t < per_head;
    const int kind = h < a.heads ? 0 : h < a.heads + kv.kv_heads ? 1 : 2;
    const int hk = kind == 0 ? h : kind == 1 ? h - a.heads : h - a.heads - kv.kv_heads;
    const char* src = kind == 0   ? a.q + r * a.q_row + hk * a.q_head
                      : kind == 1 ? a.k + r * a.k_row + hk * a.k_head
                                  : a.v + r * a.v_row + hk * a.v_head;
    uint4 ua = make_uint4(0, 0, 0, 0), ub = ua;
    if (live) {
      ua = reinterpret_cast<const uint4*>(src)[ca];
      ub = reinterpret_cast<const uint4*>(src)[cb];
    }
    const char* norm = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float fa[8], fb[8];
    unpack8<T>(ua, fa);
    unpack8<T>(ub, fb);
    if (any_norm) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(fa[j], fa[j], fmaf(fb[j], fb[j], ss));
#pragma unroll
      for (int o = HL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (norm != nullptr && live) {
        const float inv = rsqrtf(ss / static_cast<float>(d) + a.eps);
        float wa[8], wb[8];
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(norm) + ca), wa);
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(norm) + cb), wb);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          fa[j] = fa[j] * inv * wa[j];
          fb[j] = fb[j] * inv * wb[j];
        }
      }
    }
    if (kind < 2) {
      if (turns) {
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = fa[2 * j], y = fa[2 * j + 1], z = fb[2 * j], w = fb[2 * j + 1];
            fa[2 * j] = x * cf[j] - y * sf[j];
            fa[2 * j + 1] = y * cf[j] + x * sf[j];
            fb[2 * j] = z * cf[j + 4] - w * sf[j + 4];
            fb[2 * j + 1] = w * cf[j + 4] + z * sf[j + 4];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = fa[j], y = fb[j];
            fa[j] = x * cf[j] - y * sf[j];
            fb[j] = y * cf[j] + x * sf[j];
          }
        }
      }
      ua = pack8<T>(fa);
      ub = pack8<T>(fb);
    }
    if (!live) continue;
    char* dst = kind == 0 ? a.q_out + r * a.qo_row + hk * a.qo_head
                          : (kind == 1 ? kv.k : kv.v) + (base + hk * head_stride) * sizeof(T);
    reinterpret_cast<uint4*>(dst)[ca] = ua;
    reinterpret_cast<uint4*>(dst)[cb] = ub;
  }
}

template <typename T, typename R, bool INTER>
cudaError_t launch_hl(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st) {
  const int lanes = kv.head_dim / 16;
  const int hl = lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
  const int items = ((a.heads + 2 * kv.kv_heads) * hl + kWarp - 1) / kWarp * kWarp;
  const int threads = items < 1024 ? items : 1024;
  OpLaunch l(dim3(b.n_rows, 1, 1), threads, 0, st);
  switch (hl) {
    case 2: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 2>, a, b, kv, err);
    case 4: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 4>, a, b, kv, err);
    case 8: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 8>, a, b, kv, err);
    default: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 16>, a, b, kv, err);
  }
}

template <typename T>
cudaError_t launch_r(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int rope_dtype, bool inter, int* err,
                     cudaStream_t st) {
  if (rope_dtype == ALM_F32)
    return inter ? launch_hl<T, float, true>(a, b, kv, err, st) : launch_hl<T, float, false>(a, b, kv, err, st);
  if (rope_dtype == ALM_BF16)
    return inter ? launch_hl<T, __nv_bfloat16, true>(a, b, kv, err, st)
                 : launch_hl<T, __nv_bfloat16, false>(a, b, kv, err, st);
  return inter ? launch_hl<T, half, true>(a, b, kv, err, st) : launch_hl<T, half, false>(a, b, kv, err, st);
}

}  // namespace

cudaError_t launch_rope_append(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int dtype, int rope_dtype,
                               bool interleaved, int* err, cudaStream_t st) {
  return dtype == ALM_BF16 ? launch_r<__nv_bfloat16>(a, b, kv, rope_dtype, interleaved, err, st)
                           : launch_r<half>(a, b, kv, rope_dtype, interleaved, err, st);
}

}  // namespace alm

// Head norms, position rotation and the paged cache write of a pass's new
// rows in one launch (alm_rope_append).
//
//   y = x / sqrt(mean(x^2) + eps) * w        (per head, optional)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)
//
// q goes to q_out, K to its page, V to its page unchanged.  Every value is
// read once and written once, so HBM bounds long passes and the launch with
// one dependent chain of loads (row -> sequence -> page) short ones: 4 x 2047
// rows of 28 + 4 + 4 heads of 128 take 32 us (4.9 TB/s, 75% of a copy's rate),
// 1 x 5 rows 2.6 us.
//
// A thread owns two 8-value chunks of a head that hold whole rotation pairs:
// chunks t and t + rot/16 when halves are paired, two neighbours when
// adjacent values are (and behind the rotated part).  The rotation then needs
// no exchange, and the norm one sum over the head's lanes.
#include "../../include/androidllm_b200.h"
#include <algorithm>

#include "paged.cuh"

namespace alm {
namespace {

template <typename T>
struct Pack;
template <>
struct Pack<half> {
  ALM_DEV static uint64_t up(uint32_t u) {
    const float2 f = __half22float2(*reinterpret_cast<half2*>(&u));
    return pair(f.x, f.y);
  }
  ALM_DEV static uint32_t down(uint64_t v) {
    float a, b;
    unpair(v, a, b);
    half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct Pack<__nv_bfloat16> {
  ALM_DEV static uint64_t up(uint32_t u) { return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
  ALM_DEV static uint32_t down(uint64_t v) {
    float a, b;
    unpair(v, a, b);
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

// 8 values as four fp32 pairs, and back.
template <typename T>
ALM_DEV void unpack8(const uint4& u, uint64_t (&f)[4]) {
  f[0] = Pack<T>::up(u.x), f[1] = Pack<T>::up(u.y), f[2] = Pack<T>::up(u.z), f[3] = Pack<T>::up(u.w);
}
template <typename T>
ALM_DEV uint4 pack8(const uint64_t (&f)[4]) {
  return make_uint4(Pack<T>::down(f[0]), Pack<T>::down(f[1]), Pack<T>::down(f[2]), Pack<T>::down(f[3]));
}

// 8 consecutive table entries from p as fp32 pairs.
template <typename R>
ALM_DEV void table8(const char* p, uint64_t (&f)[4]) {
  if constexpr (sizeof(R) == 4) {
    const ulonglong2 a = __ldg(reinterpret_cast<const ulonglong2*>(p)), b = __ldg(reinterpret_cast<const ulonglong2*>(p) + 1);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
  } else {
    unpack8<R>(__ldg(reinterpret_cast<const uint4*>(p)), f);
  }
}

// Where row r goes: its position, and its page, -1 if there is none (the
// position or the page is out of range), -2 for a row of no sequence.
ALM_DEV int2 place_of(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int r) {
  // the last sequence that starts at r or before (row_start does not decrease)
  int lo = 0, hi = b.n_seq;   // row_start[lo] <= r (or lo = 0) and r < row_start[hi + 1]
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (__ldg(b.row_start + mid) <= r) lo = mid;
    else hi = mid - 1;
  }
  if (lo >= b.n_seq || __ldg(b.row_start + lo) > r) return make_int2(0, -2);
  const Seq q = load_seq(b, kv, lo);
  const int pos = q.n_kv - q.n_new + (r - q.row0);
  if (pos < 0 || pos >= q.n_kv || pos >= a.rope_rows || q.pages == nullptr)   // (too long a sequence has no position)
    return make_int2(0, -1);
  const int page = __ldg(q.pages + page_of(kv, pos));
  return make_int2(pos, page >= 0 && page < kv.n_pages ? page : -1);
}

// 72 registers a thread: three blocks of 288 threads (28 + 2 * 4 heads of 128)
// an SM; with 64 the prefetched row spills.
constexpr int kRopeRegs = 72;
constexpr int kRopeRows = 64;       // rows a block at most
constexpr int kRopeThreads = 768;   // at most: 768 * 72 fits the register file

// A block takes `per_block` consecutive rows; a thread has one item (two chunks
// of one head), or several a blockDim apart, and takes it through the rows.
// The next row's values and page number are on their way while a row is
// computed.  HL: lanes that
// share a head (a power of two >= head_dim / 16).
template <typename T, typename R, bool INTER, int HL>
__global__ void __maxnreg__(kRopeRegs) rope_append_kernel(const __grid_constant__ RopeAppend a,
                                                          const __grid_constant__ SeqBatch b,
                                                          const __grid_constant__ PagedKV kv, int per_block, int* err) {
  grid_dep_wait();
  grid_dep_launch();
  const int d = kv.head_dim, per_head = d / 16;
  const int n_heads = a.heads + 2 * kv.kv_heads;
  const int t = threadIdx.x % HL;
  const int half_chunks = a.rot / 16;
  // the thread's two 8-value chunks of a head
  const bool turns = t < half_chunks;
  const int ca = (INTER || !turns) ? 2 * t : t;
  const int cb = (INTER || !turns) ? 2 * t + 1 : t + half_chunks;
  const size_t head_stride = static_cast<size_t>(kv.page_size) * d;
  const int n_item = (n_heads * HL + kWarp - 1) / kWarp * kWarp;   // every thread takes part in the first round

  const int r0 = blockIdx.x * per_block, r1 = min(r0 + per_block, b.n_rows);
  __shared__ int2 places[kRopeRows];
  bool placed = false;
  for (int i = threadIdx.x; i < n_item; i += blockDim.x) {
    const int h = i / HL;
    const bool live = h < n_heads && t < per_head;
    // kind 0: q, 1: k, 2: v; hk: head of that kind
    const int kind = h < a.heads ? 0 : h < a.heads + kv.kv_heads ? 1 : 2;
    const int hk = kind == 0 ? h : kind == 1 ? h - a.heads : h - a.heads - kv.kv_heads;
    const int64_t step = kind == 0 ? a.q_row : kind == 1 ? a.k_row : a.v_row;
    const char* src = (kind == 0   ? a.q + hk * a.q_head
                       : kind == 1 ? a.k + hk * a.k_head
                                   : a.v + hk * a.v_head) + r0 * step;
    char* q_dst = a.q_out + hk * a.qo_head + r0 * a.qo_row;
    char* const kv_dst = (kind == 1 ? kv.k : kv.v) + hk * head_stride * sizeof(T);
    const char* norm = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    uint4 ua = make_uint4(0, 0, 0, 0), ub = ua;
    if (live) {
      ua = reinterpret_cast<const uint4*>(src)[ca];
      ub = reinterpret_cast<const uint4*>(src)[cb];
    }

    if (!placed) {   // (the first row's values are on their way)
      for (int j = threadIdx.x; j < r1 - r0; j += blockDim.x) places[j] = place_of(a, b, kv, r0 + j);
      __syncthreads();
      placed = true;
    }
    for (int r = r0; r < r1; ++r, q_dst += a.qo_row) {
      uint4 na = ua, nb = ub;
      if (r + 1 < r1) {
        src += step;
        if (live) {
          na = reinterpret_cast<const uint4*>(src)[ca];
          nb = reinterpret_cast<const uint4*>(src)[cb];
        }
      }
      const int pos = places[r - r0].x, page = places[r - r0].y;
      if (page == -1 && i == 0) *err = 1;
      if (page >= 0) {   // the same for the whole block
        if (kind < 2) {
          const char* cs = a.rope + static_cast<size_t>(pos) * a.rot * sizeof(R);
          uint64_t cf[4], sf[4];   // the angles of the thread's pairs 8 t .. 8 t + 7
          if (turns) {
            table8<R>(cs + 8 * t * sizeof(R), cf);
            table8<R>(cs + (a.rot / 2 + 8 * t) * sizeof(R), sf);
          }
          uint64_t fa[4], fb[4];
          unpack8<T>(ua, fa);
          unpack8<T>(ub, fb);
          if (norm != nullptr) {   // the same for a head's lanes
            uint64_t sq = mul2(fa[0], fa[0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) sq = fma2(fa[j], fa[j], sq);
#pragma unroll
            for (int j = 0; j < 4; ++j) sq = fma2(fb[j], fb[j], sq);
            float x, y;
            unpair(sq, x, y);
            float ss = x + y;
            const unsigned lanes = HL == 32 ? 0xffffffffu : ((1u << HL) - 1) << (threadIdx.x % kWarp / HL * HL);
#pragma unroll
            for (int o = HL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
            const float inv = rsqrtf(ss * (1.f / static_cast<float>(d)) + a.eps);
            const uint64_t inv2 = pair(inv, inv);
            uint64_t w[4];
            unpack8<T>(__ldg(reinterpret_cast<const uint4*>(norm) + (live ? ca : 0)), w);
#pragma unroll
            for (int j = 0; j < 4; ++j) fa[j] = mul2(mul2(fa[j], inv2), w[j]);
            unpack8<T>(__ldg(reinterpret_cast<const uint4*>(norm) + (live ? cb : 0)), w);
#pragma unroll
            for (int j = 0; j < 4; ++j) fb[j] = mul2(mul2(fb[j], inv2), w[j]);
          }
          if (turns) {
            if constexpr (INTER) {
              // a pair's two values lie side by side: (x, y) (c, c) + (y, x) (-s, s)
              auto turn = [](uint64_t v, float c, float sn) {
                float x, y;
                unpair(v, x, y);
                return fma2(pair(y, x), pair(-sn, sn), mul2(v, pair(c, c)));
              };
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float c0, c1, s0_, s1_, c2, c3, s2, s3;
                unpair(cf[j], c0, c1), unpair(sf[j], s0_, s1_);
                unpair(cf[j + 2], c2, c3), unpair(sf[j + 2], s2, s3);
                fa[2 * j] = turn(fa[2 * j], c0, s0_), fa[2 * j + 1] = turn(fa[2 * j + 1], c1, s1_);
                fb[2 * j] = turn(fb[2 * j], c2, s2), fb[2 * j + 1] = turn(fb[2 * j + 1], c3, s3);
              }
            } else {
              const uint64_t minus = pair(-1.f, -1.f);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint64_t x = fa[j], y = fb[j];
                fa[j] = fma2(mul2(y, sf[j]), minus, mul2(x, cf[j]));
                fb[j] = fma2(x, sf[j], mul2(y, cf[j]));
              }
            }
          }
          ua = pack8<T>(fa);
          ub = pack8<T>(fb);
        }
        if (live) {
          char* dst = q_dst;
          if (kind != 0) dst = kv_dst + kv_offset(kv, page, 0, pos - page_of(kv, pos) * kv.page_size) * sizeof(T);
          reinterpret_cast<uint4*>(dst)[ca] = ua;
          reinterpret_cast<uint4*>(dst)[cb] = ub;
        }
      }
      ua = na, ub = nb;
    }
  }
}

template <typename T, typename R, bool INTER>
cudaError_t launch_hl(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int n_sms, int* err, cudaStream_t st) {
  const int lanes = kv.head_dim / 16;
  const int hl = lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
  const int items = ((a.heads + 2 * kv.kv_heads) * hl + kWarp - 1) / kWarp * kWarp;
  const int threads = items < kRopeThreads ? items : kRopeThreads;
  // as many blocks as are resident at once, then more rows a block
  const int blocks = n_sms * std::min(65536 / (kRopeRegs * threads), 8);
  const int per = std::min((b.n_rows + blocks - 1) / blocks, kRopeRows);
  OpLaunch l(dim3((b.n_rows + per - 1) / per, 1, 1), threads, 0, st);
  switch (hl) {
    case 2: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 2>, a, b, kv, per, err);
    case 4: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 4>, a, b, kv, per, err);
    case 8: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 8>, a, b, kv, per, err);
    default: return cudaLaunchKernelEx(&l.cfg, rope_append_kernel<T, R, INTER, 16>, a, b, kv, per, err);
  }
}

template <typename T>
cudaError_t launch_r(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int rope_dtype, bool inter, int n_sms,
                     int* err, cudaStream_t st) {
  if (rope_dtype == ALM_F32)
    return inter ? launch_hl<T, float, true>(a, b, kv, n_sms, err, st) : launch_hl<T, float, false>(a, b, kv, n_sms, err, st);
  if (rope_dtype == ALM_BF16)
    return inter ? launch_hl<T, __nv_bfloat16, true>(a, b, kv, n_sms, err, st)
                 : launch_hl<T, __nv_bfloat16, false>(a, b, kv, n_sms, err, st);
  return inter ? launch_hl<T, half, true>(a, b, kv, n_sms, err, st) : launch_hl<T, half, false>(a, b, kv, n_sms, err, st);
}

}  // namespace

cudaError_t launch_rope_append(const RopeAppend& a, const SeqBatch& b, const PagedKV& kv, int dtype, int rope_dtype,
                               bool interleaved, int n_sms, int* err, cudaStream_t st) {
  return dtype == ALM_BF16 ? launch_r<__nv_bfloat16>(a, b, kv, rope_dtype, interleaved, n_sms, err, st)
                           : launch_r<half>(a, b, kv, rope_dtype, interleaved, n_sms, err, st);
}

}  // namespace alm

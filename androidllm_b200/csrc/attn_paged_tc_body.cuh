// Attention of many new rows over the paged cache (alm_attn_paged) on the
// fifth-generation tensor cores; instantiated in attn_paged_tc_f16.cu and
// attn_paged_tc_bf16.cu.  The mathematics and the sharing of tiles are those of
// attn_paged_body.cuh; here 128 rows (tokens times the query heads of one K/V
// head) are the M of a tcgen05.mma:
//
//   S (128 x 128 positions, tensor memory) = Q (shared memory) . K^T
//   P = 2^(c S - c m), written over S as 16-bit values
//   O (128 x head_dim, tensor memory) += P (tensor memory) . V
//
// P is of the cache's type because the product's operands have one type; its half
// step is the output's own, averaged over the row.  The sum of weights is taken in
// fp32 before that rounding.
//
// Two streams alternate, so that one's softmax runs under the other's
// products: with kNQ = 2 they are two 128-row blocks over the same K and V
// tiles, with kNQ = 1 (at most 128 rows in a sequence) the even and the odd
// tiles of one block, joined at the unit's end.
//
// Warps 0-3 and 4-7: softmax of stream 0 and 1, one row a thread.  Warps 8 and
// 11: issue the products of stream 0 and 1.  Warp 9: loads K and V tiles with
// TMA, one box per page piece and 64 columns, into a ring of tiles.  Warp 10:
// loads Q.
//
// The reference maximum m follows the row's maximum only when that has grown
// by more than kSlack (in powers of two): weights stay below 2^kSlack, and the
// rescaling of O, which has to wait for the last product, is rare.
//
// At 128 x 128 x 128 a tile's products and its exponentials both take about
// 1024 cycles of an SM, so the streams take turns at the exponential unit
// (without turns both wait for it at once and the tensor core idles: 351 us
// against 285 us at 4 x 2047 rows, 28 heads over 4 of 128).  4 x 2047 rows
// take 272 us replayed from a graph (920 TFLOP/s, 55% of a large library product's
// rate), 309 us called back to back, at the power limit (810 TFLOP/s): a stream's
// chain of product, tensor-memory read, maximum, exponentials, write and
// product is 3540 cycles a step of both streams, 2048 of them tensor work.
// 1 x 7 rows over 131 thousand positions (HBM-bound): 66 us, 4.1 TB/s, 61
// to 63 us of it this kernel.
#pragma once

#include "attn_paged_body.cuh"
#include "tc.cuh"

namespace alm {

// 12 warps launch with 168 registers a thread; the softmax warps (one row of S
// a thread) then take kSoftRegs and the others keep kRestRegs:
// 256 * 216 + 128 * 72 = 384 * 168.
constexpr int kTcPagedThreads = 384;
constexpr int kSoftRegs = 216, kRestRegs = 72;
static_assert(256 * kSoftRegs + 128 * kRestRegs == kTcPagedThreads * 168, "the shares add up to the launch's registers");
constexpr float kSlack = 8.f;

template <int HD, int NQ>
struct TcShape {
  static constexpr int kTile = 128;
  static constexpr int kChunks = HD / 64;                  // 128-byte column groups
  static constexpr int kTileBytes = 128 * HD * 2;          // Q block, K or V tile
  static constexpr int kSlots = HD == 128 ? (NQ == 2 ? 5 : 6) : 10;
  // slots of one ring: both streams follow every fill of a shared ring; where
  // each has tiles of its own it has a ring of its own (a barrier's parity
  // tells one phase from the next, not from the one after)
  static constexpr int kRing = NQ == 2 ? kSlots : kSlots / 2;
  static constexpr size_t kSmem = static_cast<size_t>(NQ + kSlots) * kTileBytes + 1024;
  static constexpr int kColS = 0, kColO = 256, kTmemCols = 512;
};

struct TcShared {
  SchedShared sched;
  uint64_t full[10], empty[10];
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2][2], pv_done[2];
  uint32_t tmem;
  Waits waits;
  int lost;      // sums that were not finite, or large scores: go through the share again
};

ALM_DEV uint64_t sdesc128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return tc_sdesc(addr, lbo, sbo) | (static_cast<uint64_t>(2) << 61);   // SWIZZLE_128B
}
ALM_DEV void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1 : 0)
      : "memory");
}
ALM_DEV void tc_ld32(uint32_t taddr, uint32_t (&d)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7]), "=r"(d[8]),
        "=r"(d[9]), "=r"(d[10]), "=r"(d[11]), "=r"(d[12]), "=r"(d[13]), "=r"(d[14]), "=r"(d[15]), "=r"(d[16]),
        "=r"(d[17]), "=r"(d[18]), "=r"(d[19]), "=r"(d[20]), "=r"(d[21]), "=r"(d[22]), "=r"(d[23]), "=r"(d[24]),
        "=r"(d[25]), "=r"(d[26]), "=r"(d[27]), "=r"(d[28]), "=r"(d[29]), "=r"(d[30]), "=r"(d[31])
      : "r"(taddr));
}
// After tc_ld32: the values have arrived (named, so that nothing that uses
// them is moved before the wait).
ALM_DEV void tc_landed(uint32_t (&d)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]), "+r"(d[4]), "+r"(d[5]), "+r"(d[6]), "+r"(d[7]),
                 "+r"(d[8]), "+r"(d[9]), "+r"(d[10]), "+r"(d[11]), "+r"(d[12]), "+r"(d[13]), "+r"(d[14]), "+r"(d[15]),
                 "+r"(d[16]), "+r"(d[17]), "+r"(d[18]), "+r"(d[19]), "+r"(d[20]), "+r"(d[21]), "+r"(d[22]),
                 "+r"(d[23]), "+r"(d[24]), "+r"(d[25]), "+r"(d[26]), "+r"(d[27]), "+r"(d[28]), "+r"(d[29]),
                 "+r"(d[30]), "+r"(d[31])::"memory");
}
// 32 columns of 16 lanes (tensor-memory lanes of the address and the 15 behind
// it): register 4 q + 2 k + e of lane l is row l / 4 + 8 k, column 8 q + 2 (l
// mod 4) + e.  Waits for the values.
ALM_DEV void tc_ld_rows(uint32_t taddr, uint32_t (&d)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7]), "=r"(d[8]),
        "=r"(d[9]), "=r"(d[10]), "=r"(d[11]), "=r"(d[12]), "=r"(d[13]), "=r"(d[14]), "=r"(d[15])
      : "r"(taddr)
      : "memory");
}
ALM_DEV void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
ALM_DEV float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
ALM_DEV float max64(const uint32_t (&a)[32], const uint32_t (&b)[32]) {
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t* v = i < 2 ? a + 16 * i : b + 16 * (i - 2);
    t[i] = fmax3(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]));
#pragma unroll
    for (int j = 3; j < 15; j += 2) t[i] = fmax3(t[i], __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
    t[i] = fmaxf(t[i], __uint_as_float(v[15]));
  }
  return fmaxf(fmax3(t[0], t[1], t[2]), t[3]);
}
// Instruction descriptor: fp32 accumulator, A and B of type T, N wide; bmn: B
// is stored with N contiguous (V: positions by head dimensions).
template <typename T>
constexpr uint32_t tc_idesc(int n, bool bmn) {
  const uint32_t f = sizeof(T) == 2 && !std::is_same<T, half>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((bmn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

template <typename T, int HD, int NQ>
__global__ void __launch_bounds__(kTcPagedThreads, 1)
attn_paged_tc_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                     const __grid_constant__ CUtensorMap q_map,
                     const __grid_constant__ AttnPaged a, const __grid_constant__ SeqBatch b,
                     const __grid_constant__ PagedKV kv, int box_rows, int* err) {
  using S = TcShape<HD, NQ>;
  extern __shared__ char smem_raw[];
  __shared__ TcShared sh;
  const uint32_t smem0 = (smem_addr(smem_raw) + 1023) & ~1023u;
  char* const smem = smem_raw + (smem0 - smem_addr(smem_raw));
  const uint32_t ring0 = smem0 + NQ * S::kTileBytes;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int cta = blockIdx.x;
  const int tq = 128 / a.group;      // tokens a 128-row block
  const int tpu = NQ * tq;

  if (warp == 8) {
    if (lane == 0) {
      for (int i = 0; i < S::kSlots; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], NQ);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh.q_full[i], 1);
        mbar_init(&sh.q_empty[i], 3 - NQ);
        mbar_init(&sh.s_full[i], 1);
        mbar_init(&sh.p_full[i][0], 128), mbar_init(&sh.p_full[i][1], 128);
        mbar_init(&sh.pv_done[i], 1);
      }
      sh.waits.dead = sh.waits.beat = sh.lost = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tc_alloc(&sh.tmem, S::kTmemCols);
  }
  grid_dep_wait();
  grid_dep_launch();
  if (warp < 8) {
    sched_init<S::kTile>(
        b, kv, tpu, a.window, sh.sched, err,
        [&](long long total) {
          const int n = static_cast<int>(min(static_cast<long long>(a.n_cta), total));
          return cta < n ? share(total, cta, n) : -1ll;
        },
        [] { bar_sync(1, kSchedThreads); });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const long long total = sh.sched.total;
  const int n_cta = static_cast<int>(min(static_cast<long long>(a.n_cta), total));
  const long long x0 = cta < n_cta ? share(total, cta, n_cta) : 0;
  const long long x1 = cta < n_cta ? share(total, cta + 1, n_cta) : 0;

  if (tid == 0) *join_record(a, cta) = make_int4(0, 0, 0, 0);
  volatile Waits* waits = &sh.waits;
  // Waits are bounded: one that runs out marks the CTA dead, and every role leaves.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_try_wait(bar, parity & 1) || slow_wait(bar, parity & 1, waits, err);
  };
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {   // the same answer for the whole warp
    const bool ok = wait(bar, parity);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  // Each role walks this CTA's part of the line by itself.
  struct Walk {
    Unit u;
    int ta, tb;   // this CTA's tiles of the unit
    long long x1;
    // false: the share has only places without a tile
    ALM_DEV bool start(const SeqBatch& b, const PagedKV& kv, int tpu, int window, const SchedShared& sc, long long x0,
                       long long x1_) {
      x1 = x1_;
      u = unit_at<S::kTile>(b, kv, tpu, window, sc.found_seq, sc.found_at, x0);
      ta = u.from(x0);
      tb = u.upto(x1);
      return ta < tb;
    }
    ALM_DEV void next(const SeqBatch& b, const PagedKV& kv, int tpu, int window) {
      next_unit<S::kTile>(b, kv, tpu, window, u);
      ta = 0;
      tb = u.upto(x1);
    }
    ALM_DEV bool more() const { return u.more(x1); }
  };
  // The CTA goes through its share once.  It does so a second time when sums were
  // not finite though their weights were, with zeros for the infinities and NaN of
  // V, which the rows that see them then get; or when scores were beyond kFarScore,
  // and takes the maximum off them before they are scaled.  The barriers' phases
  // and the counters go on.  512 rows over 30,512 positions, 28 heads over 4 of
  // 128: 243 us, 1400 us with one infinity.  (Two copies of the code: a flag
  // instead costs the first pass 8%.)
  auto again = [&] {
    bar_sync(4, kTcPagedThreads);
    return *static_cast<volatile int*>(&sh.lost) != 0;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRestRegs));
    uint32_t fills[2] = {0, 0};   // warp 9: of each ring
    uint32_t n_q = 0;             // warp 10: units so far
    uint32_t n_p = 0, n_u = 0;    // warps 8 and 11: tiles and units of the stream so far
    auto pass = [&](auto careful) {
    Walk w;
    if (x0 < x1 && w.start(b, kv, tpu, a.window, sh.sched, x0, x1)) {
    Unit& u = w.u;
    int &ta = w.ta, &tb = w.tb;
    auto next = [&] { w.next(b, kv, tpu, a.window); };
    auto more = [&] { return w.more(); };
    if (warp == 9) {
      // ---- loads ---------------------------------------------------------------
      bool bad = false, quit = false;
      const int n_box = 128 / box_rows * S::kChunks;
      auto load = [&](const CUtensorMap* map, int t, int ring) {
        const uint32_t fill = ring == 0 ? fills[0]++ : fills[1]++;
        const int at = ring * S::kRing + fill % S::kRing;
        // one box a lane: at most 128 / 8 pieces of at most 2 column groups
        const int box = lane / S::kChunks, c = lane % S::kChunks;
        const int y = piece_row(kv, u.pages, u.h, u.n_kv, (u.t0 + t) * S::kTile + box * box_rows, lane < n_box, bad);
        if (quit || !wait_warp(&sh.empty[at], fill / S::kRing + 1)) {
          quit = true;
          return;
        }
        if (lane == 0) mbar_expect_tx(&sh.full[at], S::kTileBytes);
        __syncwarp();
        if (lane < n_box)
          tma_2d(ring0 + at * S::kTileBytes + c * (128 * 128) + box * box_rows * 128, map, c * 64, y, &sh.full[at]);
        __syncwarp();
      };
      for (bool go = true; go && !quit;) {
        for (int t = ta; t < tb; ++t) {
          load(&k_map, t, NQ == 2 ? 0 : (t - ta) & 1);
          load(&v_map, t, NQ == 2 ? 0 : (t - ta) & 1);
        }
        go = more();
        if (go) next();
      }
      if (bad) *err = 1;
      // whatever happened, no copy is in flight when the CTA leaves: a slot's
      // last fill is complete once its barrier has left that phase
      if (quit) {
        for (int i = 0; i < S::kSlots; ++i) {
          mbar_wait(&sh.full[i], 0);
          mbar_wait(&sh.full[i], 1);
        }
      }
    } else if (warp == 10) {
      // ---- Q: the tokens' heads of one K/V head are a box (columns, heads,
      // tokens), which is the packed order of the block's rows; tokens of the
      // next sequence that it may hold fill rows that nothing is written from
      const uint32_t bytes = static_cast<uint32_t>(tq * a.group) * 128 * S::kChunks;
      bool quit = false;
      for (bool go = true; go && !quit; ++n_q) {
        for (int i = 0; i < NQ && !quit; ++i) {
          if (!wait_warp(&sh.q_empty[i], n_q ^ 1)) {
            quit = true;
            break;
          }
          if (lane == 0) {
            mbar_expect_tx(&sh.q_full[i], bytes);
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
              tma_3d(smem0 + i * S::kTileBytes + c * (128 * 128), &q_map, c * 64, u.h * a.group, u.row0 + i * tq,
                     &sh.q_full[i]);
          }
          __syncwarp();
        }
        go = more();
        if (go) next();
      }
      if (quit)
        for (int i = 0; i < NQ; ++i) mbar_wait(&sh.q_full[i], 0), mbar_wait(&sh.q_full[i], 1);
    } else {
      // ---- products of stream i (the whole warp walks, one lane issues) ----------
      const int i = warp == 8 ? 0 : 1;
      constexpr int kStep = NQ == 2 ? 1 : 2;           // the stream's tiles of a unit: every, or every second
      const int q_blk = NQ == 2 ? i : 0;
      const uint32_t id_s = tc_idesc<T>(128, false), id_o = tc_idesc<T>(HD, true);
      const uint32_t qa = smem0 + q_blk * S::kTileBytes;
      const uint32_t d_s = tmem + S::kColS + i * 128, d_o = tmem + S::kColO + i * HD;
      // K and V of the stream's n-th tile are fills 2 n and 2 n + 1 of its ring
      const uint32_t ring = NQ == 2 ? 0 : i * S::kRing;
      int t = ta, t_first = ta;
      bool quit = false;
      auto ready = [&](uint64_t* bar, uint32_t parity) {
        if (!quit && !wait_warp(bar, parity)) quit = true;
        tc_fence_after();
      };
      // K tile of the stream's n-th tile
      auto k_ready = [&](uint32_t n) { ready(&sh.full[ring + 2 * n % S::kRing], 2 * n / S::kRing); };
      // S = Q . K^T of tile t, whose K is there.  One commit tells that all
      // products so far are done, the last P . V among them; then its K (and a V
      // that is done with) may go, and after the unit's last so may Q.
      auto qk = [&](int v_slot) {
        if (quit || !elect_one()) return;
        const uint32_t at = ring + 2 * n_p % S::kRing, ka = ring0 + at * S::kTileBytes;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = (k / 4) * (128 * 128) + (k % 4) * 32;
          tc_mma_ss(d_s, sdesc128(qa + off, 16, 1024), sdesc128(ka + off, 16, 1024), id_s, k > 0);
        }
        tc_commit(&sh.s_full[i]);
        tc_commit(&sh.empty[at]);
        if (v_slot >= 0) tc_commit(&sh.empty[v_slot]);
        if (t + kStep >= tb) tc_commit(&sh.q_empty[q_blk]);
      };
      // O += P . V of tile t in two halves of 64 positions: the first product
      // runs while the second half's weights are made.  Returns V's slot.
      auto pv = [&](bool last) {
        const uint32_t fill = 2 * n_p + 1, at = ring + fill % S::kRing;
        ready(&sh.full[at], fill / S::kRing);
        const int base = (u.t0 + t) * S::kTile, r0 = u.n_kv - base;
        if (r0 < S::kTile && r0 > 0 && !quit) {
          // The sequence ends in this tile, and its last page piece goes on
          // behind it: those rows hold anything, and a zero weight times NaN
          // is NaN.  (Both streams of a shared tile write the same zeros.)
          const int r1 = (r0 + box_rows - 1) / box_rows * box_rows;   // box_rows divides the tile
          char* v = smem + (NQ + at) * S::kTileBytes;
          for (int j = lane; j < (r1 - r0) * 8; j += kWarp)
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
              *reinterpret_cast<uint4*>(v + c * (128 * 128) + (r0 + j / 8) * 128 + (j % 8) * 16) =
                  make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (decltype(careful)::value && !quit) {   // (both streams of a shared tile write the same zeros here too)
          uint4* v = reinterpret_cast<uint4*>(smem + (NQ + at) * S::kTileBytes);
#pragma unroll 4
          for (int j = lane; j < S::kTileBytes / 16; j += kWarp) {
            const uint4 x = v[j];
            const uint4 y = make_uint4(finite_only<T>(x.x), finite_only<T>(x.y), finite_only<T>(x.z), finite_only<T>(x.w));
            if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) v[j] = y;
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        // the next tile's K before the weights: it is there long since, and
        // then nothing stands between this product and the next
        if (!last) k_ready(n_p + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ready(&sh.p_full[i][h], n_p);
          if (quit) return -1;
          if (elect_one()) {
            const uint32_t va = ring0 + at * S::kTileBytes;
#pragma unroll
            for (int k = 4 * h; k < 4 * h + 4; ++k)   // 16 positions: two groups of 8 rows of 128 bytes
              tc_mma_ts(d_o, d_s + 8 * k, sdesc128(va + k * 2048, 128 * 128, 1024), id_o, t > t_first || k > 0);
            if (last && h == 1) {
              tc_commit(&sh.pv_done[i]);
              tc_commit(&sh.empty[at]);
            }
          }
        }
        ++n_p;
        return static_cast<int>(at);
      };
      // the stream's first tile of this unit or a later one; false: there is none
      auto enter = [&] {
        for (;;) {
          t = t_first = NQ == 2 ? ta : ta + i;
          ready(&sh.q_full[q_blk], n_u++);
          if (quit) return false;
          if (t < tb) return true;
          if (lane == 0) mbar_arrive(&sh.q_empty[q_blk]);   // reads nothing of this Q
          if (!more()) return false;
          next();
        }
      };
      bool go = enter();
      if (go) {
        k_ready(n_p);
        qk(-1);
      }
      while (go && !quit) {
        if (t + kStep < tb) {
          const int v_slot = pv(false);
          t += kStep;
          qk(v_slot);
        } else {
          pv(true);
          if (!more()) break;
          next();
          go = enter();
          if (go) {
            k_ready(n_p);
            qk(-1);
          }
        }
      }
    }
    }
    };
    pass(std::false_type());
    if (again()) pass(std::true_type());
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int st = warp / 4;                         // stream
    uint32_t n_s = 0;                                // tiles of this stream so far
    uint32_t n_u = 0, n_done = 0;                    // units so far, and those with a tile
    if (NQ == 2 && st == 1) bar_arrive(2, 256);      // stream 0 has the first turn
    auto pass = [&](auto careful) {
    Walk w;
    if (x0 < x1 && w.start(b, kv, tpu, a.window, sh.sched, x0, x1)) {
      Unit& u = w.u;
      int &ta = w.ta, &tb = w.tb;
      auto next = [&] { w.next(b, kv, tpu, a.window); };
      auto more = [&] { return w.more(); };
      // ---- softmax -------------------------------------------------------------
      const int r = tid % 128;                         // row of the block = lane of tensor memory
      const uint32_t t_s = tc_addr(tmem + S::kColS + st * 128, (warp % 4) * 32, 0);
      const uint32_t t_o = tc_addr(tmem + S::kColO + st * HD, (warp % 4) * 32, 0);
      const int blk = NQ == 2 ? st : 0;                // 128-row block of the unit
      for (bool go = true; go;) {
        const Unit cu = u;
        const int ca = ta, cb = tb;
        go = more();
        if (go) next();                                  // early: its lengths are loads
        const int tk = r / a.group, tok = blk * tq + tk, head = cu.h * a.group + r - tk * a.group;
        const bool live = tk < tq && tok < cu.n_tok;
        const int hi = live ? max(cu.pos0 + tok, -1) : -1;   // last position the row sees
        // of the block: the first token's position and the last's
        const int pos_a = cu.pos0 + blk * tq, pos_b = max(min(pos_a + tq, cu.pos0 + cu.n_tok) - 1, -1);
        const bool any_live = __any_sync(0xffffffffu, live);
        float m = kNegInf, l = 0.f;
        int n_mine = 0;
        for (int t = ca + (NQ == 1 ? st : 0); t < cb; t += NQ == 1 ? 2 : 1) {
          wait_warp(&sh.s_full[st], n_s);
          tc_fence_after();
          if (!any_live) {
            if (NQ == 2) bar_sync(2 + st, 256);
            mbar_arrive(&sh.p_full[st][0]);
            mbar_arrive(&sh.p_full[st][1]);
            if (NQ == 2) bar_arrive(3 - st, 256);
          } else {
            uint32_t sr[4][32];
            tc_ld32(t_s, sr[0]);
            tc_ld32(t_s + 32, sr[1]);
            const int p0 = (cu.t0 + t) * S::kTile;
            const bool mask = p0 + S::kTile - 1 > pos_a || (a.window > 0 && p0 <= pos_b - a.window);
            // columns > n_hi, and with a window <= n_lo, are hidden
            const int n_hi = hi - p0, n_lo = max(n_hi, -1) - a.window;
            auto hide = [&](int h) {
#pragma unroll
              for (int i = 64 * h; i < 64 * h + 64; ++i)
                sr[i / 32][i % 32] = i > n_hi ? 0xff800000u : sr[i / 32][i % 32];
              if (a.window > 0) {
#pragma unroll
                for (int i = 64 * h; i < 64 * h + 64; ++i)
                  sr[i / 32][i % 32] = i <= n_lo ? 0xff800000u : sr[i / 32][i % 32];
              }
            };
            tc_landed(sr[0]);
            tc_landed(sr[1]);
            tc_ld32(t_s + 64, sr[2]);
            tc_ld32(t_s + 96, sr[3]);
            if (mask) hide(0);
            float row_top = max64(sr[0], sr[1]);
            tc_landed(sr[2]);
            tc_landed(sr[3]);
            if (mask) hide(1);
            row_top = fmaxf(row_top, max64(sr[2], sr[3]));
            // (m moves rarely: no test in every tile; rows behind the block's tokens hold anything)
            auto note_far = [&] {
              if (!decltype(careful)::value && live && m != kNegInf && fabsf(m * a.scale_log2) > kFarScore) sh.lost = 1;
            };
            if (n_mine == 0) {
              m = row_top;
              note_far();
            } else {
              const bool grow = row_top > m && !((row_top - m) * a.scale_log2 <= kSlack);
              if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2((m - row_top) * a.scale_log2) : 1.f;
                if (grow) m = row_top;
                note_far();
                l *= f;
                // (the scores' commit covers the product before them, so O is at rest)
#pragma unroll 1
                for (int c = 0; c < HD / 16; ++c) {
                  uint32_t ov[16];
                  tc_ld16(t_o + 16 * c, ov);
                  tc_wait_ld();
#pragma unroll
                  for (int j = 0; j < 16; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * f);
                  tc_st16(t_o + 16 * c, ov);
                }
              }
            }
            const float base = m == kNegInf ? 0.f : m, mc = base * a.scale_log2;
            const uint64_t c2 = pair(a.scale_log2, a.scale_log2);
            const uint64_t m2 = decltype(careful)::value ? pair(-base, -base) : pair(-mc, -mc);
            uint64_t sum[2] = {0, 0};   // (+0, +0)
            uint32_t pr[2][32];
            auto weights = [&](int h, int j0, int j1) {
#pragma unroll
              for (int j = j0; j < j1; ++j) {
                const int e = 64 * h + 2 * j;
                float p, q;
                const uint64_t s2 = pair(__uint_as_float(sr[e / 32][e % 32]), __uint_as_float(sr[e / 32][e % 32 + 1]));
                unpair(decltype(careful)::value ? mul2(add2(s2, m2), c2) : fma2(s2, c2, m2), p, q);
                p = ex2(p);
                q = ex2(q);
                sum[j & 1] = add2(sum[j & 1], pair(p, q));
                pr[h][j] = Elem<T>::pack(p, q);
              }
            };
            // The streams take turns at the exponentials: together they would
            // share that unit first and the tensor core afterwards.  A turn is
            // filled with them: the first half's weights leave while the
            // second's are made.
            if (NQ == 2) bar_sync(2 + st, 256);
            weights(0, 0, 32);
            tc_st32(t_s, pr[0]);
            weights(1, 0, 12);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&sh.p_full[st][0]);
            weights(1, 12, 32);
            if (NQ == 2) bar_arrive(3 - st, 256);
            tc_st32(t_s + 32, pr[1]);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&sh.p_full[st][1]);
            float s0, s1, s2, s3;
            unpair(sum[0], s0, s1);
            unpair(sum[1], s2, s3);
            l += (s0 + s1) + (s2 + s3);
          }
          ++n_s;
          ++n_mine;
        }

        // ---- the unit's end ------------------------------------------------------
        if (n_mine > 0) {
          wait_warp(&sh.pv_done[st], n_done++);
          tc_fence_after();
        }
        const bool whole = ca == 0 && cb == cu.n_tile;
        float* part = partial_at<HD>(a.work, NQ * 128, cta, ca == 0 ? 1 : 0);
        if (tid == 0 && !whole && ca == 0) *join_record(a, cta) = record_of(cu, cta, n_cta, total);
        // stream 1 of a single block leaves its sums in global memory for
        // stream 0, in two places in turn: one is read while the next is written
        float* half_sum = NQ == 1 ? partial_at<HD>(a.work, 128, a.n_cta + cta, n_u++ & 1) : nullptr;
        const bool two = NQ == 1 && cb - ca >= 2;
        if (NQ == 1 && st == 1) {
          if (two) {
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t ov[16];
                tc_ld_rows(t_o + (16u << 16) * hh + 32 * c, ov);
#pragma unroll
                for (int j = 0; j < 16; ++j) half_sum[((hh * (HD / 32) + c) * 16 + j) * 128 + r] = __uint_as_float(ov[j]);
              }
            half_sum[128 * HD + r] = m;
            half_sum[128 * HD + 128 + r] = l;
          }
          tc_fence_before();
          bar_sync(2, 256);
          continue;
        }
        float f0 = 1.f, f1 = 0.f;
        if (NQ == 1) {
          bar_sync(2, 256);
          if (two) {
            const float m1 = half_sum[128 * HD + r], l1 = half_sum[128 * HD + 128 + r];
            const float mm = fmaxf(m, m1), base = mm == kNegInf ? 0.f : mm;
            f0 = ex2((m - base) * a.scale_log2);
            f1 = ex2((m1 - base) * a.scale_log2);
            l = l * f0 + l1 * f1;
            m = mm;
          }
        }
        const bool none = m == kNegInf && l == 0.f;
        const float inv = whole ? (none ? 0.f : 1.f / l) : 1.f;
        const float w0 = f0 * inv, w1 = f1 * inv;
        char* dst = a.out + (cu.row0 + tok) * a.out_row + head * a.out_head;
        const int prow = blk * 128 + r;
        // Rows leave through the load that spreads a row over four lanes (two
        // columns of every eight each), so that a store covers whole 32-byte
        // sectors of 8 rows instead of half ones of 32.
        unsigned mine4 = 0;   // four lanes speak for a row: those of this lane's
        if (any_live) {
          const unsigned live_rows = __ballot_sync(0xffffffffu, live);
          const int g = lane / 4, t4 = lane % 4;
#pragma unroll 1   // (unrolled, the loops above get fewer registers: a prefill takes 2% longer)
          for (int hh = 0; hh < 2; ++hh) {
            char* d[2];        // of rows 16 hh + g and 16 hh + g + 8
            float s0[2], s1[2], zero[2] = {0.f, 0.f};
            bool on[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int src = 16 * hh + g + 8 * k;
              d[k] = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), src));
              s0[k] = __shfl_sync(0xffffffffu, w0, src);
              s1[k] = NQ == 1 ? __shfl_sync(0xffffffffu, w1, src) : 0.f;
              on[k] = (live_rows >> src) & 1;
              if (!whole) d[k] = reinterpret_cast<char*>(part + (prow - lane + src) * HD);
            }
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t ov[16];
              tc_ld_rows(t_o + (16u << 16) * hh + 32 * c, ov);
              float o[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                o[j] = __uint_as_float(ov[j]) * s0[(j >> 1) & 1];
                if (two) o[j] = fmaf(half_sum[((hh * (HD / 32) + c) * 16 + j) * 128 + r], s1[(j >> 1) & 1], o[j]);
                zero[(j >> 1) & 1] = fmaf(0.f, o[j], zero[(j >> 1) & 1]);   // NaN if any is NaN or infinite
              }
              if (whole) {
#pragma unroll
                for (int q = 0; q < 4; q += 2)     // columns 32 c + 8 q .. + 15 of both rows
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    const uint32_t x0 = Elem<T>::pack(o[4 * q + 2 * k], o[4 * q + 2 * k + 1]);
                    const uint32_t x1 = Elem<T>::pack(o[4 * q + 4 + 2 * k], o[4 * q + 5 + 2 * k]);
                    // four neighbouring columns a lane: lanes 0, 1 the first eight, 2, 3 the others
                    const uint32_t y = __shfl_xor_sync(0xffffffffu, (t4 & 2) ? x0 : x1, 2);
                    const uint32_t lo = (t4 & 2) ? y : x0, hi2 = (t4 & 2) ? x1 : y;
                    const uint32_t z = __shfl_xor_sync(0xffffffffu, (t4 & 1) ? lo : hi2, 1);
                    if (on[k])
                      *reinterpret_cast<uint2*>(d[k] + (32 * c + 8 * q + 4 * t4) * 2) =
                          (t4 & 1) ? make_uint2(z, hi2) : make_uint2(lo, z);
                  }
              } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                  for (int k = 0; k < 2; ++k)
                    if (on[k])
                      *reinterpret_cast<float2*>(d[k] + (32 * c + 8 * q + 2 * t4) * 4) =
                          make_float2(o[4 * q + 2 * k], o[4 * q + 2 * k + 1]);
              }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const unsigned spoilt = __ballot_sync(0xffffffffu, zero[k] != 0.f);
              if (lane / 16 == hh && lane / 8 % 2 == k) mine4 = spoilt;
            }
          }
        }
        const bool odd = ((mine4 >> (4 * (lane & 7))) & 15u) != 0;
        tc_fence_before();
        if (live) {
          if (!whole) {
            part[NQ * 128 * HD + prow] = m;
            part[NQ * 128 * HD + NQ * 128 + prow] = l;
          } else if (a.lse) {
            a.lse[(cu.row0 + tok) * a.lse_row + head] =
                none ? kNegInf : (m * a.scale_log2 + log2f(l)) * 0.693147180559945309f;
          }
        }
        // (a NaN score spoils its whole row)
        if (!decltype(careful)::value && odd && live && l == l) sh.lost = 1;
        if (decltype(careful)::value && any_live) {
          __syncwarp();   // the warp's rows lie in memory
          mend_rows<T, HD>(a, kv, cu.pages, cu.h, cu.row0 + blk * tq, pos_a, r - lane, 1,
                           __ballot_sync(0xffffffffu, live && l == l), m, inv, (cu.t0 + ca) * S::kTile,
                           (cu.t0 + cb) * S::kTile, whole ? nullptr : part + blk * 128 * HD, waits);
        }
      }
    }
    };
    pass(std::false_type());
    if (again()) pass(std::true_type());
  }
  // a wait that ran out has left products in flight: give them time, then free
  __syncthreads();
  if (waits->dead && tid == 0) {
    mbar_wait(&sh.pv_done[0], 0), mbar_wait(&sh.pv_done[0], 1);
    mbar_wait(&sh.pv_done[1], 0), mbar_wait(&sh.pv_done[1], 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tc_dealloc(tmem, S::kTmemCols);
  }
}

// ---- host --------------------------------------------------------------------
// What the tensor-core kernels take: pages that TMA reads, and Q strides that
// are positive and below 2^40 bytes, as a tensor map's have to be.
inline bool tc_paged_fits(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv) {
  auto stride = [](int64_t bytes, int n) { return n <= 1 || (bytes > 0 && bytes < (1ll << 40)); };
  return tma_pages(kv) && stride(a.q_head, a.heads) && stride(a.q_row, b.n_rows);
}

// Q as (columns, heads, rows): boxes of 64 columns x the heads of one K/V head
// x the tokens of a block.
template <typename T>
bool encode_q(CUtensorMap* map, const AttnPaged& a, const SeqBatch& b, int head_dim) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = cu_tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(a.heads),
                        static_cast<cuuint64_t>(b.n_rows)};
  // (a stride that nothing is stepped with may be 0)
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.heads > 1 ? a.q_head : head_dim * 2),
                           static_cast<cuuint64_t>(b.n_rows > 1 ? a.q_row : head_dim * 2)};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(128 / a.group)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, std::is_same<T, half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
             const_cast<char*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, int NQ>
cudaError_t launch_tc(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int* err, cudaStream_t st) {
  using S = TcShape<HD, NQ>;
  CUtensorMap km, vm, qm;
  const int box = page_box_rows(kv);
  if (!encode_pages<T>(&km, kv.k, kv, box) || !encode_pages<T>(&vm, kv.v, kv, box) ||
      !encode_q<T>(&qm, a, b, HD))
    return cudaErrorInvalidValue;
  OpLaunch l(dim3(a.n_cta, 1, 1), kTcPagedThreads, S::kSmem, st);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, attn_paged_tc_kernel<T, HD, NQ>, km, vm, qm, a, b, kv, box, err);
  return e != cudaSuccess ? e : launch_join<T, HD, NQ * 128, 128>(a, st);
}

template <typename T>
cudaError_t launch_tc_t(const AttnPaged& a, const SeqBatch& b, const PagedKV& kv, int nq, int* err, cudaStream_t st) {
  if (kv.head_dim == 64)
    return nq == 2 ? launch_tc<T, 64, 2>(a, b, kv, err, st) : launch_tc<T, 64, 1>(a, b, kv, err, st);
  return nq == 2 ? launch_tc<T, 128, 2>(a, b, kv, err, st) : launch_tc<T, 128, 1>(a, b, kv, err, st);
}

template <typename T>
cudaError_t tc_paged_attrs() {
  auto set = [](auto* f, size_t n) {
    return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(n));
  };
  cudaError_t e = set(attn_paged_tc_kernel<T, 64, 1>, TcShape<64, 1>::kSmem);
  if (e == cudaSuccess) e = set(attn_paged_tc_kernel<T, 64, 2>, TcShape<64, 2>::kSmem);
  if (e == cudaSuccess) e = set(attn_paged_tc_kernel<T, 128, 1>, TcShape<128, 1>::kSmem);
  if (e == cudaSuccess) e = set(attn_paged_tc_kernel<T, 128, 2>, TcShape<128, 2>::kSmem);
  return e;
}

}  // namespace alm

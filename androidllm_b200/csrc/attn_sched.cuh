// How the paged attention kernels share a ragged batch among their CTAs.
//
// A unit is (sequence, block of up to `tpu` tokens, K/V head): its rows are
// the tokens' query heads of that K/V head, its work the TILE-position tiles
// its rows can see (one at least, so that rows that see nothing are written).
// All units, in the order sequence, token block, head, lie on one line of T
// places: kUnitCost places for what a unit costs beside its tiles (its first
// scores, its result), then one a tile.  CTA i of n takes the tiles of places
// [T i / n, T (i + 1) / n).  Every CTA gets the same share whatever the lengths
// are, with lengths that only the device knows, and the split points depend on
// nothing but the batch, so results do not change from run to run.  A unit cut
// by a share's end leaves one partial result per CTA; a CTA owns at most two of
// those (its first and last unit).
#pragma once
#include "paged.cuh"

namespace alm {

constexpr int kSchedThreads = 256;   // threads that run sched_init (warps 0 .. 7)
// In tiles.  0 / 1 / 2 / 4 take 371 / 302 / 268 / 268 us at 4 x 2047 rows, 62 /
// 38.1 / 38.8 / 44.3 us at 64 decodes, 27.7 / 27.5 / 26.1 / 27.8 us at 9 chunks
// of 1 to 701 rows.
constexpr int kUnitCost = 2;

struct Unit {
  int s, mb, h;       // sequence, token block, K/V head
  int row0;           // first packed row
  int n_tok;          // tokens in the block
  int pos0;           // position of the first token (may be negative)
  int n_kv;           // positions of the sequence
  const int* pages;
  int t0, n_tile;     // first tile and number of tiles
  long long start;    // place of the first tile on the line (kUnitCost places after the unit's)
  // whether the share's end x1 leaves tiles for a unit behind this one
  ALM_DEV bool more(long long x1) const { return start + n_tile + kUnitCost < x1; }
  // its tiles in a share [x0, x1): [from(x0), upto(x1))
  ALM_DEV int from(long long x0) const { return x0 > start ? static_cast<int>(min(x0 - start, static_cast<long long>(n_tile))) : 0; }
  ALM_DEV int upto(long long x1) const { return x1 > start ? static_cast<int>(min(x1 - start, static_cast<long long>(n_tile))) : 0; }
};

struct SchedShared {
  long long warp_sum[kSchedThreads / kWarp];
  long long total, goal;
  long long found_at;   // line place where the found sequence starts
  int found_seq;
};

// Tiles of token block mb (n_new rows, tpu tokens a block).
template <int TILE>
ALM_DEV void block_tiles(const Seq& q, int tpu, int window, int mb, int& t0, int& n_tile) {
  const int first = q.n_kv - q.n_new + mb * tpu;
  const int last = min(first + tpu, q.n_kv) - 1;   // last token's position, n_kv - 1 at most
  const int lo = window > 0 && first >= window ? first - window + 1 : 0;   // (first may be far below 0)
  t0 = lo / TILE;
  n_tile = last < 0 ? 1 : last / TILE - t0 + 1;
  if (last < 0) t0 = 0;
}

// Places of one K/V head of sequence q, by one thread.
template <int TILE>
ALM_DEV long long seq_tiles(const Seq& q, int tpu, int window) {
  long long n = 0;
  for (int mb = 0; mb * tpu < q.n_new; ++mb) {
    int t0, nt;
    block_tiles<TILE>(q, tpu, window, mb, t0, nt);
    n += nt + kUnitCost;
  }
  return n;
}

// Sequences with at least this many token blocks are summed by a whole warp.
constexpr int kManyBlocks = 8;

// The line's length and the sequence that holds place goal(total): every one
// of the first kSchedThreads threads calls it; sync() is their barrier.  The
// first CTA reports sequences that their row of the table does not hold.
template <int TILE, typename Goal, typename Sync>
ALM_DEV void sched_init(const SeqBatch& b, const PagedKV& kv, int tpu, int window, SchedShared& sh, int* err, Goal goal,
                        Sync sync) {
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  // thread t sums sequences [t per, (t + 1) per); per is 1 up to 256 sequences
  const int per = (b.n_seq + kSchedThreads - 1) / kSchedThreads;
  auto tiles_of = [&](int s) {   // by the whole warp, one sequence a lane
    Seq q;
    q.n_new = 0;
    q.n_kv = 0;
    q.fits = true;
    if (s < b.n_seq) q = load_seq(b, kv, s);
    const bool in = q.n_new > 0;
    if (in && !q.fits && blockIdx.x == 0) *err = 1;
    const bool many = in && q.n_new > kManyBlocks * tpu;
    long long n = in && !many ? seq_tiles<TILE>(q, tpu, window) : 0;
    unsigned todo = __ballot_sync(0xffffffffu, many);
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      Seq w;
      w.n_new = __shfl_sync(0xffffffffu, q.n_new, src);
      w.n_kv = __shfl_sync(0xffffffffu, q.n_kv, src);
      long long part = 0;
      for (int mb = lane; mb * tpu < w.n_new; mb += kWarp) {
        int t0, nt;
        block_tiles<TILE>(w, tpu, window, mb, t0, nt);
        part += nt + kUnitCost;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == src) n = part;
    }
    return n * kv.kv_heads;
  };
  long long mine = 0;
  for (int i = 0; i < per; ++i) mine += tiles_of(min(tid * per + i, b.n_seq) );
  long long scan = mine;
#pragma unroll
  for (int o = 1; o < kWarp; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += v;
  }
  if (lane == kWarp - 1) sh.warp_sum[warp] = scan;
  sync();
  long long before = scan - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kSchedThreads / kWarp; ++w) {
    const long long v = sh.warp_sum[w];
    if (w < warp) before += v;
    total += v;
  }
  const long long g = goal(total);
  if (tid == 0) sh.total = total;
  // the owner's warp walks the owner's sequences (one when per is 1)
  const bool own = mine > 0 && g >= before && g < before + mine;
  const unsigned owner = __ballot_sync(0xffffffffu, own);
  if (owner) {
    const int src = __ffs(owner) - 1;
    const int s0 = __shfl_sync(0xffffffffu, tid * per, src);
    long long at = __shfl_sync(0xffffffffu, before, src);
    if (per == 1) {
      if (lane == 0) sh.found_seq = s0, sh.found_at = at;
    } else {
      // lane l takes sequence s0 + l; per is at most 4096 / 256 = 16 < 32
      const long long n = tiles_of(lane < per ? min(s0 + lane, b.n_seq) : b.n_seq);
      long long sc = n;
#pragma unroll
      for (int o = 1; o < kWarp; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sc, o);
        if (lane >= o) sc += v;
      }
      if (n > 0 && g >= at + sc - n && g < at + sc) sh.found_seq = s0 + lane, sh.found_at = at + sc - n;
    }
  }
  sync();
}

// The unit of sequence s (which starts at line place `at`) that holds place
// g, by a whole warp: token blocks 32 at a time.
template <int TILE>
ALM_DEV Unit unit_at(const SeqBatch& b, const PagedKV& kv, int tpu, int window, int s, long long at, long long g) {
  const int lane = threadIdx.x % kWarp;
  const Seq q = load_seq(b, kv, s);
  Unit u;
  u.s = s;
  u.mb = 0;
  for (int mb0 = 0; mb0 * tpu < q.n_new; mb0 += kWarp) {
    const int mb = mb0 + lane;
    int t0 = 0, nt = 0;
    if (mb * tpu < q.n_new) block_tiles<TILE>(q, tpu, window, mb, t0, nt);
    long long sc = nt > 0 ? static_cast<long long>(nt + kUnitCost) * kv.kv_heads : 0;
    const long long mine = sc;
#pragma unroll
    for (int o = 1; o < kWarp; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, sc, o);
      if (lane >= o) sc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, mine > 0 && g < at + sc);
    if (hit) {
      const int src = __ffs(hit) - 1;
      u.mb = mb0 + src;
      at = __shfl_sync(0xffffffffu, at + sc - mine, src);
      break;
    }
    at += __shfl_sync(0xffffffffu, sc, kWarp - 1);
  }
  block_tiles<TILE>(q, tpu, window, u.mb, u.t0, u.n_tile);
  u.h = min(static_cast<int>((g - at) / (u.n_tile + kUnitCost)), kv.kv_heads - 1);
  u.start = at + static_cast<long long>(u.h) * (u.n_tile + kUnitCost) + kUnitCost;
  u.row0 = q.row0 + u.mb * tpu;
  u.n_tok = min(tpu, q.n_new - u.mb * tpu);
  u.pos0 = q.n_kv - q.n_new + u.mb * tpu;
  u.n_kv = q.n_kv;
  u.pages = q.pages;
  return u;
}

// The next unit on the line (there is one).
template <int TILE>
ALM_DEV void next_unit(const SeqBatch& b, const PagedKV& kv, int tpu, int window, Unit& u) {
  u.start += u.n_tile + kUnitCost;
  if (++u.h < kv.kv_heads) return;
  u.h = 0;
  Seq q = load_seq(b, kv, u.s);
  ++u.mb;
  while (u.mb * tpu >= q.n_new) {
    u.mb = 0;
    ++u.s;
    if (u.s >= b.n_seq) return;   // behind the line's end: the caller does not use it
    q = load_seq(b, kv, u.s);
  }
  block_tiles<TILE>(q, tpu, window, u.mb, u.t0, u.n_tile);
  u.row0 = q.row0 + u.mb * tpu;
  u.n_tok = min(tpu, q.n_new - u.mb * tpu);
  u.pos0 = q.n_kv - q.n_new + u.mb * tpu;
  u.n_kv = q.n_kv;
  u.pages = q.pages;
}

// Share of CTA i of n on a line of `total` tiles.
ALM_DEV long long share(long long total, int i, int n) { return total * i / n; }

}  // namespace alm

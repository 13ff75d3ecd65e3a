// paged_tile.cu -- attention over a paged K/V cache for many rows per key, on the tensor cores.
//
// Two uses, one kernel:
//   * a batch that shares a prefix: the rows of all sequences (sequence, query head of the group,
//     token) are stacked into tiles of 128 over the prefix's keys, which are read once per tile of
//     rows instead of once per sequence.  Everything it computes is partial (the sequences' own
//     keys follow elsewhere): normalised o and log2 of the sum, in 32 bits;
//   * many new tokens of one sequence (drafts, a chunk of a prompt): tiles of rows of one sequence,
//     whose key tiles end at the last row's position.
// Per tile of 128 rows x 128 keys: 4 * 128^3 operations against 64 KB of keys and values, so full
// tiles of rows are bound by the tensor cores and the exponentials, sparse ones by memory.
//
// The work is cut like the few-row kernel's: the key tiles of all (tile of rows, K/V head) items
// form one line in equal pieces, one per CTA.  A CTA is a pipeline of sixteen warps:
//   warp 0, 3   producers of Q and K, and of V, by TMA: one box per page and 64-column half, the
//               lanes of a warp issuing the boxes of a tile.  The page table is read one tile ahead.
//               With small pages the issue of the boxes is what bounds a producer, hence two.  Rows
//               of V behind the sequence's end (recycled slots may hold NaN, and 0 * NaN is NaN) are
//               overwritten with zeros in shared memory once the copy has landed, before the tile is
//               handed on; rows of K need not be, their scores are masked;
//   warp 1, 2   tcgen05 issuers of P V and of Q K^T;
//   warps 4-11  softmax, two warpgroups, keys 0..63 and 64..127 of every tile: thread t owns row t.
//               They exchange row maxima through shared memory; the running maximum moves only when
//               passed by more than 2^8, and O is rescaled in tensor memory only then;
//   warps 12-15 epilogue: o = O / l, to o (a whole item) or to the partial buffer, which is laid out
//               [32 pieces of four columns][128 rows] so that the threads of a warp, one row each,
//               write side by side.
// P is rounded to the type of V, as in the few-row kernel; everything else is held in 32 bits.
// Tensor memory: S[2] at columns 0 and 128 (P overwrites S), O[2] at 256 and 384.  Every wait is
// bounded; on expiry all roles leave, copies and MMAs in flight are drained and the call reports
// BSATTN_E_TIMEOUT.
#include <cuda.h>

#include <algorithm>

#include "paged_tile.cuh"
#include "sm100_ptx.cuh"

namespace bsattn {
namespace paged {
namespace tile {

constexpr int kRows = 128;
// Two tiles of K and of V each, and two of Q.  A third of V in place of the second Q was measured: it
// does not help where the keys come from HBM (that is what bounds it then) and costs 2 % elsewhere.
constexpr int kStages = 2;
constexpr int kTileBytes = kTileKeys * kHeadDim * 2;  // 32 KB
constexpr int kHalfBytes = kTileBytes / 2;            // 128 rows x 64 columns, 128-byte swizzle
constexpr int kThreads = 512;
constexpr int kSoftmaxWarp0 = 4, kEpiWarp0 = 12;
constexpr uint32_t kTmemCols = 512, kOCol = 256;
constexpr float kRescaleLog2 = 8.0f;
constexpr float kNoMax = -3e38f;        // running maximum before the first visible key
constexpr float kNoMaxBelow = -2.9e38f;
// The exponent is one FMA, score * scale - maximum, and the maximum is that product rounded, so the largest
// exponent is what the rounding lost: from 2^28 on up to 16 and more, where P would pass what fp16 holds.
// Past 2^27 a row's unit is therefore the next power of two above the scale, whose products are exact.
// That makes weights steeper by less than twice where 32-bit scores lie 8 apart and are themselves off by
// more.  (117.3 us for 2 x 512 tokens over 8,192 keys without it, 117.5 with it; rounding the products of
// such rows first, behind a vote of the warp, 121.)
constexpr float kFar = 134217728.0f;
constexpr int kPolyEvery = 4;           // every 4th pair of exponentials runs on the FMA pipe
constexpr unsigned long long kDrainNs = 100000000ull;  // floor of the teardown waits
constexpr int kRing = 8;
constexpr int kRingReaders = 256 + 128 + 3;  // softmax, epilogue, S issuer, PV issuer, V stream
// Register split of the 512 x 128 launch registers: the shares per warpgroup sum to 4 x 128.
constexpr uint32_t kLaunchRegs = 128, kSoftmaxRegs = 168, kControlRegs = 88, kEpilogueRegs = 88;
static_assert(2 * kSoftmaxRegs + kControlRegs + kEpilogueRegs <= 4 * kLaunchRegs,
              "register split exceeds the launch allocation");

struct Params {
  Cache c;
  Rule rule;
  RowTiles rt;
  int prefix_len;
  int page_size, box_rows, box_shift, boxes;  // rows of one box (log2), boxes per 64-column half of a tile
  void* o;
  float* lse;
  int Hq;
  float scale_log2;
  int out_bf16;
  TileCut* cuts;
  float* part_o;
  float* part_l;
  unsigned long long timeout_ns;
  int test_wait;  // test hook: the Q K^T issuer first waits on a barrier that nothing signals
};

// A piece of an item: steps tile0 .. tile0 + n - 1 of virtual sequence v, K/V head h.
struct Seg {
  int v, h, tile0, n;
  int b0, t0;          // first sequence and first token of the tile of rows
  int first, rows;     // of sequence b0 (one-sequence tiles)
  int load_end;        // keys from here on hold nothing
  int n_glob, lo_block;
  int whole;
};

// The key tiles of virtual sequence v: those its last live row sees, at least one.
struct VTiles {
  int b0, t0, n;
  int len, n_glob, lo_block;
  Rows r;
};

struct alignas(1024) Smem {
  uint8_t q[2][kTileBytes];
  uint8_t k[kStages][kTileBytes];
  uint8_t v[kStages][kTileBytes];
  float xmax[2][2][kRows];
  float stats[2][3][kRows];
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kStages], k_empty[kStages];
  uint64_t v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_rdy[2][2], pv_done[2], xchg[2][4];
  uint64_t o_full[2], o_free[2], stats_rdy[2];
  Seg segs[kRing];
  uint64_t seg_full[kRing], seg_empty[kRing];
  uint64_t tail[2];  // copies of a tile (of K, of V) whose rest is filled with zeros
  uint64_t drain, unsignalled;
  int warp_sum[kThreads / 32];
  VTiles found;      // where the CTA's piece of the line starts
  int found_v, found_h, found_tile;
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* map, uint32_t bar, int x,
                                            int y, int z, int w, int u) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z),
      "r"(w), "r"(u), "r"(bar)
      : "memory");
}
// ---------------------------------------------------------------- waits
__device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, Smem& sh, const Params& p) {
  const uint64_t t0 = ptx::globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0) {
      if (*reinterpret_cast<volatile int*>(&sh.abort_flag) != 0) return false;
      if (ptx::globaltimer_ns() - t0 > p.timeout_ns) {
        *reinterpret_cast<volatile int*>(&sh.abort_flag) = 1;
        raise(p.c.err, BSATTN_E_TIMEOUT);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, Smem& sh, const Params& p) {
  if (ptx::mbar_test_wait(bar, parity)) return true;
  return wait_slow(bar, parity, sh, p);
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, Smem& sh, const Params& p) {
  return __all_sync(0xffffffffu, wait_one(bar, parity, sh, p));
}
__device__ __forceinline__ void wait_drain(uint32_t bar, uint32_t parity, const Params& p) {
  const uint64_t bound = p.timeout_ns > kDrainNs ? p.timeout_ns : kDrainNs;
  const uint64_t t0 = ptx::globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (ptx::mbar_try_wait(bar, parity)) return;
    if ((it & 63u) == 0 && ptx::globaltimer_ns() - t0 > bound) {
      raise(p.c.err, BSATTN_E_TIMEOUT);
      return;
    }
  }
}

// ---------------------------------------------------------------- items
__device__ __forceinline__ VTiles vtiles(const Params& p, int v) {
  VTiles x;
  if (p.prefix_len > 0) {
    x.b0 = v * p.rt.n_b;
    x.t0 = 0;
    x.len = p.prefix_len;
    x.r = Rows{0, 0};
    x.n_glob = x.lo_block = 0;
    x.n = (p.prefix_len + kTileKeys - 1) / kTileKeys;
    return x;
  }
  x.b0 = v / p.rt.per_seq;
  x.t0 = (v - x.b0 * p.rt.per_seq) * p.rt.n_t;
  const SeqLen s = seq_len(p.c, x.b0);
  x.len = s.len;
  x.r.rows = s.rows;
  x.r.first = s.len - s.rows;
  x.n_glob = 0;
  x.lo_block = 0;
  const int last = x.r.first + min(x.t0 + p.rt.n_t, s.rows) - 1;  // position of the last live row
  int n = 0;
  if (x.t0 < s.rows && last >= 0) {
    if (p.rule.window > 0) {
      x.lo_block = max(0, max(x.r.first + x.t0, 0) / kTileKeys - p.rule.window + 1);
      x.n_glob = min(p.rule.glob, x.lo_block);
    }
    n = x.n_glob + last / kTileKeys - x.lo_block + 1;
  } else {
    x.len = 0;  // no live row: one tile of zeros
  }
  x.n = max(n, 1);
  return x;
}
__device__ __forceinline__ int seg_key(const Seg& s, int j) {
  const int tile = s.tile0 + j;
  return (tile < s.n_glob ? tile : s.lo_block + tile - s.n_glob) * kTileKeys;
}

__device__ __forceinline__ bool ring_write(Smem& sh, const Params& p, int k, const Seg& s, bool lead) {
  const int slot = k & (kRing - 1);
  if (k >= kRing && !wait_warp(ptx::smem_u32(&sh.seg_empty[slot]),
                               static_cast<uint32_t>(k / kRing + 1) & 1u, sh, p))
    return false;
  if (lead) {
    sh.segs[slot] = s;
    ptx::mbar_arrive(ptx::smem_u32(&sh.seg_full[slot]));
  }
  __syncwarp();
  return true;
}
// One reader thread; n == 0 marks the end (also returned after an abort).
__device__ __forceinline__ bool ring_read(Smem& sh, const Params& p, int k, Seg& s) {
  const int slot = k & (kRing - 1);
  if (!wait_one(ptx::smem_u32(&sh.seg_full[slot]), static_cast<uint32_t>(k / kRing) & 1u, sh, p))
    return false;
  s = sh.segs[slot];
  ptx::mbar_arrive(ptx::smem_u32(&sh.seg_empty[slot]));
  return true;
}

// Tile t of the CTA: step j of its ii-th segment.
struct Walk {
  Seg s;
  int ii, j, t;
  bool valid;
};
__device__ __forceinline__ void walk_begin(Walk& x, Smem& sh, const Params& p) {
  x.ii = x.j = x.t = 0;
  x.valid = ring_read(sh, p, 0, x.s) && x.s.n > 0;
}
__device__ __forceinline__ void walk_next(Walk& x, Smem& sh, const Params& p) {
  ++x.t;
  if (x.j + 1 < x.s.n) {
    ++x.j;
    return;
  }
  x.j = 0;
  ++x.ii;
  x.valid = ring_read(sh, p, x.ii, x.s) && x.s.n > 0;
}

// ------------------------------------------------------------------------------------------
// Producers: a whole warp for K (and Q, and the segments), one for V.
// ------------------------------------------------------------------------------------------
struct Stream {
  int is_v, stage;
  uint32_t phase, issued, last_parity;  // bit per stage: a copy was issued, its phase
  uint32_t tail_phase, tail_busy;
  uint64_t *full, *empty;
  uint8_t* tiles;
  uint32_t lane_at;  // where this lane's box lies in a tile
};
__device__ __forceinline__ uint32_t lane_box_at(const Params& p) {
  return (threadIdx.x & 1) * kHalfBytes + ((threadIdx.x & 31) >> 1) * p.box_rows * 128;
}

// Page of this lane's box (lane / 2) of the tile at key0, or -1: past the end, or no such box.
__device__ __forceinline__ int box_page(const Params& p, const Seg& s, int j) {
  const int box = (threadIdx.x & 31) >> 1;
  const int key = seg_key(s, j) + box * p.box_rows;
  if (box >= p.boxes || key >= s.load_end) return -1;
  const int b = p.prefix_len > 0 ? 0 : s.b0;
  return __ldg(p.c.table + b * p.c.table_stride + (key >> p.c.page_shift));
}

// A tile with rows that must be zero: of V behind the sequence's end, of both where there is no page.
__device__ __forceinline__ bool load_ragged(Smem& sh, const Params& p, Stream& x, const CUtensorMap* map, int key0,
                                         int have, int h, int page, uint32_t dst) {
  const int lane = threadIdx.x & 31, box = lane >> 1, half = lane & 1;
  const bool lead = lane == 0;
  const uint32_t full = ptx::smem_u32(x.full + x.stage);
  const uint32_t tail = ptx::smem_u32(&sh.tail[x.is_v]);
  const bool mine = box < p.boxes && box * p.box_rows < have;
  if (mine) page = page_checked(p.c, page);
  const bool get = mine && page >= 0;
  const uint32_t got = __ballot_sync(0xffffffffu, get);
  const bool hole = __any_sync(0xffffffffu, mine && !get);
  const uint32_t bytes = __popc(got) * p.box_rows * 128;
  const bool fill = hole || (x.is_v && have < kTileKeys);
  const uint32_t bar = fill ? tail : full;
  if (lead && bytes > 0) ptx::mbar_expect_tx(bar, bytes);
  if (lead && bytes == 0 && !fill) ptx::mbar_arrive(bar);
  __syncwarp();
  if (get)
    tma_load_5d(dst + half * kHalfBytes + box * p.box_rows * 128, map, bar, 0, key0 & (p.page_size - 1), h, page,
                half);
  if (!fill) return true;
  if (bytes > 0) {
    x.tail_busy = 1;
    if (!wait_warp(tail, x.tail_phase, sh, p)) return false;
    x.tail_phase ^= 1u;
    x.tail_busy = 0;
  }
  // Lane l writes piece l % 8 of half (l / 8) % 2, rows l / 16, + 2, ...
  const uint32_t at = dst + ((lane >> 3) & 1) * kHalfBytes + (lane & 7) * 16;
  if (hole) {
    for (int row = lane >> 4; row < min(have, kTileKeys); row += 2)
      if (!((got >> ((row >> p.box_shift) * 2)) & 1u)) ptx::sts128(at + row * 128, 0, 0, 0, 0);
  }
#pragma unroll 4
  for (int row = max(have, 0) + (lane >> 4); row < kTileKeys; row += 2)
    ptx::sts128(at + row * 128, 0, 0, 0, 0);
  ptx::fence_async_smem();
  __syncwarp();
  if (lead) ptx::mbar_arrive(full);
  return true;
}

__device__ __forceinline__ bool load_tile(Smem& sh, const Params& p, Stream& x, const CUtensorMap* map,
                                          const Seg& s, int j, int page) {
  const int lane = threadIdx.x & 31;
  const int key0 = seg_key(s, j), have = s.load_end - key0;  // rows that hold a token
  const bool mine = (lane >> 1) < p.boxes;
  const bool whole = __all_sync(0xffffffffu, have >= kTileKeys && (!mine || static_cast<unsigned>(page) <
                                                                           static_cast<unsigned>(p.c.n_pages)));
  if (!wait_warp(ptx::smem_u32(x.empty + x.stage), x.phase ^ 1u, sh, p)) return false;
  const uint32_t dst = ptx::smem_u32(x.tiles) + x.stage * kTileBytes;
  if (whole) {
    const uint32_t full = ptx::smem_u32(x.full + x.stage);
    if (lane == 0) ptx::mbar_expect_tx(full, kTileBytes);
    __syncwarp();
    if (mine) tma_load_5d(dst + x.lane_at, map, full, 0, key0 & (p.page_size - 1), s.h, page, lane & 1);
  } else if (!load_ragged(sh, p, x, map, key0, have, s.h, page, dst)) {
    return false;
  }
  x.issued |= 1u << x.stage;
  x.last_parity = (x.last_parity & ~(1u << x.stage)) | (x.phase << x.stage);
  if (++x.stage == kStages) x.stage = 0, x.phase ^= 1u;
  return true;
}

// No copy may still be landing in shared memory when the CTA exits.
__device__ __forceinline__ void drain_stream(Smem& sh, const Params& p, const Stream& x) {
  if ((threadIdx.x & 31) == 0) {
    for (int i = 0; i < kStages; ++i)
      if ((x.issued >> i) & 1u) wait_drain(ptx::smem_u32(x.full + i), (x.last_parity >> i) & 1u, p);
    if (x.tail_busy) wait_drain(ptx::smem_u32(&sh.tail[x.is_v]), x.tail_phase, p);
  }
  __syncwarp();
}

__device__ void producer_k_role(Smem& sh, const CUtensorMap* tq, const CUtensorMap* tk, const Params& p,
                                int begin, int end, int quota) {
  const bool lead = (threadIdx.x & 31) == 0;
  int q_loads = 0;
  Stream x{0, 0, 0, 0, 0, 0, 0, sh.k_full, sh.k_empty, sh.k[0], lane_box_at(p)};
  int v = sh.found_v, h = sh.found_h, tl = sh.found_tile;
  VTiles vt = sh.found;
  int left = end - begin;
  Seg s, next;
  // The next segment of the line (n == 0: none).
  auto step = [&](Seg& o) {
    o.n = 0;
    if (left == 0) return;
    o.v = v;
    o.h = h;
    o.tile0 = tl;
    o.n = min(vt.n - tl, left);
    o.b0 = vt.b0;
    o.t0 = vt.t0;
    o.first = vt.r.first;
    o.rows = vt.r.rows;
    o.load_end = vt.len;
    o.n_glob = vt.n_glob;
    o.lo_block = vt.lo_block;
    o.whole = tl == 0 && o.n == vt.n;
    if (lead && p.prefix_len == 0 && tl == 0 && o.n < vt.n)
      p.cuts[blockIdx.x] = TileCut{v, h, 1 + (vt.n - o.n + quota - 1) / quota, 0};
    left -= o.n;
    tl += o.n;
    if (tl < vt.n) return;
    tl = 0;
    if (++h < p.c.Hkv) return;
    h = 0;
    if (++v < p.rt.count) vt = vtiles(p, v);
  };
  step(s);
  bool ok = ring_write(sh, p, 0, s, lead);
  int page = box_page(p, s, 0);
  for (int k = 0; ok && s.n > 0; ++k) {
    for (int j = 0; ok && j < s.n; ++j) {
      const int now = page;
      const bool last = j + 1 == s.n;
      if (last) {
        step(next);
        if (next.n > 0) page = box_page(p, next, 0);
      } else {
        page = box_page(p, s, j + 1);
      }
      if (j == 0) {
        const int qb = k & 1;
        ok = wait_warp(ptx::smem_u32(&sh.q_empty[qb]), ((static_cast<uint32_t>(k) >> 1) & 1u) ^ 1u, sh, p);
        if (ok && lead) {
          const uint32_t full = ptx::smem_u32(&sh.q_full[qb]);
          ptx::mbar_expect_tx(full, 2 * p.rt.n_t * p.rt.G * p.rt.n_b * 128);
          for (int z = 0; z < 2; ++z)
            tma_load_5d(ptx::smem_u32(sh.q[qb]) + z * kHalfBytes, tq, full, 0, s.t0, s.h * p.rt.G, s.b0, z);
        }
        if (ok) ++q_loads;
      }
      if (ok) ok = load_tile(sh, p, x, tk, s, j, now);
      if (ok && last) ok = ring_write(sh, p, k + 1, next, lead);
    }
    s = next;
  }
  drain_stream(sh, p, x);
  if (lead)
    for (int i = max(q_loads - 2, 0); i < q_loads; ++i)
      wait_drain(ptx::smem_u32(&sh.q_full[i & 1]), (static_cast<uint32_t>(i) >> 1) & 1u, p);
  __syncwarp();
}

__device__ void producer_v_role(Smem& sh, const CUtensorMap* tv, const Params& p) {
  const bool lead = (threadIdx.x & 31) == 0;
  Stream x{1, 0, 0, 0, 0, 0, 0, sh.v_full, sh.v_empty, sh.v[0], lane_box_at(p)};
  bool ok = true;
  for (int k = 0; ok; ++k) {
    const int slot = k & (kRing - 1);
    if (!wait_warp(ptx::smem_u32(&sh.seg_full[slot]), static_cast<uint32_t>(k / kRing) & 1u, sh, p)) break;
    const Seg s = sh.segs[slot];
    __syncwarp();
    if (lead) ptx::mbar_arrive(ptx::smem_u32(&sh.seg_empty[slot]));
    if (s.n == 0) break;
    int page = box_page(p, s, 0);
    for (int j = 0; ok && j < s.n; ++j) {
      const int now = page;
      if (j + 1 < s.n) page = box_page(p, s, j + 1);
      ok = load_tile(sh, p, x, tv, s, j, now);
    }
  }
  drain_stream(sh, p, x);
}

// ------------------------------------------------------------------------------------------
// MMA issuers (lane 0 of their warps).  Tile t uses stage t % 2 of K and of V, and S buffer t % 2.
// ------------------------------------------------------------------------------------------
template <bool BF16>
__device__ void mma_s_role(Smem& sh, const Params& p, uint32_t tmem) {
  constexpr uint32_t idesc = ptx::idesc_f16_f32(128, 128, false, BF16);
  const uint64_t q_desc0 = ptx::sdesc_sw128(ptx::smem_u32(sh.q[0]), 16, 1024);
  const uint64_t k_desc0 = ptx::sdesc_sw128(ptx::smem_u32(sh.k[0]), 16, 1024);
  if (p.test_wait && !wait_one(ptx::smem_u32(&sh.unsignalled), 0, sh, p)) return;
  Walk x;
  walk_begin(x, sh, p);
  while (x.valid) {
    const int qb = x.ii & 1, sb = x.t & 1;
    const uint32_t tph = (static_cast<uint32_t>(x.t) >> 1) & 1u;
    if (x.j == 0 &&
        !wait_one(ptx::smem_u32(&sh.q_full[qb]), (static_cast<uint32_t>(x.ii) >> 1) & 1u, sh, p))
      return;
    if (!wait_one(ptx::smem_u32(&sh.k_full[sb]), tph, sh, p)) return;
    if (x.t >= 2 &&  // P V(t-2) has read the P stored in S[sb]
        !wait_one(ptx::smem_u32(&sh.pv_done[sb]), tph ^ 1u, sh, p))
      return;
    ptx::tc_fence_after();
    const uint64_t qd = q_desc0 + static_cast<uint32_t>((qb * kTileBytes) >> 4);
    const uint64_t kd = k_desc0 + static_cast<uint32_t>((sb * kTileBytes) >> 4);
#pragma unroll
    for (int kk = 0; kk < kHeadDim / 16; ++kk) {
      const uint32_t off = ((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4;
      ptx::mma_ss(tmem + sb * 128, qd + off, kd + off, idesc, kk > 0 ? 1u : 0u);
    }
    ptx::tc_commit(ptx::smem_u32(&sh.k_empty[sb]));
    ptx::tc_commit(ptx::smem_u32(&sh.s_full[sb]));
    if (x.j == x.s.n - 1) ptx::tc_commit(ptx::smem_u32(&sh.q_empty[qb]));
    walk_next(x, sh, p);
  }
}

template <bool BF16>
__device__ void mma_pv_role(Smem& sh, const Params& p, uint32_t tmem) {
  constexpr uint32_t idesc = ptx::idesc_f16_f32(128, 128, true, BF16);
  const uint64_t v_desc0 = ptx::sdesc_sw128(ptx::smem_u32(sh.v[0]), kHalfBytes, 1024);
  Walk x;
  walk_begin(x, sh, p);
  while (x.valid) {
    const int ob = x.ii & 1, sb = x.t & 1;
    const uint32_t tph = (static_cast<uint32_t>(x.t) >> 1) & 1u;
    if (!wait_one(ptx::smem_u32(&sh.v_full[sb]), tph, sh, p)) return;
    if (x.j == 0 && x.ii >= 2 &&  // O[ob] read out by the epilogue of segment ii - 2
        !wait_one(ptx::smem_u32(&sh.o_free[ob]), ((static_cast<uint32_t>(x.ii) >> 1) + 1u) & 1u, sh, p))
      return;
    if (!wait_one(ptx::smem_u32(&sh.p_rdy[sb][0]), tph, sh, p)) return;
    if (!wait_one(ptx::smem_u32(&sh.p_rdy[sb][1]), tph, sh, p)) return;
    ptx::tc_fence_after();
    const uint64_t vd = v_desc0 + static_cast<uint32_t>((sb * kTileBytes) >> 4);
#pragma unroll
    for (int kk = 0; kk < kTileKeys / 16; ++kk)
      ptx::mma_ts(tmem + kOCol + ob * 128, tmem + sb * 128 + (kk >> 2) * 64 + (kk & 3) * 8,
                  vd + static_cast<uint32_t>((kk * 2048) >> 4), idesc, (x.j > 0 || kk > 0) ? 1u : 0u);
    ptx::tc_commit(ptx::smem_u32(&sh.v_empty[sb]));
    ptx::tc_commit(ptx::smem_u32(&sh.pv_done[sb]));
    if (x.j == x.s.n - 1) ptx::tc_commit(ptx::smem_u32(&sh.o_full[ob]));
    walk_next(x, sh, p);
  }
}

// Row t of a tile: its sequence, query head and token, and the keys it sees.
struct Row {
  int b, g, t;
  RowKeys k;  // limit == 0: dead (or padding of the tile)
};
__device__ __forceinline__ Row row_of(const Params& p, const Seg& s, int t) {
  Row r;
  const int nt = p.rt.n_t, g_all = t / nt;
  const int bb = g_all / p.rt.G;
  r.g = g_all - bb * p.rt.G;
  r.t = s.t0 + t - g_all * nt;
  r.b = s.b0 + bb;
  r.k = RowKeys{0, 0};
  if (bb >= p.rt.n_b || r.b >= p.c.B || r.t >= p.c.Tq) {
    r.b = -1;
    return r;
  }
  Rows rows{s.rows, s.first};
  if (p.prefix_len > 0) {
    const SeqLen q = seq_len(p.c, r.b);
    rows = Rows{q.rows, q.len - q.rows};
  }
  r.k = row_keys(rows, p.rule, r.t);
  if (p.prefix_len > 0) r.k.limit = min(r.k.limit, p.prefix_len);
  return r;
}

// ------------------------------------------------------------------------------------------
// Softmax warpgroup `half`: keys 64 half .. 64 half + 63 of every tile, thread t owns row t.
// ------------------------------------------------------------------------------------------
template <bool BF16>
__device__ void softmax_role(Smem& sh, const Params& p, int half, uint32_t tmem) {
  const int t = threadIdx.x - kSoftmaxWarp0 * 32 - half * 128;
  const int wq = t >> 5;
  const uint32_t lane_addr = tmem + (static_cast<uint32_t>(wq * 32) << 16);
  const float sl2 = p.scale_log2;
  // The power of two that is not below the scale.
  const float far_scale = __uint_as_float((__float_as_uint(sl2) + 0x7fffffu) & 0x7f800000u);
  const int glob_end = p.rule.glob * kTileKeys;
  int tile = 0;
  for (int ii = 0;; ++ii) {
    const int slot = ii & (kRing - 1);
    if (!wait_warp(ptx::smem_u32(&sh.seg_full[slot]), static_cast<uint32_t>(ii / kRing) & 1u, sh, p))
      return;
    const Seg sg = sh.segs[slot];
    ptx::mbar_arrive(ptx::smem_u32(&sh.seg_empty[slot]));
    if (sg.n == 0) break;
    const int ob = ii & 1;
    const RowKeys rk = row_of(p, sg, t).k;
    // Nobody reads what becomes of a warp's rows if none of them is live.
    const bool dead = __all_sync(0xffffffffu, rk.limit <= 0);
    float m_run = kNoMax, l_run = 0.0f;
    for (int j = 0; j < sg.n; ++j, ++tile) {
      const int sb = tile & 1;
      const uint32_t s_addr = lane_addr + sb * 128 + half * 64;
      if (!wait_warp(ptx::smem_u32(&sh.s_full[sb]), (static_cast<uint32_t>(tile) >> 1) & 1u, sh, p))
        return;
      if (dead) {
        ptx::mbar_arrive(ptx::smem_u32(&sh.xchg[sb][wq]));
        ptx::mbar_arrive(ptx::smem_u32(&sh.p_rdy[sb][half]));
        continue;
      }
      ptx::tc_fence_after();
      uint32_t sr[64];
      ptx::tmem_ld32(s_addr + 0, sr + 0);
      ptx::tmem_ld32(s_addr + 32, sr + 32);
      ptx::tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 64; ++c) ptx::reg_fence(sr[c]);
      float s[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) s[c] = __uint_as_float(sr[c]);
      // A window holds whole tiles (lo and glob_end are multiples of 128); the limit may cut one.
      const int key0 = seg_key(sg, j);
      const int n_keep = (key0 < rk.lo && key0 >= glob_end)
                             ? 0 : min(max(rk.limit - key0 - 64 * half, 0), 64);
      if (n_keep < 64) {
#pragma unroll
        for (int c = 0; c < 64; ++c) s[c] = (c < n_keep) ? s[c] : -INFINITY;
      }
      float a0 = s[0], a1 = s[1], a2 = s[2], a3 = s[3];
#pragma unroll
      for (int c = 4; c < 60; c += 8) {
        a0 = ptx::fmax3(a0, s[c + 0], s[c + 1]);
        a1 = ptx::fmax3(a1, s[c + 2], s[c + 3]);
        a2 = ptx::fmax3(a2, s[c + 4], s[c + 5]);
        a3 = ptx::fmax3(a3, s[c + 6], s[c + 7]);
      }
      a0 = ptx::fmax3(a0, s[60], s[61]);
      a1 = ptx::fmax3(a1, s[62], s[63]);
      const float pmax = ptx::fmax3(a0, a1, fmaxf(a2, a3));
      sh.xmax[sb][half][t] = pmax;
      ptx::mbar_arrive(ptx::smem_u32(&sh.xchg[sb][wq]));
      if (!wait_warp(ptx::smem_u32(&sh.xchg[sb][wq]), (static_cast<uint32_t>(tile) >> 1) & 1u, sh, p))
        return;
      const float top = fmaxf(pmax, sh.xmax[sb][half ^ 1][t]);
      float m_cand = top * sl2;
      if (fabsf(m_cand) > kFar) m_cand = top * far_scale;
      float alpha = 1.0f;
      bool rescale = false;
      if (j == 0) {
        m_run = fmaxf(m_run, m_cand);
      } else {
        rescale = __any_sync(0xffffffffu, m_cand > m_run + kRescaleLog2);
        if (rescale) {
          const float m_new = fmaxf(m_run, m_cand);
          alpha = ptx::ex2(m_run - m_new);
          l_run *= alpha;
          m_run = m_new;
        }
      }
      const float sc = fabsf(m_run) > kFar ? far_scale : sl2;
      const uint64_t sc2 = ptx::pack2(sc, sc);
      const uint64_t nm2 = ptx::pack2(-m_run, -m_run);
      uint64_t acc0 = 0, acc1 = 0;
      uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint64_t x2 = ptx::ffma2(ptx::pack2(s[2 * i], s[2 * i + 1]), sc2, nm2);
        float x0, x1, p0, p1;
        ptx::unpack2(x2, x0, x1);
        if ((i % kPolyEvery) == kPolyEvery - 1) {
          ptx::exp2_poly_pair(x0, x1, p0, p1);
        } else {
          p0 = ptx::ex2(x0);
          p1 = ptx::ex2(x1);
        }
        const uint64_t p2 = ptx::pack2(p0, p1);
        if (i & 1) acc1 = ptx::fadd2(acc1, p2); else acc0 = ptx::fadd2(acc0, p2);
        pk[i] = pack16<BF16>(p0, p1);
      }
      ptx::tmem_st32(s_addr, pk);
      if (rescale) {
        // O holds PV up to tile - 1 once pv_done says so; PV(tile + 1) needs this tile's P first.
        const uint32_t pb = static_cast<uint32_t>(tile - 1) & 1u;
        if (!wait_warp(ptx::smem_u32(&sh.pv_done[pb]), (static_cast<uint32_t>(tile - 1) >> 1) & 1u, sh, p))
          return;
        ptx::tc_fence_after();
        const uint32_t o_addr = lane_addr + kOCol + ob * 128 + half * 64;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t orow[32];
          ptx::tmem_ld32(o_addr + c * 32, orow);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            ptx::reg_fence(orow[i]);
            orow[i] = __float_as_uint(__uint_as_float(orow[i]) * alpha);
          }
          ptx::tmem_st32(o_addr + c * 32, orow);
        }
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      ptx::mbar_arrive(ptx::smem_u32(&sh.p_rdy[sb][half]));
      float l0, l1;
      ptx::unpack2(ptx::fadd2(acc0, acc1), l0, l1);
      l_run += l0 + l1;
    }
    if (ii >= 2) {  // stats[ob] read by the epilogue of segment ii - 2
      if (!wait_warp(ptx::smem_u32(&sh.o_free[ob]), ((static_cast<uint32_t>(ii) >> 1) + 1u) & 1u, sh, p))
        return;
    }
    if (half == 0)  // back in the scale's unit
      sh.stats[ob][0][t] = fabsf(m_run) > kFar && m_run > kNoMaxBelow ? m_run * (sl2 / far_scale) : m_run;
    sh.stats[ob][1 + half][t] = l_run;
    ptx::mbar_arrive(ptx::smem_u32(&sh.stats_rdy[ob]));
  }
}

// ------------------------------------------------------------------------------------------
// Epilogue warpgroup
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ bool epi_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\tbar.red.or.pred b, 1, 128, a;"
      "\n\tselp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(r) : "r"(v ? 1u : 0u) : "memory");
  return r != 0;
}

__device__ void epilogue_role(Smem& sh, const Params& p, uint32_t tmem) {
  const int t = threadIdx.x - kEpiWarp0 * 32;
  const int wq = t >> 5;
  const uint32_t lane_addr = tmem + (static_cast<uint32_t>(wq * 32) << 16);
  for (int ii = 0;; ++ii) {
    const int slot = ii & (kRing - 1);
    const int ob = ii & 1;
    const uint32_t ph = (static_cast<uint32_t>(ii) >> 1) & 1u;
    bool ok = wait_warp(ptx::smem_u32(&sh.seg_full[slot]), static_cast<uint32_t>(ii / kRing) & 1u, sh, p);
    if (epi_any(!ok)) return;
    const Seg sg = sh.segs[slot];
    ptx::mbar_arrive(ptx::smem_u32(&sh.seg_empty[slot]));
    if (sg.n == 0) return;
    ok = wait_warp(ptx::smem_u32(&sh.o_full[ob]), ph, sh, p);
    if (ok) ok = wait_warp(ptx::smem_u32(&sh.stats_rdy[ob]), ph, sh, p);
    if (epi_any(!ok)) return;
    ptx::tc_fence_after();
    const Row row = row_of(p, sg, t);
    const float m_run = sh.stats[ob][0][t];
    const float l_run = sh.stats[ob][1][t] + sh.stats[ob][2][t];
    const bool live = row.k.limit > 0 && m_run > kNoMaxBelow && l_run > 0.0f;
    const float inv_l = live ? 1.0f / l_run : 0.0f;
    const float lg = live ? m_run + log2f(l_run) : -INFINITY;
    const uint32_t o_addr = lane_addr + kOCol + ob * 128;
    if (p.prefix_len == 0 && sg.whole) {
      const long long gr =
          row.b < 0 ? 0
                    : (static_cast<long long>(row.b) * p.Hq + sg.h * p.rt.G + row.g) * p.c.Tq + row.t;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t orow[32];
        ptx::tmem_ld32(o_addr + c * 32, orow);
        ptx::tmem_wait_ld();
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          ptx::reg_fence(orow[2 * i]);
          ptx::reg_fence(orow[2 * i + 1]);
          w[i] = pack_out(live ? __uint_as_float(orow[2 * i]) * inv_l : 0.0f,
                          live ? __uint_as_float(orow[2 * i + 1]) * inv_l : 0.0f, p.out_bf16);
        }
        if (row.b >= 0) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + gr * kHeadDim + c * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
      }
      if (p.lse != nullptr && row.b >= 0) p.lse[gr] = lg * 0.69314718055994531f;
    } else {
      // Partial slots: (item, CTA) pairs for a prefix; else this CTA's head piece or its other one.
      const int slot_o = p.prefix_len > 0
                             ? sg.v * p.c.Hkv + sg.h + static_cast<int>(blockIdx.x)
                             : 2 * static_cast<int>(blockIdx.x) + (sg.tile0 == 0 ? 1 : 0);
      float4* const dst = reinterpret_cast<float4*>(p.part_o) +
                          static_cast<long long>(slot_o) * (kRows * kHeadDim / 4) + t;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t orow[32];
        ptx::tmem_ld32(o_addr + c * 32, orow);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          ptx::reg_fence(orow[i]);
          orow[i] = live ? __float_as_uint(__uint_as_float(orow[i]) * inv_l) : 0u;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          dst[(c * 8 + k) * kRows] =
              make_float4(__uint_as_float(orow[4 * k]), __uint_as_float(orow[4 * k + 1]),
                          __uint_as_float(orow[4 * k + 2]), __uint_as_float(orow[4 * k + 3]));
      }
      p.part_l[static_cast<long long>(slot_o) * kRows + t] = lg;
    }
    ptx::tc_fence_before();
    ptx::mbar_arrive(ptx::smem_u32(&sh.o_free[ob]));
  }
}

struct Launch {
  CUtensorMap q, k, v;
  Params p;
};

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ Launch l) {
  const CUtensorMap &tq = l.q, &tk = l.k, &tv = l.v;
  const Params& p = l.p;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  Smem& sh = *reinterpret_cast<Smem*>(smem_raw + (((raw + 1023u) & ~1023u) - raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 2) {
    // Side by side on the lanes of a warp: one thread would take a microsecond.
    auto init = [&](uint64_t& bar, uint32_t n) { ptx::mbar_init(ptx::smem_u32(&bar), n); };
    if (lane < 2) {
      init(sh.s_full[lane], 1);
      init(sh.pv_done[lane], 1);
      init(sh.o_full[lane], 1);
      init(sh.o_free[lane], 128);
      init(sh.stats_rdy[lane], 256);
      init(sh.tail[lane], 1);
      init(sh.q_full[lane], 1);
      init(sh.q_empty[lane], 1);
    } else if (lane < 6) {
      init(sh.p_rdy[(lane - 2) >> 1][lane & 1], 128);
      init(sh.xchg[0][lane - 2], 64);
      init(sh.xchg[1][lane - 2], 64);
    } else if (lane < 6 + kStages) {
      init(sh.k_full[lane - 6], 1);
      init(sh.k_empty[lane - 6], 1);
      init(sh.v_full[lane - 6], 1);
      init(sh.v_empty[lane - 6], 1);
    } else if (lane >= 16 && lane < 16 + kRing) {
      init(sh.seg_full[lane - 16], 1);
      init(sh.seg_empty[lane - 16], kRingReaders);
    } else if (lane == 31) {
      init(sh.drain, 2);
      init(sh.unsignalled, 1);
      sh.abort_flag = 0;
    }
    ptx::fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    ptx::tma_prefetch_desc(&tq);
    ptx::tma_prefetch_desc(&tk);
    ptx::tma_prefetch_desc(&tv);
  }

  const int cta = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
  pdl_wait();
  pdl_trigger();
  // Tensor memory only now: a predecessor that still has to allocate its own on this SM must not find
  // it taken by a kernel that waits for it.
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&sh.tmem_base), kTmemCols);
    ptx::tmem_relinquish();
  }
  // This CTA's piece of the line (as in the few-row kernel).
  const int chunk = (p.rt.count + kThreads - 1) / kThreads;
  const int v0 = min(static_cast<int>(threadIdx.x) * chunk, p.rt.count);
  const int v1 = min(v0 + chunk, p.rt.count);
  int mine = 0;
  VTiles vt;  // of v0, the only one in most calls
  for (int v = v0; v < v1; ++v) {
    const VTiles y = vtiles(p, v);
    if (v == v0) vt = y;
    mine += y.n;
  }
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) sh.warp_sum[warp] = incl;
  __syncthreads();
  int total = 0, before = incl - mine;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sh.warp_sum[w];
    total += sh.warp_sum[w];
  }
  const int line = total * p.c.Hkv;
  const int quota = (line + ctas - 1) / ctas;
  const int begin = min(cta * quota, line);
  const int end = min(begin + quota, line);
  for (int v = v0; v < v1; ++v) {
    if (v > v0) vt = vtiles(p, v);
    const int n = vt.n;
    const int rel = begin - before * p.c.Hkv;
    if (rel >= 0 && rel < n * p.c.Hkv) {
      sh.found = vt;
      sh.found_v = v;
      sh.found_h = rel / n;
      sh.found_tile = rel % n;
    }
    before += n;
  }
  if (threadIdx.x == 0 && p.prefix_len == 0) p.cuts[cta] = TileCut{-1, 0, 0, 0};
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  if (begin >= end) {  // the whole CTA
    if (warp == 1) ptx::tmem_dealloc(tmem, kTmemCols);
    return;
  }

  if (warp >= kSoftmaxWarp0 && warp < kEpiWarp0) {
    ptx::setmaxnreg_inc<kSoftmaxRegs>();
    softmax_role<BF16>(sh, p, (warp - kSoftmaxWarp0) >> 2, tmem);
  } else if (warp < kSoftmaxWarp0) {
    ptx::setmaxnreg_dec<kControlRegs>();
    if (warp == 0) {
      producer_k_role(sh, &tq, &tk, p, begin, end, quota);
    } else if (warp == 3) {
      producer_v_role(sh, &tv, p);
    } else if (warp == 1) {
      if (lane == 0) mma_pv_role<BF16>(sh, p, tmem);
    } else if (warp == 2) {
      if (lane == 0) mma_s_role<BF16>(sh, p, tmem);
    }
  } else {
    ptx::setmaxnreg_dec<kEpilogueRegs>();
    epilogue_role(sh, p, tmem);
  }
  __syncwarp();
  ptx::tmem_wait_ld();
  ptx::tmem_wait_st();
  ptx::tc_fence_before();
  __syncthreads();
  // Both issuing threads commit once more; then every MMA of the CTA has completed.
  if ((warp == 1 || warp == 2) && lane == 0) ptx::tc_commit(ptx::smem_u32(&sh.drain));
  if (warp == 1) {
    if (lane == 0) wait_drain(ptx::smem_u32(&sh.drain), 0, p);
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeFn>(ptr);
  }();
  return fn;
}

static int encode(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                  const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const EncodeFn fn = encode_fn();
  if (!fn) return BSATTN_E_TMA;
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(map, type, rank, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BSATTN_OK : BSATTN_E_TMA;
}

constexpr size_t kSmemBytes = sizeof(Smem) + 1024;

}  // namespace tile

int tile_setup() {
  const void* kernels[] = {reinterpret_cast<const void*>(tile::tile_kernel<false>),
                           reinterpret_cast<const void*>(tile::tile_kernel<true>)};
  for (const void* k : kernels) {
    // The register split needs exactly the launch registers it assumes: with fewer, setmaxnreg.inc
    // would never return.
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, k) != cudaSuccess) return BSATTN_E_CUDA;
    if (fa.numRegs != static_cast<int>(tile::kLaunchRegs)) return BSATTN_E_CUDA;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(tile::kSmemBytes)) != cudaSuccess)
      return BSATTN_E_CUDA;
  }
  return BSATTN_OK;
}

int tile_launch(const TileCall& call, int page_size, cudaStream_t stream) {
  using namespace tile;
  const Cache& c = call.c;
  const RowTiles& rt = call.rt;
  const CUtensorMapDataType type =
      call.in_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  Params p;
  p.box_rows = std::min(page_size, kTileKeys);
  p.boxes = kTileKeys / p.box_rows;
  p.box_shift = 0;
  while ((1 << p.box_shift) < p.box_rows) ++p.box_shift;
  CUtensorMap tq, tk, tv;
  int rc;
  {
    const cuuint64_t tok = kHeadDim * 2, head = tok * c.Tq, seq = head * call.Hq;
    const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(c.Tq), static_cast<cuuint64_t>(call.Hq),
                                static_cast<cuuint64_t>(c.B), 2};
    const cuuint64_t strides[4] = {tok, head, seq, 128};
    const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(rt.n_t), static_cast<cuuint32_t>(rt.G),
                               static_cast<cuuint32_t>(rt.n_b), 1};
    if ((rc = encode(&tq, type, 5, call.q, dims, strides, box)) != BSATTN_OK) return rc;
  }
  for (int i = 0; i < 2; ++i) {
    // {64 columns, tokens of a page, heads, pages, 2 halves}.  The stride of a dimension of one
    // entry is never used; any legal value will do.
    const long long st[3] = {i ? c.v_tok : c.k_tok, i ? c.v_head : c.k_head, i ? c.v_page : c.k_page};
    const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(page_size), static_cast<cuuint64_t>(c.Hkv),
                                static_cast<cuuint64_t>(c.n_pages), 2};
    cuuint64_t strides[4] = {0, 0, 0, 128};
    for (int d = 0; d < 3; ++d)
      strides[d] = dims[d + 1] > 1 ? static_cast<cuuint64_t>(st[d]) : kHeadDim * 2;
    const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(p.box_rows), 1, 1, 1};
    if ((rc = encode(i ? &tv : &tk, type, 5, i ? c.v : c.k, dims, strides, box)) != BSATTN_OK) return rc;
  }
  p.c = c;
  p.rule = call.rule;
  p.rt = rt;
  p.prefix_len = call.prefix_len;
  p.page_size = page_size;
  p.o = call.o;
  p.lse = call.lse;
  p.Hq = call.Hq;
  p.scale_log2 = call.scale_log2;
  p.out_bf16 = call.out_bf16;
  p.cuts = call.cuts;
  p.part_o = call.part_o;
  p.part_l = call.part_l;
  p.timeout_ns = launch_timeout_ns();
  p.test_wait = launch_test_wait();
  const Launch l{tq, tk, tv, p};
  return launch(call.in_bf16 ? tile_kernel<true> : tile_kernel<false>,
                dim3(static_cast<unsigned>(call.pieces)), kThreads, kSmemBytes, stream, l);
}

}  // namespace paged
}  // namespace bsattn

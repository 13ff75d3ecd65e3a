// paged_attn.cu -- attention of new tokens over a paged K/V cache.
//
// Rows: q [B, Hq, Tq, 128]; the G = Hq / Hkv query heads that share a K/V head form, with their Tq
// tokens, the G * Tq rows (g-major) that one pass over that head's keys serves.  For row (g, t) at
// position p = seq_lens[b] - q_lens[b] + t:
//     o = sum_j softmax_j(scale q . k_j) v_j over the keys j <= p (and the window rule),
//     lse = ln sum_j exp(scale q . k_j);  no key: o = 0, lse = -inf.
//
// Few rows (the decode form).  Every key costs 512 bytes of HBM and G * Tq * 512 operations, so
// the bound is memory; what matters is that all SMs read all the time and that nothing waits for
// anything else.
//   * Work: an item is (sequence, K/V head, tile of rows), a tile is 64 keys.  All items form one
//     line, measured in units of 16 keys (plus a few per item for what its end costs); it is cut
//     into equal pieces, and a CTA takes the tiles that begin in its piece.  So a long sequence is
//     split over many CTAs, a short one shares a CTA with others, and half-empty tiles do not
//     unbalance them.  The lengths are on the device: each CTA adds them up itself, in a few
//     microseconds at most, and no host copy is needed.
//   * A CTA is four warps on their own, and two CTAs share an SM, so that one's item ends are hidden
//     behind the other's work: warp w owns keys 16w .. 16w+15 of every tile, loads them with cp.async
//     into a private ring (16-byte pieces swizzled so that ldmatrix reads without
//     bank conflicts) and keeps its own running maximum, sum and output.  No barrier is met until
//     a piece of an item ends; the ring runs across item borders.
//   * Keys are the M dimension of the warp MMAs (m16n8k16): S^T = K Q^T and O^T = V^T P^T, so eight
//     rows fill an MMA's N and none of it is spent on padding; P^T moves from the accumulator to
//     the operand layout with movmatrix, in registers.
//   * The running maximum moves only when a score passes it by more than 2^8 (then P stays within
//     2^8, far inside fp16 and bf16); the usual step costs one vote instead of a reduction.
//   * At the end of a piece the warps' outputs are merged through shared memory in warp
//     order.  A piece that is a whole item writes o and lse; others leave (o, log2 sum) in 32 bits,
//     and the warp that finds its row's pieces complete adds them, in the order of the line: results
//     do not depend on timing.
// Keys past a sequence's end are loaded as zeros, never read: a recycled page may hold anything.
// P is rounded to the type of V, as the tensor cores take it; its sum is of the unrounded values.
#include <algorithm>
#include <mutex>

#include "paged_common.cuh"
#include "paged_tile.cuh"
#include "sm100_ptx.cuh"

namespace bsattn {
namespace paged {

constexpr int kWarps = 4;
constexpr int kCtasPerSm = 2;
constexpr int kThreadsD = kWarps * 32;
constexpr int kStages = 3;
constexpr int kSlice = 16;                        // keys of a tile per warp
constexpr int kSliceBytes = kSlice * kHeadDim * 2;  // 4 KB of K or of V
constexpr int kOPitch = kHeadDim + 4;             // floats between rows of the merge buffer
constexpr float kRescaleLog2 = 8.0f;
constexpr int kMaxSms = 160;     // SMs a call uses at most (a B200 has 148)
constexpr int kFewRows = 16;     // rows of one tile of the few-row kernel
constexpr int kStep = kWarps * kSlice;  // keys of a tile
static_assert(kTileKeys % kStep == 0, "the window rule counts whole tiles");

struct AttnParams {
  Cache c;
  Rule rule;
  const void* q;
  void* o;
  float* lse;
  int rows, row_tiles;  // rows = G * Tq; row_tiles = ceil(rows / R)
  float scale_log2;
  int out_bf16;
  int all_partial;  // behind a shared prefix: no piece is a whole result
  // Scratch: for the row join the sequences' places on the line [B + 1], its quota and alignment;
  // partial outputs and their log2 sums.
  int* cum;
  float* part_o;
  float* part_l;
  int* counters;  // [pieces, kFewRows], zero between calls: written pieces of a split item, by warp
};

template <int NB>
struct DecodeSmem {
  uint8_t ring[kWarps][kStages][2][kSliceBytes];
  float o[kWarps][8][kOPitch];
  float m[kWarps][8], l[kWarps][8];
  uint64_t o_free;  // all warps have read `o`
  unsigned long long warp_sum[kWarps];
  int found[4];
};

// Where a piece of item `item` that CTA `cta` holds leaves its partial output.  A CTA holds at most
// one piece that begins its item and one other; when whole items are partial too, item + cta
// numbers all pieces, since along the line one of the two always grows.
__device__ __forceinline__ long long part_slot(int all_partial, long long item, int cta, bool head) {
  return all_partial ? item + cta : 2ll * cta + (head ? 1 : 0);
}

// The key tiles of one sequence, those any live row sees, in ascending order: n_glob leading ones,
// then those from key `lo` on.  A sequence without a key still gets one tile, so that every row is
// written by the same path.
struct Tiles {
  int len;
  Rows r;
  int n, n_glob, lo;
  int last;  // keys of the last tile
};
__device__ __forceinline__ int tile_key(const Tiles& t, int tile) {
  return tile < t.n_glob ? tile * kStep : t.lo + (tile - t.n_glob) * kStep;
}
__device__ __forceinline__ Tiles tiles_of(const Cache& c, const Rule& r, int b) {
  const SeqLen s = seq_len(c, b);
  Tiles t;
  t.len = s.len;
  t.r = Rows{s.rows, s.len - s.rows};
  t.lo = r.k0;
  t.n_glob = 0;
  t.n = 1;
  t.last = 0;
  if (s.rows > 0 && s.len > r.k0) {
    if (r.window > 0) {
      const int block = max(0, max(t.r.first, 0) / kTileKeys - r.window + 1);
      t.lo = block * kTileKeys;
      t.n_glob = min(r.glob, block) * (kTileKeys / kStep);
    }
    const int n = (s.len - t.lo + kStep - 1) / kStep;
    t.last = s.len - t.lo - (n - 1) * kStep;
    t.n = t.n_glob + n;
  }
  return t;
}

// The line.  Tile k of an item begins kTileUnits k units behind it.  Small calls are cut item by item
// (align > 0: items are rounded up to pieces of `align` units, so no CTA has two), larger ones in
// equal pieces wherever that falls.
constexpr int kTileUnits = kStep / kSlice;
constexpr int kItemUnits = 2;
constexpr int kAlign = 16;
__device__ __forceinline__ int units_of(const Tiles& t, int align) {
  const int starts = kTileUnits * (t.n - 1);
  return align > 0 ? (starts / align + 1) * align
                   : starts + max((t.last + kSlice - 1) / kSlice, 1) + kItemUnits;
}
// Pieces of an item of that many units that begins at unit `at`: every CTA from the first one to
// that of the last tile holds a tile, since a piece is no shorter than one.
struct Line {
  int quota, align;
};
__device__ __forceinline__ int last_piece(const Line& x, int at, int units) {
  if (x.align > 0) return (at + units) / x.quota - 1;
  return (at + (units - kItemUnits - 1) / kTileUnits * kTileUnits) / x.quota;
}

// A split item of this CTA: the CTAs it lies in, its first row of q and its rows.
struct Split {
  int first, last, rows;
  long long q_row;
};

// A tile on the line.
struct Cursor {
  int b, h, tile;  // h counts (K/V head, row tile)
  int item, u;     // first unit of the item, and of the tile
  Tiles t;
};

__device__ __forceinline__ void store_row(void* o, float* lse, int out_bf16, long long row, float4 v,
                                          float lg, int lane) {
  reinterpret_cast<uint2*>(o)[row * (kHeadDim / 4) + lane] =
      make_uint2(pack_out(v.x, v.y, out_bf16), pack_out(v.z, v.w, out_bf16));
  if (lse != nullptr && lane == 0) lse[row] = lg * 0.69314718055994531f;
}

// A weighted sum of partial rows, which are read past L1: other SMs may have written them while
// this kernel ran.
struct PartSum {
  float4 acc;
  float sum;
  __device__ __forceinline__ void add(float4 y, float w) {
    acc.x += y.x * w;
    acc.y += y.y * w;
    acc.z += y.z * w;
    acc.w += y.w * w;
    sum += w;
  }
};
__device__ __forceinline__ float4 part_row(const float* po, long long row, int lane) {
  return __ldcg(reinterpret_cast<const float4*>(po) + row * (kHeadDim / 4) + lane);
}

// One warp, kRowsPerWarp rows: o = sum_c o_c 2^(l_c - l), l = log2 sum 2^l_c over the pieces of CTAs
// first .. last, in that order, eight pieces of each row asked for at a time.
constexpr int kRowsPerWarp = 8 / kWarps;
__device__ __noinline__ void join_own(const AttnParams& p, long long row, int r, int live, int R,
                                      int first, int last, int lane) {
  constexpr int kAtOnce = 8;
  const int n = last - first + 1;
  float mx[kRowsPerWarp];
  PartSum s[kRowsPerWarp];
#pragma unroll
  for (int k = 0; k < kRowsPerWarp; ++k) {
    mx[k] = -INFINITY;
    s[k] = PartSum{make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f};
  }
  for (int c0 = 0; c0 < n; c0 += kAtOnce) {
    float4 y[kRowsPerWarp][kAtOnce];
    float lg[kRowsPerWarp][kAtOnce];
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c)
#pragma unroll
      for (int k = 0; k < kRowsPerWarp; ++k) {
        lg[k][c] = -INFINITY;
        y[k][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c0 + c < n && k < live) {
          const long long at = part_slot(0, 0, first + c0 + c, c0 + c == 0) * R + r + k;
          lg[k][c] = __ldcg(p.part_l + at);
          y[k][c] = part_row(p.part_o, at, lane);
        }
      }
#pragma unroll
    for (int k = 0; k < kRowsPerWarp; ++k) {
      float top = mx[k];
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) top = fmaxf(top, lg[k][c]);
      if (top == -INFINITY) continue;
      const float f = ptx::ex2(mx[k] - top);
      mx[k] = top;
      s[k].acc = make_float4(s[k].acc.x * f, s[k].acc.y * f, s[k].acc.z * f, s[k].acc.w * f);
      s[k].sum *= f;
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) s[k].add(y[k][c], ptx::ex2(lg[k][c] - top));
    }
  }
#pragma unroll
  for (int k = 0; k < kRowsPerWarp; ++k) {
    if (k >= live) continue;
    const float inv = s[k].sum > 0.0f ? 1.0f / s[k].sum : 0.0f;
    const float4 a = s[k].acc;
    store_row(p.o, p.lse, p.out_bf16, row + k, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv),
              s[k].sum > 0.0f ? mx[k] + log2f(s[k].sum) : -INFINITY, lane);
  }
}

// The other warps of this CTA are past a __syncthreads and on their way to this arrival: the wait
// ends within the few hundred cycles that they take to read the buffer.
__device__ __forceinline__ void wait_merge(uint32_t bar, uint32_t parity) {
  for (int it = 0; it < (1 << 20) && !ptx::mbar_try_wait(bar, parity); ++it) {
  }
}

template <bool BF16, int NB>
__global__ void __launch_bounds__(kThreadsD, kCtasPerSm) decode_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  DecodeSmem<NB>& sh = *reinterpret_cast<DecodeSmem<NB>*>(smem_raw);
  constexpr int R = 8 * NB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int per_seq = p.c.Hkv * p.row_tiles;
  const uint32_t o_free = ptx::smem_u32(&sh.o_free);
  pdl_trigger();
  if (threadIdx.x == 0) {
    ptx::mbar_init(o_free, kWarps);
    ptx::fence_mbar_init();
    sh.found[0] = -1;
  }

  // Where this CTA's piece of the line starts.
  const int chunk = (p.c.B + kThreadsD - 1) / kThreadsD;
  const int b0 = min(static_cast<int>(threadIdx.x) * chunk, p.c.B);
  const int b1 = min(b0 + chunk, p.c.B);
  unsigned long long mine = 0;  // units, and in the upper half aligned ones
  for (int b = b0; b < b1; ++b) {
    const Tiles t = tiles_of(p.c, p.rule, b);
    mine += static_cast<unsigned>(units_of(t, 0)) +
            (static_cast<unsigned long long>(units_of(t, kAlign)) << 32);
  }
  unsigned long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) sh.warp_sum[warp] = incl;
  __syncthreads();
  unsigned long long total2 = 0, before2 = incl - mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before2 += sh.warp_sum[w];
    total2 += sh.warp_sum[w];
  }
  const int pieces = static_cast<int>(gridDim.x);
  Line ln;
  ln.align = static_cast<long long>(total2 >> 32) * per_seq <= static_cast<long long>(pieces) * kAlign
                 ? kAlign : 0;
  const int total = static_cast<int>(ln.align ? total2 >> 32 : total2 & 0xffffffffu);
  int before = static_cast<int>(ln.align ? before2 >> 32 : before2 & 0xffffffffu);
  const int line = total * per_seq;
  ln.quota = ln.align ? kAlign : max((line + pieces - 1) / pieces, kTileUnits);
  const int begin = static_cast<int>(
      min(static_cast<long long>(blockIdx.x) * ln.quota, static_cast<long long>(line)));
  const int end = min(begin + ln.quota, line);
  for (int b = b0; b < b1; ++b) {
    const Tiles t = tiles_of(p.c, p.rule, b);
    const int n = units_of(t, ln.align);
    if (blockIdx.x == 0 && p.all_partial) p.cum[b] = before;
    const int rel = begin - before * per_seq;
    if (rel >= 0 && rel < n * per_seq) {
      // The first tile that begins at or behind `begin`, maybe of the next item.
      int h = rel / n, tile = (rel - h * n + kTileUnits - 1) / kTileUnits;
      if (tile >= t.n) ++h, tile = 0;
      const bool roll = h == per_seq;
      sh.found[1] = roll ? 0 : h;
      sh.found[2] = tile;
      sh.found[3] = before * per_seq + h * n;
      sh.found[0] = b + roll;
    }
    before += n;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.all_partial) {
    p.cum[p.c.B] = total;
    p.cum[p.c.B + 1] = ln.quota;
    p.cum[p.c.B + 2] = ln.align;
  }
  __syncthreads();
  const int b_first = sh.found[0];
  if (begin >= end || b_first < 0 || b_first >= p.c.B ||
      sh.found[3] + sh.found[2] * kTileUnits >= end) {
    pdl_wait();
    return;
  }

  auto advance = [&](Cursor& x) {
    if (++x.tile < x.t.n) {
      x.u += kTileUnits;
      return;
    }
    x.tile = 0;
    x.item += units_of(x.t, ln.align);
    x.u = x.item;
    if (++x.h < per_seq) return;
    x.h = 0;
    if (++x.b < p.c.B) x.t = tiles_of(p.c, p.rule, x.b);
  };
  // First key of this warp's slice.
  auto slice_key = [&](const Cursor& x) { return tile_key(x.t, x.tile) + warp * kSlice; };
  auto page_at = [&](const Cursor& x) {
    const int key = slice_key(x);
    return key < x.t.len ? __ldg(p.c.table + x.b * p.c.table_stride + (key >> p.c.page_shift)) : 0;
  };

  // Loads.  Lane l moves piece l % 16 of rows l / 16, l / 16 + 2, ...; the page of the next slice
  // is asked for one step ahead.
  Cursor ld;
  ld.b = b_first;
  ld.h = sh.found[1];
  ld.tile = sh.found[2];
  ld.item = sh.found[3];
  ld.u = ld.item + ld.tile * kTileUnits;
  ld.t = tiles_of(p.c, p.rule, ld.b);
  Cursor cx = ld;
  int ld_page = page_at(ld);
  const uint32_t ring = ptx::smem_u32(sh.ring[warp]);
  const int lr = lane >> 4, lc = lane & 15;
  int ld_i = 0;
  auto load_next = [&]() {
    if (ld.u < end) {
      const int key = slice_key(ld);
      if (key < ld.t.len) {
        const int page = page_checked(p.c, ld_page);
        const long long pg = max(page, 0);
        const long long head = ld.h / p.row_tiles;
        const long long slot = key & ((1 << p.c.page_shift) - 1);
        const char* ks = p.c.k + pg * p.c.k_page + head * p.c.k_head + (slot + lr) * p.c.k_tok + lc * 16;
        const char* vs = p.c.v + pg * p.c.v_page + head * p.c.v_head + (slot + lr) * p.c.v_tok + lc * 16;
        const uint32_t dst = ring + (ld_i % kStages) * (2 * kSliceBytes);
        const int have = page < 0 ? 0 : ld.t.len - key;
#pragma unroll
        for (int i = 0; i < kSlice / 2; ++i) {
          const int row = 2 * i + lr;
          const uint32_t d = dst + row * (kHeadDim * 2) + ((lc ^ (row & 7)) << 4);
          const uint32_t bytes = row < have ? 16u : 0u;
          cp_async16(d, ks + 2 * i * p.c.k_tok, bytes);
          cp_async16(d + kSliceBytes, vs + 2 * i * p.c.v_tok, bytes);
        }
      }
      ++ld_i;
      advance(ld);
      if (ld.u < end) ld_page = page_at(ld);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load_next();

  // Per-lane state: columns (rows of q) 8 nb + 2 t4 and + 1.
  uint32_t qf[NB][8][2];
  float o[NB][8][4];
  float m[NB][2], l[NB][2];
  RowKeys rk[NB][2];
  int min_limit = 0, max_lo = 0;
  bool fresh = true;
  int seg_tile0 = 0;
  uint32_t merges = 0;  // uses of the merge buffer so far
  Split rest{0, 0, 0, 0}, head{0, 0, 0, 0};

  // First row of q of item (b, h).
  auto q_row_of = [&](int b, int h) {
    const int head = h / p.row_tiles;
    return (static_cast<long long>(b) * p.c.Hkv + head) * p.rows + (h - head * p.row_tiles) * R;
  };
  auto load_q = [&](int b, int h, uint32_t(&f)[NB][8][2]) {
    const int left = p.rows - (h % p.row_tiles) * R;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q) +
                            (q_row_of(b, h) + nb * 8 + g) * (kHeadDim / 2) + t4;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        f[nb][kk][0] = nb * 8 + g < left ? __ldg(src + kk * 8) : 0u;
        f[nb][kk][1] = nb * 8 + g < left ? __ldg(src + kk * 8 + 4) : 0u;
      }
    }
  };
  // With registers to spare (NB == 1) the next item's rows are fetched while this one is computed.
  constexpr bool kAhead = NB == 1;
  uint32_t qn[kAhead ? NB : 1][8][2];
  if constexpr (kAhead) load_q(cx.b, cx.h, qn);

  for (int i = 0; cx.u < end; ++i) {
    const int row0 = (cx.h % p.row_tiles) * R;
    if (fresh) {
      fresh = false;
      seg_tile0 = cx.tile;
      min_limit = 0x7fffffff;
      max_lo = 0;
      if constexpr (kAhead) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qf[0][kk][0] = qn[0][kk][0];
          qf[0][kk][1] = qn[0][kk][1];
        }
        const bool roll = cx.h + 1 == per_seq;
        if (cx.item + units_of(cx.t, ln.align) < end) load_q(cx.b + roll, roll ? 0 : cx.h + 1, qn);
      } else {
        load_q(cx.b, cx.h, qf);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rr = row0 + nb * 8 + 2 * t4 + e;
          rk[nb][e] = row_keys(cx.t.r, p.rule, p.c.Tq == 1 ? 0 : rr % p.c.Tq);
          if (rr >= p.rows) rk[nb][e] = RowKeys{0x7fffffff, 0};
          min_limit = min(min_limit, rk[nb][e].limit);
          max_lo = max(max_lo, rk[nb][e].lo);
          m[nb][e] = -INFINITY;
          l[nb][e] = 0.0f;
        }
#pragma unroll
        for (int a = 0; a < 8; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nb][a][e] = 0.0f;
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        min_limit = min(min_limit, __shfl_xor_sync(0xffffffffu, min_limit, d));
        max_lo = max(max_lo, __shfl_xor_sync(0xffffffffu, max_lo, d));
      }
    }

    cp_async_wait<kStages - 2>();
    __syncwarp();
    load_next();

    const int key0 = slice_key(cx);
    if (key0 < cx.t.len) {
      const uint32_t kb = ring + (i % kStages) * (2 * kSliceBytes);
      // S^T: lanes 0-15 address keys 0-15 of the lower 8 columns, lanes 16-31 of the upper.
      float s[NB][2][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[nb][e >> 2][e & 3] = 0.0f;
      {
        const int row = lane & 15, up = lane >> 4;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          uint32_t a[4];
          ldsm4(kb + row * (kHeadDim * 2) + (((2 * kk + up) ^ (row & 7)) << 4), a);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma16816<BF16>(s[nb][kk & 1], a, qf[nb][kk]);
        }
      }
      // Scores of lane (g, t4): keys key0 + g (e = 0, 1) and + 8 (e = 2, 3); columns 2 t4 + (e & 1).
      float x[NB][4];
      bool over = false;
      const bool masked = key0 + kSlice > min_limit ||
                          (key0 < max_lo && key0 >= p.rule.glob * kTileKeys);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[nb][e] = (s[nb][0][e] + s[nb][1][e]) * p.scale_log2;
          if (masked) {
            const int key = key0 + g + (e >> 1) * 8;
            const RowKeys k = rk[nb][e & 1];
            if (key >= k.limit || (key < k.lo && key >= p.rule.glob * kTileKeys))
              x[nb][e] = -INFINITY;
          }
          over |= x[nb][e] > m[nb][e & 1] + kRescaleLog2;
        }
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(x[nb][c], x[nb][c + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float mn = fmaxf(m[nb][c], mx);
            const float f = mn == -INFINITY ? 1.0f : ptx::ex2(m[nb][c] - mn);
            m[nb][c] = mn;
            l[nb][c] *= f;
#pragma unroll
            for (int a = 0; a < 8; ++a) {
              o[nb][a][c] *= f;
              o[nb][a][c + 2] *= f;
            }
          }
      }
      uint32_t pf[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float mm = m[nb][e & 1];
          pr[e] = ptx::ex2(x[nb][e] - (mm == -INFINITY ? 0.0f : mm));
          l[nb][e & 1] += pr[e];
        }
        pf[nb][0] = movm_trans(pack16<BF16>(pr[0], pr[1]));
        pf[nb][1] = movm_trans(pack16<BF16>(pr[2], pr[3]));
      }
      // O^T: 16 columns of d per step; lanes 0-7 / 8-15 address keys 0-7 of the lower / upper
      // eight columns, lanes 16-31 keys 8-15.
      {
        const uint32_t vb = kb + kSliceBytes;
        const int row = (lane & 7) + ((lane >> 4) << 3), up = (lane >> 3) & 1;
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          uint32_t f[4];
          ldsm4_trans(vb + row * (kHeadDim * 2) + (((2 * a + up) ^ (row & 7)) << 4), f);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma16816<BF16>(o[nb][a], f, pf[nb]);
        }
      }
    }

    if (cx.tile + 1 == cx.t.n || cx.u + kTileUnits >= end) {
      // The piece ends: join the warps, eight rows at a time.  One barrier: the buffer was read long
      // ago (o_free), and each warp adds up its share of the rows with everyone's maxima in hand.
      const bool whole = !p.all_partial && seg_tile0 == 0 && cx.tile + 1 == cx.t.n;
      const long long q_row = q_row_of(cx.b, cx.h);
      const long long slot = part_slot(p.all_partial, static_cast<long long>(cx.b) * per_seq + cx.h,
                                       static_cast<int>(blockIdx.x), seg_tile0 == 0);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (merges > 0) wait_merge(o_free, (merges - 1) & 1u);
        ++merges;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], d);
          if (g == 0) {
            sh.m[warp][2 * t4 + c] = m[nb][c];
            sh.l[warp][2 * t4 + c] = l[nb][c];
          }
        }
#pragma unroll
        for (int a = 0; a < 8; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sh.o[warp][2 * t4 + (e & 1)][a * 16 + g + (e >> 1) * 8] = o[nb][a][e];
        __syncthreads();
        const int rb = warp * kRowsPerWarp, r = nb * 8 + rb;
        const int live = min(max(p.rows - row0 - r, 0), kRowsPerWarp);  // rows of this warp
        float4 acc[kRowsPerWarp];
        float mx[kRowsPerWarp], sum[kRowsPerWarp];
#pragma unroll
        for (int k = 0; k < kRowsPerWarp; ++k) {
          mx[k] = -INFINITY;
          sum[k] = 0.0f;
          acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (k >= live) continue;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) mx[k] = fmaxf(mx[k], sh.m[w][rb + k]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float mw = sh.m[w][rb + k];
            const float f = mw == -INFINITY ? 0.0f : ptx::ex2(mw - mx[k]);
            const float4 y = *reinterpret_cast<const float4*>(&sh.o[w][rb + k][lane * 4]);
            sum[k] += sh.l[w][rb + k] * f;
            acc[k].x += y.x * f;
            acc[k].y += y.y * f;
            acc[k].z += y.z * f;
            acc[k].w += y.w * f;
          }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(o_free);
#pragma unroll
        for (int k = 0; k < kRowsPerWarp; ++k) {
          if (k >= live) continue;
          const float inv = sum[k] > 0.0f ? 1.0f / sum[k] : 0.0f;
          const float lg = sum[k] > 0.0f ? mx[k] + log2f(sum[k]) : -INFINITY;
          const float4 v = make_float4(acc[k].x * inv, acc[k].y * inv, acc[k].z * inv, acc[k].w * inv);
          if (whole) {
            store_row(p.o, p.lse, p.out_bf16, q_row + r + k, v, lg, lane);
          } else {
            reinterpret_cast<float4*>(p.part_o)[(slot * R + r + k) * (kHeadDim / 4) + lane] = v;
            if (lane == 0) p.part_l[slot * R + r + k] = lg;
          }
        }
      }
      if (!whole) {
        Split& sp = seg_tile0 == 0 ? head : rest;
        sp.first = cx.item / ln.quota;
        sp.last = last_piece(ln, cx.item, units_of(cx.t, ln.align));
        sp.q_row = q_row;
        sp.rows = min(p.rows - row0, R);
      }
      fresh = true;
    }
    advance(cx);
  }
  cp_async_wait<0>();
  if (!p.all_partial && (head.rows > 0 || rest.rows > 0)) {
    // The warp that finds its rows' pieces complete adds them up, in the order of the line.  Asked
    // for once, at the CTA's end: the fence and the counter cost a round trip to L2 each.
    int done[2][NB];
    __threadfence();
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const Split& sp = e ? head : rest;
        const int r = nb * 8 + warp * kRowsPerWarp;
        done[e][nb] = -1;
        if (lane == 0 && r < sp.rows)
          done[e][nb] = atomicAdd(p.counters + sp.first * kFewRows + nb * kWarps + warp, 1);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const Split& sp = e ? head : rest;
        const int r = nb * 8 + warp * kRowsPerWarp;
        if (__shfl_sync(0xffffffffu, done[e][nb], 0) != sp.last - sp.first || r >= sp.rows) continue;
        __threadfence();
        if (lane == 0) p.counters[sp.first * kFewRows + nb * kWarps + warp] = 0;
        join_own(p, sp.q_row + r, r, min(sp.rows - r, kRowsPerWarp), R, sp.first, sp.last, lane);
      }
  }
  // Behind a shared prefix this kernel starts while the prefix's still runs, and must not end
  // before it: the join waits for this kernel only.
  pdl_wait();
}

// Joins behind a shared prefix: every row of the call, W warps a row, over the pieces of its own
// keys in the order of the line, then over those of the prefix.
struct RowJoin {
  int Hkv, rows;         // rows = G * Tq
  long long total;       // B * Hq * Tq
  void* o;
  float* lse;
  int out_bf16;
  const int* cum;        // own keys, by the few-row kernel
  const float* part_o;
  const float* part_l;
  int B, R, row_tiles;
  const float* pre_o;    // prefix: n_b sequences per tile of rows, tiles_p tiles per item
  const float* pre_l;
  int n_b, tiles_p, quota_p;
};
constexpr int kJoinWarps = 4;
template <int W>
__global__ void __launch_bounds__(kJoinWarps * 32) join_rows_kernel(const __grid_constant__ RowJoin p) {
  __shared__ float4 so[kJoinWarps][32];
  __shared__ float sl[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = W == 1 ? static_cast<long long>(blockIdx.x) * kJoinWarps + warp : blockIdx.x;
  if (row >= p.total) return;
  const int bh = static_cast<int>(row / p.rows), rr = static_cast<int>(row - static_cast<long long>(bh) * p.rows);
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int hr = h * p.row_tiles + rr / p.R, r = rr % p.R;
  const int heads = p.Hkv * p.row_tiles;
  const long long item_p = static_cast<long long>(b / p.n_b) * p.Hkv + h;
  const int rp = (b % p.n_b) * p.rows + rr;
  const long long sp = item_p * p.tiles_p;
  const int first_p = static_cast<int>(sp / p.quota_p);
  const int pre = static_cast<int>((sp + p.tiles_p - 1) / p.quota_p) - first_p + 1;
  pdl_wait();
  const int c0 = p.cum[b], n = p.cum[b + 1] - c0;
  const Line ln{p.cum[p.B + 1], p.cum[p.B + 2]};
  const int s = c0 * heads + hr * n;
  const int first = s / ln.quota, own = last_piece(ln, s, n) - first + 1;
  const long long item = static_cast<long long>(b) * heads + hr;
  const float *po[2] = {p.part_o, p.pre_o}, *pl[2] = {p.part_l, p.pre_l};
  const long long at[2] = {(item + first) * p.R + r, (item_p + first_p) * 128 + rp};
  const int step[2] = {p.R, 128}, count[2] = {own, pre};
  float mx = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int c = lane; c < count[k]; c += 32)
      mx = fmaxf(mx, pl[k][at[k] + static_cast<long long>(c) * step[k]]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  PartSum acc{make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f};
  if (mx > -INFINITY) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll 4
      for (int c = W == 1 ? 0 : warp; c < count[k]; c += W) {
        const long long x = at[k] + static_cast<long long>(c) * step[k];
        acc.add(part_row(po[k], x, lane), ptx::ex2(pl[k][x] - mx));
      }
    }
  }
  if (W > 1) {
    so[warp][lane] = acc.acc;
    if (lane == 0) sl[warp] = acc.sum;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float4 y = so[w][lane];
      acc.acc.x += y.x;
      acc.acc.y += y.y;
      acc.acc.z += y.z;
      acc.acc.w += y.w;
      acc.sum += sl[w];
    }
  }
  const float inv = acc.sum > 0.0f ? 1.0f / acc.sum : 0.0f;
  store_row(p.o, p.lse, p.out_bf16, row,
            make_float4(acc.acc.x * inv, acc.acc.y * inv, acc.acc.z * inv, acc.acc.w * inv),
            acc.sum > 0.0f ? mx + log2f(acc.sum) : -INFINITY, lane);
}

// Joins the items that the many-row kernel's line was cut in: at most one begins in each CTA and
// goes on in the next ones (TileCut).  Block (c, y): rows 16 y .. of that item, a warp each four.
struct CutJoin {
  const TileCut* cuts;
  RowTiles rt;
  int Hkv, Tq;
  void* o;
  float* lse;
  int out_bf16;
  const float* part_o;
  const float* part_l;
};
__global__ void __launch_bounds__(kJoinWarps * 32) join_cuts_kernel(const __grid_constant__ CutJoin p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x;
  pdl_wait();
  const TileCut cut = p.cuts[first];
  if (cut.v < 0) return;
  const int b = cut.v / p.rt.per_seq, t0 = (cut.v - b * p.rt.per_seq) * p.rt.n_t;
  for (int k = 0; k < 4; ++k) {
    const int r = blockIdx.y * 16 + warp * 4 + k;
    const int g = r / p.rt.n_t, t = t0 + r - g * p.rt.n_t;
    if (g >= p.rt.G || t >= p.Tq) continue;
    float mx = -INFINITY;
    for (int c = lane; c < cut.pieces; c += 32)
      mx = fmaxf(mx, p.part_l[part_slot(0, 0, first + c, c == 0) * 128 + r]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    PartSum acc{make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f};
    if (mx > -INFINITY) {
#pragma unroll 4
      for (int c = 0; c < cut.pieces; ++c) {
        const long long x = part_slot(0, 0, first + c, c == 0) * 128 + r;
        acc.add(part_row(p.part_o, x, lane), ptx::ex2(p.part_l[x] - mx));
      }
    }
    const float inv = acc.sum > 0.0f ? 1.0f / acc.sum : 0.0f;
    const long long row = ((static_cast<long long>(b) * p.Hkv + cut.h) * p.rt.G + g) * p.Tq + t;
    store_row(p.o, p.lse, p.out_bf16, row,
              make_float4(acc.acc.x * inv, acc.acc.y * inv, acc.acc.z * inv, acc.acc.w * inv),
              acc.sum > 0.0f ? mx + log2f(acc.sum) : -INFINITY, lane);
  }
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
int device_sms(int* sms) {
  static std::mutex mu;
  static int known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return BSATTN_E_CUDA;
  std::lock_guard<std::mutex> lk(mu);
  if (known[dev] == 0) {
    const int rc = bsattn_setup();
    if (rc != BSATTN_OK) return rc;
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return BSATTN_E_CUDA;
    n = std::min(n, kMaxSms);
    const void* kernels[] = {
        reinterpret_cast<const void*>(decode_kernel<false, 1>),
        reinterpret_cast<const void*>(decode_kernel<true, 1>),
        reinterpret_cast<const void*>(decode_kernel<false, 2>),
        reinterpret_cast<const void*>(decode_kernel<true, 2>)};
    for (int i = 0; i < 4; ++i)
      if (cudaFuncSetAttribute(kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(i < 2 ? sizeof(DecodeSmem<1>)
                                                      : sizeof(DecodeSmem<2>))) != cudaSuccess)
        return BSATTN_E_CUDA;
    const int rt = tile_setup();
    if (rt != BSATTN_OK) return rt;
    known[dev] = n;
  }
  *sms = known[dev];
  return BSATTN_OK;
}

int fill_cache(Cache* c, const bsattn_paged_call* a) {
  if (!a || !a->k_pages || !a->v_pages || !a->block_table || !a->seq_lens) return BSATTN_E_NULL;
  if (a->B < 1 || a->Hkv < 1 || a->Tq < 1 || a->max_pages < 1 || a->n_pages < 1 || a->table_stride < 0)
    return BSATTN_E_SHAPE;
  if (a->page_size < 16 || a->page_size > 1024 || (a->page_size & (a->page_size - 1)) != 0)
    return BSATTN_E_SHAPE;
  if (static_cast<long long>(a->max_pages) * a->page_size > (1ll << 31) - 2 * kTileKeys)
    return BSATTN_E_SHAPE;
  if (!a->workspace || a->workspace_bytes < bsattn_workspace_bytes()) return BSATTN_E_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(a->k_pages) & 15u) != 0 ||
      (reinterpret_cast<uintptr_t>(a->v_pages) & 15u) != 0)
    return BSATTN_E_ALIGN;
  const int dims[3] = {a->n_pages, a->Hkv, a->page_size};
  for (int i = 0; i < 6; ++i) {
    const int64_t st = a->page_strides[i];
    if (st < 0 || st % 8 != 0 || (st == 0 && dims[i % 3] > 1)) return BSATTN_E_ALIGN;
  }
  c->k = static_cast<const char*>(a->k_pages);
  c->v = static_cast<const char*>(a->v_pages);
  c->k_page = a->page_strides[0] * 2;
  c->k_head = a->page_strides[1] * 2;
  c->k_tok = a->page_strides[2] * 2;
  c->v_page = a->page_strides[3] * 2;
  c->v_head = a->page_strides[4] * 2;
  c->v_tok = a->page_strides[5] * 2;
  c->table = a->block_table;
  c->table_stride = a->table_stride;
  c->seq_lens = a->seq_lens;
  c->q_lens = a->q_lens;
  c->max_pages = a->max_pages;
  c->n_pages = a->n_pages;
  c->page_shift = 0;
  while ((1 << c->page_shift) < a->page_size) ++c->page_shift;
  c->B = a->B;
  c->Hkv = a->Hkv;
  c->Tq = a->Tq;
  c->err = static_cast<int*>(a->workspace);
  return BSATTN_OK;
}

// The launches of one call and their scratch.
struct Shape {
  int rows;         // G * Tq
  bool few;         // own keys by the few-row kernel
  bool prefix;      // prefix keys by the many-row kernel, stacked over the batch
  int k0;           // first own key
  int R, row_tiles, pieces, count;
  bool all_partial;
  RowTiles rt;      // of the many-row kernel's launch
  int tiles_p, pieces_p;
  long long slots, slots_p;
  size_t cum, cuts, part_o, part_l, pre_o, pre_l, bytes;  // offsets into the scratch
};

constexpr int kStackedRows = 64; // more rows of one sequence fill a tile without its neighbours

static int shape_of(int B, int Hq, int Hkv, int Tq, int max_pages, int page_size, int prefix_len,
                    int sms, Shape* s) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 || Tq < 1) return BSATTN_E_SHAPE;
  const int G = Hq / Hkv;
  const long long rows = static_cast<long long>(G) * Tq;
  if (rows * B * Hkv > (1ll << 31) - 1) return BSATTN_E_SHAPE;
  s->rows = static_cast<int>(rows);
  s->prefix = prefix_len > 0 && rows <= kStackedRows;
  s->few = s->prefix || rows <= kFewRows || G > 128;
  s->k0 = s->prefix ? prefix_len : 0;
  s->all_partial = s->prefix;
  // Most tiles one item can have.
  const int step = s->few ? kStep : kTileKeys;
  const long long tiles = (static_cast<long long>(max_pages) * page_size + step - 1) / step + 1;
  long long items;
  if (s->few) {
    s->R = rows <= 8 ? 8 : kFewRows;
    s->row_tiles = static_cast<int>((rows + s->R - 1) / s->R);
    s->count = B;
    items = static_cast<long long>(B) * Hkv * s->row_tiles;
  } else {
    s->R = 128;
    s->row_tiles = 1;
    s->rt.G = G;
    s->rt.n_t = std::min(Tq, 128 / G);
    s->rt.n_b = 1;
    s->rt.per_seq = (Tq + s->rt.n_t - 1) / s->rt.n_t;
    const long long count = static_cast<long long>(B) * s->rt.per_seq;
    items = count * Hkv;
    if (items * tiles > (1ll << 30)) return BSATTN_E_SHAPE;
    s->rt.count = s->count = static_cast<int>(count);
  }
  if (items * (tiles * kTileUnits + kAlign) > (1ll << 30)) return BSATTN_E_SHAPE;
  s->pieces = static_cast<int>(std::min<long long>(s->few ? sms * kCtasPerSm : sms, items * tiles));
  s->slots = s->all_partial ? items + s->pieces : 2ll * s->pieces;
  s->tiles_p = s->pieces_p = 0;
  s->slots_p = 0;
  if (s->prefix) {
    s->rt.G = G;
    s->rt.n_t = Tq;
    s->rt.n_b = std::min(B, 128 / s->rows);
    s->rt.per_seq = 1;
    s->rt.count = (B + s->rt.n_b - 1) / s->rt.n_b;
    s->tiles_p = (prefix_len + kTileKeys - 1) / kTileKeys;
    const long long items_p = static_cast<long long>(s->rt.count) * Hkv;
    if (items_p * s->tiles_p > (1ll << 30)) return BSATTN_E_SHAPE;
    s->pieces_p = static_cast<int>(std::min<long long>(sms, items_p * s->tiles_p));
    s->slots_p = items_p + s->pieces_p;
  }
  if (s->slots * s->R > (1ll << 31) - 1 || s->slots_p * 128 > (1ll << 31) - 1) return BSATTN_E_SHAPE;
  size_t at = 0;
  auto take = [&](long long n) {
    const size_t here = at;
    at += (static_cast<size_t>(n) * sizeof(float) + 255) / 256 * 256;
    return here;
  };
  s->cum = take(s->prefix ? s->count + 3 : 0);
  s->cuts = take(s->few ? 0 : s->pieces * static_cast<long long>(sizeof(TileCut) / sizeof(float)));
  s->part_o = take(s->slots * s->R * kHeadDim);
  s->part_l = take(s->slots * s->R);
  s->pre_o = take(s->slots_p * 128 * kHeadDim);
  s->pre_l = take(s->slots_p * 128);
  s->bytes = at;
  return BSATTN_OK;
}

// A launch that may start while its predecessor still runs.
template <class P>
static bool launch_overlapped(void (*kernel)(P), dim3 grid, int threads, size_t smem,
                              cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}

static int launch_paged(const void* q, const Cache& cache, Rule rule, int prefix_len, int Hq,
                        float scale, int dtype_flags, int page_size, void* o, float* lse,
                        void* scratch, size_t scratch_bytes, int* counters, cudaStream_t stream) {
  if (!q || !o || !counters) return BSATTN_E_NULL;
  if ((dtype_flags & ~(BSATTN_OUT_BF16 | BSATTN_IN_BF16)) != 0) return BSATTN_E_DTYPE;
  if ((reinterpret_cast<uintptr_t>(q) & 15u) != 0 || (reinterpret_cast<uintptr_t>(o) & 15u) != 0 ||
      (reinterpret_cast<uintptr_t>(scratch) & 15u) != 0)
    return BSATTN_E_ALIGN;
  int sms = 0;
  int rc = device_sms(&sms);
  if (rc != BSATTN_OK) return rc;
  Shape s;
  rc = shape_of(cache.B, Hq, cache.Hkv, cache.Tq, cache.max_pages, page_size, prefix_len, sms, &s);
  if (rc != BSATTN_OK) return rc;
  if (!scratch || scratch_bytes < s.bytes) return BSATTN_E_WORKSPACE;
  char* const base = static_cast<char*>(scratch);
  const double sc = scale > 0.0f ? static_cast<double>(scale) : 0.08838834764831845;
  const bool bf16 = (dtype_flags & BSATTN_IN_BF16) != 0;
  const int out_bf16 = (dtype_flags & BSATTN_OUT_BF16) != 0;
  const float scale_log2 = static_cast<float>(sc * 1.4426950408889634);
  rule.k0 = s.k0;

  if (s.prefix || !s.few) {
    TileCall t;
    t.c = cache;
    t.rule = rule;
    t.rule.k0 = 0;
    t.rt = s.rt;
    t.prefix_len = s.prefix ? prefix_len : 0;
    t.q = q;
    t.o = o;
    t.lse = lse;
    t.Hq = Hq;
    t.scale_log2 = scale_log2;
    t.in_bf16 = bf16;
    t.out_bf16 = out_bf16;
    t.pieces = s.prefix ? s.pieces_p : s.pieces;
    t.slots = s.prefix ? s.slots_p : s.slots;
    t.cuts = reinterpret_cast<TileCut*>(base + s.cuts);
    t.part_o = reinterpret_cast<float*>(base + (s.prefix ? s.pre_o : s.part_o));
    t.part_l = reinterpret_cast<float*>(base + (s.prefix ? s.pre_l : s.part_l));
    if ((rc = tile_launch(t, page_size, stream)) != BSATTN_OK) return rc;
  }
  if (s.few) {
    AttnParams p;
    p.c = cache;
    p.rule = rule;
    p.q = q;
    p.o = o;
    p.lse = lse;
    p.rows = s.rows;
    p.row_tiles = s.row_tiles;
    p.scale_log2 = scale_log2;
    p.out_bf16 = out_bf16;
    p.all_partial = s.all_partial;
    p.cum = reinterpret_cast<int*>(base + s.cum);
    p.part_o = reinterpret_cast<float*>(base + s.part_o);
    p.part_l = reinterpret_cast<float*>(base + s.part_l);
    p.counters = counters;
    const unsigned grid = static_cast<unsigned>(s.pieces);
    void (*kernel)(AttnParams) = s.R == 8 ? (bf16 ? decode_kernel<true, 1> : decode_kernel<false, 1>)
                                          : (bf16 ? decode_kernel<true, 2> : decode_kernel<false, 2>);
    const size_t smem = s.R == 8 ? sizeof(DecodeSmem<1>) : sizeof(DecodeSmem<2>);
    if (s.prefix) {
      if (!launch_overlapped(kernel, grid, kThreadsD, smem, stream, p)) return BSATTN_E_CUDA;
    } else {
      kernel<<<grid, kThreadsD, smem, stream>>>(p);
      if (cudaGetLastError() != cudaSuccess) return BSATTN_E_CUDA;
    }
  }
  if (s.prefix) {
    RowJoin j;
    j.Hkv = cache.Hkv;
    j.rows = s.rows;
    j.total = static_cast<long long>(cache.B) * Hq * cache.Tq;
    j.o = o;
    j.lse = lse;
    j.out_bf16 = out_bf16;
    j.cum = reinterpret_cast<const int*>(base + s.cum);
    j.part_o = reinterpret_cast<const float*>(base + s.part_o);
    j.part_l = reinterpret_cast<const float*>(base + s.part_l);
    j.B = cache.B;
    j.R = s.R;
    j.row_tiles = s.row_tiles;
    j.pre_o = reinterpret_cast<const float*>(base + s.pre_o);
    j.pre_l = reinterpret_cast<const float*>(base + s.pre_l);
    j.n_b = s.rt.n_b;
    j.tiles_p = s.tiles_p;
    const long long items_p = static_cast<long long>(s.rt.count) * cache.Hkv;
    j.quota_p = static_cast<int>((items_p * s.tiles_p + s.pieces_p - 1) / s.pieces_p);
    // A row of many pieces is shared by four warps.
    const bool ok =
        s.pieces_p / items_p >= 8
            ? launch_overlapped(join_rows_kernel<kJoinWarps>, static_cast<unsigned>(j.total),
                                kJoinWarps * 32, 0, stream, j)
            : launch_overlapped(join_rows_kernel<1>,
                                static_cast<unsigned>((j.total + kJoinWarps - 1) / kJoinWarps),
                                kJoinWarps * 32, 0, stream, j);
    if (!ok) return BSATTN_E_CUDA;
  } else if (!s.few) {
    CutJoin j;
    j.cuts = reinterpret_cast<const TileCut*>(base + s.cuts);
    j.rt = s.rt;
    j.Hkv = cache.Hkv;
    j.Tq = cache.Tq;
    j.o = o;
    j.lse = lse;
    j.out_bf16 = out_bf16;
    j.part_o = reinterpret_cast<const float*>(base + s.part_o);
    j.part_l = reinterpret_cast<const float*>(base + s.part_l);
    const unsigned groups = static_cast<unsigned>((s.rt.n_t * s.rt.G + 15) / 16);
    if (!launch_overlapped(join_cuts_kernel, dim3(static_cast<unsigned>(s.pieces), groups),
                           kJoinWarps * 32, 0, stream, j))
      return BSATTN_E_CUDA;
  }
  return BSATTN_OK;
}

}  // namespace paged
}  // namespace bsattn

using namespace bsattn;
using namespace bsattn::paged;

extern "C" {

int bsattn_paged_scratch_bytes(int B, int Hq, int Hkv, int Tq, int max_pages, int page_size,
                               int prefix_len, size_t* bytes) {
  if (!bytes) return BSATTN_E_NULL;
  if (prefix_len < 0) return BSATTN_E_SHAPE;
  if (max_pages < 1 || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
    return BSATTN_E_SHAPE;
  int sms = 0;
  int rc = device_sms(&sms);
  if (rc != BSATTN_OK) return rc;
  Shape s;
  rc = shape_of(B, Hq, Hkv, Tq, max_pages, page_size, prefix_len, sms, &s);
  if (rc != BSATTN_OK) return rc;
  *bytes = s.bytes;
  return BSATTN_OK;
}

int bsattn_paged_counters(void) { return kMaxSms * kCtasPerSm * kFewRows; }

int bsattn_paged_fwd(const bsattn_paged_call* call, const void* q, void* o, float* lse, int window,
                     int global_blocks, int prefix_len, float scale, void* scratch,
                     size_t scratch_bytes, int32_t* counters) {
  Cache c;
  const int rc = fill_cache(&c, call);
  if (rc != BSATTN_OK) return rc;
  constexpr int kMaxWindow = 1 << 24;
  if (window < 0 || window > kMaxWindow || global_blocks < 0 || global_blocks > kMaxWindow ||
      (window == 0 && global_blocks != 0))
    return BSATTN_E_SHAPE;
  if (prefix_len < 0 || prefix_len % call->page_size != 0 ||
      prefix_len > static_cast<long long>(call->max_pages) * call->page_size ||
      (prefix_len > 0 && window > 0))
    return BSATTN_E_SHAPE;
  const Rule rule{0, window, global_blocks};
  return launch_paged(q, c, rule, prefix_len, call->Hq, scale, call->dtype_flags, call->page_size, o,
                      lse, scratch, scratch_bytes, counters, static_cast<cudaStream_t>(call->stream));
}

}  // extern "C"

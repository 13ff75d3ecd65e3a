// paged_few.cu -- attention of a few rows per key over a paged K/V cache: the decode form.
//
// Rows: q [B, Hq, Tq, 128]; the G = Hq / Hkv query heads that share a K/V head form, with their Tq
// tokens, the G * Tq rows (g-major) that one pass over that head's keys serves.  For row (g, t) at
// position p = seq_lens[b] - q_lens[b] + t:
//     o = sum_j softmax_j(scale q . k_j) v_j over the keys j <= p (and the window rule),
//     lse = ln sum_j exp(scale q . k_j);  no key: o = 0, lse = -inf.
//
// Every key costs 512 bytes of HBM and G * Tq * 512 operations, so the bound is memory; what matters
// is that all SMs read all the time and that nothing waits for anything else.
//   * Every warp is on its own.  It owns a share of the line of all (sequence, K/V head) items
//     (paged_few.cuh), in units of 16 keys, loads its slices with cp.async into a private ring (16-byte
//     pieces swizzled so that ldmatrix reads without bank conflicts) and keeps its own running maximum,
//     sum and output.  The ring runs across item borders.  A short item lies inside one warp's share
//     and is written by it, with no barrier at all; only at the CTA's end do its warps meet, once, to
//     add up the items that lie across their shares.  Cutting by units balances sequences of any mix of
//     lengths.  The lengths are on the device: each CTA adds them up itself.
//   * Keys are the M dimension of the warp MMAs (m16n8k16): S^T = K Q^T and O^T = V^T P^T, so eight
//     rows fill an MMA's N and none of it is spent on padding; P^T moves from the accumulator to the
//     operand layout with movmatrix, in registers.
//   * The running maximum moves only when a score passes it by more than 2^8 (then P stays within
//     2^8, far inside fp16 and bf16); the usual step costs one vote instead of a reduction.
//   * Parts of an item that lies across CTAs are left as (o, log2 sum) in 32 bits, and the warp that
//     finds its row's parts complete adds them, in the order of the line: results do not depend on
//     timing.
// Keys past a sequence's end are loaded as zeros, never read: a recycled page may hold anything.
// P is rounded to the type of V (fp16: 11 bits, bf16: 8), since one MMA takes both operands in one type and
// a V converted to fp16 would lose what lies past its range; its sum is of the unrounded values.
#include <algorithm>
#include <atomic>

#include "paged_few.cuh"
#include "sm100_ptx.cuh"

namespace bsattn {
namespace paged {
namespace few {

constexpr int kStages = 3;
constexpr int kSliceBytes = kSlice * kHeadDim * 2;  // 4 KB of K or of V
constexpr int kStageBytes = 2 * kSliceBytes;
constexpr float kRescaleLog2 = 8.0f;
// When to give every item CTAs of its own (Line::align).  A part of at least kPartUnits units, since
// joining parts takes 3 us and a CTA 16 units in 1.5; up to kWholeUnits an item is not cut at all (512
// keys: 11.1 us, cut in two 11.9); and rather than cutting the line in equal pieces as long as a part is
// no more than kCutUnits units longer than such a piece, of which most CTAs hold two (16 heads, 8,192
// keys: 21.5 us in parts of 64 units, 23.6 in pieces of 56).
constexpr int kPartUnits = 16, kWholeUnits = 32, kCutUnits = 16;
constexpr int kWarps = 8, kThreads = kWarps * 32;

struct Params {
  Cache c;
  Rule rule;
  const void* q;
  void* o;
  float* lse;
  int rows, row_tiles;
  float scale_log2;
  int out_bf16, all_partial, packed;
  int* cum;
  float* part_o;
  float* part_l;
  int* counters;
  int* others;  // the half of them that this call does not use
};

// What a warp leaves of an item that is not its own alone: which item, and the rows' maxima and sums.
struct Part {
  float m[kFewRows], l[kFewRows];
  int item;           // b * per_seq + h; < 0: none
  int first, last;    // the CTAs it lies in
  int live;           // its rows
  long long q_row;    // the first of them
};

// The slices of one sequence, those any live row sees, in ascending order: n_glob leading ones, then
// those from key `lo` on.  A sequence without a key or a live row still gets one slice, so that every
// row is written by the same path; its length is 0 here, so nothing of it is read.
struct Slices {
  int len;
  Rows r;
  int n, n_glob, lo;
};
__device__ __forceinline__ Slices slices_of(const Params& p, int b) {
  const SeqLen s = seq_len(p.c, b);
  Slices t;
  t.len = s.rows > 0 ? s.len : 0;
  t.r = Rows{s.rows, s.len - s.rows};
  t.lo = p.rule.k0;
  t.n_glob = 0;
  t.n = 1;
  if (s.rows > 0 && s.len > p.rule.k0) {
    if (p.rule.window > 0) {
      const int block = max(0, max(t.r.first, 0) / kTileKeys - p.rule.window + 1);
      t.lo = block * kTileKeys;
      t.n_glob = min(p.rule.glob, block) * (kTileKeys / kSlice);
    }
    t.n = t.n_glob + (s.len - t.lo + kSlice - 1) / kSlice;
  }
  return t;
}

// A slice on the line.
struct Cursor {
  int b, h, k;  // h counts (K/V head, tile of rows)
  int at;       // first unit of the item
  Slices t;
  __device__ __forceinline__ int key() const {
    return k < t.n_glob ? k * kSlice : t.lo + (k - t.n_glob) * kSlice;
  }
};

struct Smem {
  uint8_t ring[kWarps][kStages][kStageBytes];
  float rest_o[kWarps][kFewRows][kHeadDim];    // of the item that began before the warp's share
  Part part[kWarps][2];                        // that one, and the one that goes on behind the share
  int warp_sum[2][kWarps], longest[kWarps];
  Cursor found;
};

// Where 16-byte piece c (0 .. 31) of row r of a warp's outputs lies: the four rows that the lanes of
// an accumulator store write at once fall into different banks.
__device__ __forceinline__ int piece(int r, int c) { return c ^ (r & 6); }

// One warp, one row: o = sum_c o_c 2^(l_c - l), l = log2 sum 2^l_c over the parts of CTAs first ..
// last, in that order, eight asked for at a time.
__device__ __noinline__ void join_row(const Params& p, long long row, int r, int R, int first, int last,
                                      int lane) {
  constexpr int kAtOnce = 8;
  const int n = last - first + 1;
  float mx = -INFINITY;
  PartSum s;
  s.clear();
  for (int c0 = 0; c0 < n; c0 += kAtOnce) {
    float4 y[kAtOnce];
    float lg[kAtOnce];
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c) {
      lg[c] = -INFINITY;
      y[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (c0 + c < n) {
        const long long at = part_slot(0, 0, first + c0 + c, c0 + c == 0) * R + r;
        lg[c] = __ldcg(p.part_l + at);
        y[c] = part_row(p.part_o, at, lane);
      }
    }
    float top = mx;
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c) top = fmaxf(top, lg[c]);
    if (top == -INFINITY) continue;
    s.scale(ptx::ex2(mx - top));
    mx = top;
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c) s.add(y[c], ptx::ex2(lg[c] - top));
  }
  store_row(p.o, p.lse, p.out_bf16, row, s.normal(), s.log2_total(mx), lane);
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1) few_kernel(const __grid_constant__ Params p) {
  constexpr int W = kWarps, R = kFewRows;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sh = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int per_seq = p.c.Hkv * p.row_tiles;
  // Behind a shared prefix this kernel runs beside the prefix's (paged_attn.cu says how).
  if (!p.all_partial) pdl_wait();
  pdl_trigger();

  // The line.  Up to 32 sequences every warp lays out by itself, one per lane, with no barrier (8 sequences
  // of 1,000 keys: 14.8 us against 15.1); more of them the block's threads, some each.
  const bool alone = p.c.B <= 32;
  const int chunk = alone ? 1 : (p.c.B + kThreads - 1) / kThreads;
  const int b0 = min((alone ? lane : static_cast<int>(threadIdx.x)) * chunk, p.c.B);
  const int b1 = min(b0 + chunk, p.c.B);
  int mine = 0, longest = 0;
  Slices t0 = {};  // of sequence b0; the only one in most calls
  for (int b = b0; b < b1; ++b) {
    const Slices t = slices_of(p, b);
    if (b == b0) t0 = t;
    mine += units_of(t.n, 0);
    longest = max(longest, t.n);
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  // What lies before this thread's sequences, and in all.
  auto sums = [&](int x, int* shared, int& before, int& total) {
    int incl = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    before = incl - x;
    total = __shfl_sync(0xffffffffu, incl, 31);
    if (alone) return;
    if (lane == 0) {
      shared[warp] = total;
      sh.longest[warp] = longest;
    }
    __syncthreads();
    total = 0;
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += shared[w];
      total += shared[w];
      longest = max(longest, sh.longest[w]);
    }
  };
  int before, total;
  sums(mine, sh.warp_sum[0], before, total);
  const int ctas = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
  const int line_plain = total * per_seq, quota_plain = (line_plain + ctas - 1) / ctas;
  Line ln{quota_plain, 0};
  const int spare = max(ctas - p.c.B * per_seq, 1);  // CTAs behind one for every item
  if (ctas >= p.c.B * per_seq) {
    // Two part lengths that fit: each item in as many parts as there are CTAs for every item, or as many
    // as its length gives beside one CTA of its own.
    const int each = ctas / (p.c.B * per_seq);
    const int fit = min((longest + each - 1) / each, (line_plain + spare - 1) / spare);
    const int align = longest <= kWholeUnits ? kWholeUnits : max(fit, kPartUnits);
    if (align <= max(quota_plain, kPartUnits) + kCutUnits) ln = Line{align, align};
  }
  if (ln.align > 0) sums(b0 < b1 ? units_of(t0.n, ln.align) : 0, sh.warp_sum[1], before, total);
  const int line = total * per_seq;
  const int cta_begin =
      static_cast<int>(min(static_cast<long long>(cta) * ln.quota, static_cast<long long>(line)));
  const int cta_end = min(cta_begin + ln.quota, line);
  // The item that holds the CTA's first unit.
  Cursor ld = {};
  bool here = false;
  for (int b = b0; b < b1; ++b) {
    if (b > b0) t0 = slices_of(p, b);
    const int n = units_of(t0.n, ln.align);
    if (cta == 0 && p.all_partial) p.cum[b] = before;
    const int rel = cta_begin - before * per_seq;
    if (rel >= 0 && rel < n * per_seq) {
      const int h = rel / n;
      ld = Cursor{b, h, 0, before * per_seq + h * n, t0};
      here = true;
    }
    before += n;
  }
  if (cta == 0 && threadIdx.x == 0 && p.all_partial) {
    p.cum[p.c.B] = total;
    p.cum[p.c.B + 1] = ln.quota;
    p.cum[p.c.B + 2] = ln.align;
  }
  if (alone) {
    const uint32_t at = __ballot_sync(0xffffffffu, here);
    int* const words = reinterpret_cast<int*>(&ld);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(Cursor) / sizeof(int)); ++i)
      words[i] = __shfl_sync(0xffffffffu, words[i], at ? __ffs(at) - 1 : 0);
  } else {
    if (here) sh.found = ld;
    __syncthreads();
    ld = sh.found;
  }
  if (cta_begin >= cta_end) {
    if (p.all_partial && blockIdx.x + 1 == gridDim.x) pdl_wait();
    return;
  }

  // This warp's share, and its first slice.
  const int stop = ln.align > 0 ? min(cta_end, ld.at + ld.t.n) : cta_end;
  const int units = stop - cta_begin;
  const int begin = cta_begin + units * warp / W, end = cta_begin + units * (warp + 1) / W;
  auto next_item = [&](Cursor& x) {
    x.at += units_of(x.t.n, ln.align);
    x.k = 0;
    if (++x.h < per_seq) return;
    x.h = 0;
    if (++x.b < p.c.B) x.t = slices_of(p, x.b);
  };
  while (ld.at < end && ld.at + ld.t.n <= begin) next_item(ld);
  ld.k = max(begin - ld.at, 0);
  auto valid = [&](const Cursor& x) { return x.at + x.k < end; };
  auto advance = [&](Cursor& x) {
    if (++x.k == x.t.n) next_item(x);
  };
  auto page_at = [&](const Cursor& x) {
    const int key = x.key();
    return key < x.t.len ? __ldg(p.c.table + x.b * p.c.table_stride + (key >> p.c.page_shift)) : 0;
  };
  Cursor cx = ld;

  // Loads.  Lane l moves piece l % 16 of rows l / 16, l / 16 + 2, ...; the page of the next slice is
  // asked for one step ahead.
  int ld_page = valid(ld) ? page_at(ld) : 0;
  const uint32_t ring = ptx::smem_u32(sh.ring[warp]);
  const int lr = lane >> 4, lc = lane & 15;
  const uint32_t ld_dst = lr * (kHeadDim * 2) + ((lc ^ lr) << 4);
  int ld_stage = 0;
  // Behind a prefix this leaves its keys and the partial results in L2: 256 sequences behind 8,192 tokens
  // 107 us without it, 100 with it; 64 behind 32,768 81 and 78.
  const uint64_t pol = evict_first_policy();
  auto load_next = [&]() {
    if (valid(ld)) {
      const int key = ld.key();
      if (key < ld.t.len) {
        const int page = page_checked(p.c, ld_page);
        const long long pg = max(page, 0);
        const long long head = ld.h / p.row_tiles;
        const long long slot = (key & ((1 << p.c.page_shift) - 1)) + lr;
        const char* ks = p.c.k + pg * p.c.k_page + head * p.c.k_head + slot * p.c.k_tok + lc * 16;
        const char* vs = p.c.v + pg * p.c.v_page + head * p.c.v_head + slot * p.c.v_tok + lc * 16;
        const uint32_t dst = ring + ld_stage * kStageBytes + ld_dst;
        const int have = page < 0 ? 0 : ld.t.len - key - lr;
        // Row 2 i + lr of the slice; its piece c lies at c ^ (row % 8).  With the tokens of a head side
        // by side every address is a constant away from the first.
        if (p.packed && page >= 0 && key + kSlice <= ld.t.len) {
#pragma unroll
          for (int i = 0; i < kSlice / 2; ++i) {
            const uint32_t d = (dst ^ ((2 * i & 7) << 4)) + 2 * i * (kHeadDim * 2);
            cp_async16(d, ks + i * (kHeadDim * 4), pol);
            cp_async16(d + kSliceBytes, vs + i * (kHeadDim * 4), pol);
          }
        } else {
          const char *ka[kSlice / 2], *va[kSlice / 2];
#pragma unroll
          for (int i = 0; i < kSlice / 2; ++i) {
            ka[i] = ks + i * 2 * p.c.k_tok;
            va[i] = vs + i * 2 * p.c.v_tok;
          }
#pragma unroll
          for (int i = 0; i < kSlice / 2; ++i) {
            const uint32_t d = (dst ^ ((2 * i & 7) << 4)) + 2 * i * (kHeadDim * 2);
            const uint32_t bytes = 2 * i < have ? 16u : 0u;
            cp_async16(d, ka[i], bytes, pol);
            cp_async16(d + kSliceBytes, va[i], bytes, pol);
          }
        }
      }
      if (++ld_stage == kStages) ld_stage = 0;
      advance(ld);
      if (valid(ld)) ld_page = page_at(ld);
    }
    cp_async_commit();
  };
  // First row of q of an item.
  auto q_row_of = [&](int b, int h) {
    const int head = h / p.row_tiles;
    return (static_cast<long long>(b) * p.c.Hkv + head) * p.rows + (h - head * p.row_tiles) * R;
  };
  auto load_q = [&](int b, int h, uint32_t(&f)[8][2]) {
    const bool live = g < p.rows - (h % p.row_tiles) * R;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q) + (q_row_of(b, h) + g) * (kHeadDim / 2) + t4;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      f[kk][0] = live ? __ldg(src + kk * 8) : 0u;
      f[kk][1] = live ? __ldg(src + kk * 8 + 4) : 0u;
    }
  };

  // Per-lane state: columns (rows of q) 2 t4 and + 1.  The next item's q is fetched while this one is
  // computed.
  uint32_t qf[8][2], qn[8][2];
  float o[8][4], m[2], l[2];
  RowKeys rk[2];
  int min_limit = 0, max_lo = 0;
  bool fresh = true;
  int seg_k0 = 0;
  int stage = 0;
  if (valid(cx)) load_q(cx.b, cx.h, qn);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load_next();
  // Every call leaves its counters zero, unless its lengths are rewritten while it runs; then a later call
  // must not begin with what it left.  The first CTA always gets here.
  if (cta == 0 && !p.all_partial)
    for (int i = threadIdx.x; i < kMaxSms * R; i += kThreads) p.others[i] = 0;
  if (lane == 0) sh.part[warp][0].item = sh.part[warp][1].item = -1;
  __syncwarp();

  for (; valid(cx); stage = stage + 1 == kStages ? 0 : stage + 1) {
    if (fresh) {
      fresh = false;
      seg_k0 = cx.k;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        qf[kk][0] = qn[kk][0];
        qf[kk][1] = qn[kk][1];
      }
      const bool roll = cx.h + 1 == per_seq;
      if (cx.at + units_of(cx.t.n, ln.align) < end) load_q(cx.b + roll, roll ? 0 : cx.h + 1, qn);
      if (p.c.Tq == 1) {
        const RowKeys k = row_keys(cx.t.r, p.rule, 0);
        min_limit = k.limit;
        max_lo = k.lo;
        rk[0] = rk[1] = k;
      } else {
        min_limit = 0x7fffffff;
        max_lo = 0;
        const int row0 = (cx.h % p.row_tiles) * R;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rr = row0 + 2 * t4 + e;
          rk[e] = row_keys(cx.t.r, p.rule, rr % p.c.Tq);
          if (rr >= p.rows) rk[e] = RowKeys{0x7fffffff, 0};
          min_limit = min(min_limit, rk[e].limit);
          max_lo = max(max_lo, rk[e].lo);
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          min_limit = min(min_limit, __shfl_xor_sync(0xffffffffu, min_limit, d));
          max_lo = max(max_lo, __shfl_xor_sync(0xffffffffu, max_lo, d));
        }
      }
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.0f;
#pragma unroll
      for (int a = 0; a < 8; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[a][e] = 0.0f;
    }

    cp_async_wait<kStages - 2>();
    __syncwarp();
    load_next();

    const int key0 = cx.key();
    if (key0 < cx.t.len) {
      const uint32_t kb = ring + stage * kStageBytes;
      // S^T: lanes 0-15 address keys 0-15 of the lower 8 columns, lanes 16-31 of the upper.
      float s[2][4];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] = 0.0f;
      {
        const int row = lane & 15, up = lane >> 4;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          uint32_t a[4];
          ldsm4(kb + row * (kHeadDim * 2) + (((2 * kk + up) ^ (row & 7)) << 4), a);
          mma16816<BF16>(s[kk & 1], a, qf[kk]);
        }
      }
      // Scores of lane (g, t4): keys key0 + g (e = 0, 1) and + 8 (e = 2, 3); columns 2 t4 + (e & 1).
      float x[4];
      bool over = false;
      const bool masked = key0 + kSlice > min_limit ||
                          (key0 < max_lo && key0 >= p.rule.glob * kTileKeys);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = (s[0][e] + s[1][e]) * p.scale_log2;
        if (masked) {
          const int key = key0 + g + (e >> 1) * 8;
          const RowKeys k = rk[e & 1];
          if (key >= k.limit || (key < k.lo && key >= p.rule.glob * kTileKeys)) x[e] = -INFINITY;
        }
        over |= x[e] > m[e & 1] + kRescaleLog2;
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(x[c], x[c + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m[c], mx);
          const float f = mn == -INFINITY ? 1.0f : ptx::ex2(m[c] - mn);
          m[c] = mn;
          l[c] *= f;
#pragma unroll
          for (int a = 0; a < 8; ++a) {
            o[a][c] *= f;
            o[a][c + 2] *= f;
          }
        }
      }
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mm = m[e & 1];
        pr[e] = ptx::ex2(x[e] - (mm == -INFINITY ? 0.0f : mm));
        l[e & 1] += pr[e];
      }
      const uint32_t pf[2] = {movm_trans(pack16<BF16>(pr[0], pr[1])), movm_trans(pack16<BF16>(pr[2], pr[3]))};
      // O^T: 16 columns of d per step; lanes 0-7 / 8-15 address keys 0-7 of the lower / upper
      // eight columns, lanes 16-31 keys 8-15.
      {
        const uint32_t vb = kb + kSliceBytes;
        const int row = (lane & 7) + ((lane >> 4) << 3), up = (lane >> 3) & 1;
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          uint32_t f[4];
          ldsm4_trans(vb + row * (kHeadDim * 2) + (((2 * a + up) ^ (row & 7)) << 4), f);
          mma16816<BF16>(o[a], f, pf);
        }
      }
    }

    const bool done = cx.k + 1 == cx.t.n;
    if (done || cx.at + cx.k + 1 >= end) {
      // The item, or this warp's part of it, ends.  Rows go through shared memory: this slice's stage,
      // which the next load_next refills only after this, or the room for a part that is kept.
      const bool began = seg_k0 == 0;
      const bool keep = !(done && began);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], d);
      // A part that goes on behind the share is the warp's last: every copy has landed by now, and it
      // lies in the ring (stage 0); one that began before it has room of its own.
      const int at_end = began ? 1 : 0;
      float* rows = keep && !began ? &sh.rest_o[warp][0][0]
                                   : reinterpret_cast<float*>(
                                         sh.ring[warp][keep ? 0 : stage]);
      if (keep && began) cp_async_wait<0>();
      __syncwarp();
      float inv[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) inv[c] = keep ? 1.0f : l[c] > 0.0f ? 1.0f / l[c] : 0.0f;
#pragma unroll
      for (int a = 0; a < 8; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 2 * t4 + (e & 1), d = a * 16 + g + (e >> 1) * 8;
          rows[r * kHeadDim + piece(r, d >> 2) * 4 + (d & 3)] = o[a][e] * inv[e & 1];
        }
      const int item = cx.b * per_seq + cx.h;
      if (keep) {
        Part& pt = sh.part[warp][at_end];
        if (g == 0)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            pt.m[2 * t4 + c] = m[c];
            pt.l[2 * t4 + c] = l[c];
          }
        if (lane == 0) {
          pt.item = item;
          pt.first = cx.at / ln.quota;
          pt.last = last_cta(ln, cx.at, units_of(cx.t.n, ln.align));
          pt.live = min(p.rows - (cx.h % p.row_tiles) * R, R);
          pt.q_row = q_row_of(cx.b, cx.h);
        }
      } else {
        __syncwarp();
        const long long q_row = q_row_of(cx.b, cx.h);
        const int live = min(p.rows - (cx.h % p.row_tiles) * R, R);
        const long long slot = part_slot(1, item, cta, true) * R;
        if (g == 0)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int r = 2 * t4 + c;
            const float lg = l[c] > 0.0f ? m[c] + log2f(l[c]) : -INFINITY;
            if (r < live) {
              if (p.all_partial) p.part_l[slot + r] = lg;
              else if (p.lse != nullptr) p.lse[q_row + r] = lg * 0.69314718055994531f;
            }
          }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r >= live) continue;
          const float4 v = reinterpret_cast<const float4*>(rows)[r * (kHeadDim / 4) + piece(r, lane)];
          if (p.all_partial)
            reinterpret_cast<float4*>(p.part_o)[(slot + r) * (kHeadDim / 4) + lane] = v;
          else
            store_row(p.o, nullptr, p.out_bf16, q_row + r, v, 0.0f, lane);
        }
        __syncwarp();
      }
      fresh = true;
    }
    advance(cx);
  }
  cp_async_wait<0>();
  __syncthreads();

  // The warps' parts in the order of the line, one per lane; runs of one item are added up, a row per
  // warp.  An item that lies across CTAs is left for whoever completes it.
  struct Split {
    int first, last, live;
    long long q_row;
  };
  Split split[2] = {{0, -1, 0, 0}, {0, -1, 0, 0}};
  int turn = 0;  // spreads the rows of the runs over the warps
  const int my_item = lane < 2 * W ? sh.part[lane >> 1][lane & 1].item : -1;
  const uint32_t there = __ballot_sync(0xffffffffu, my_item >= 0);
  const uint32_t below = there & ((1u << lane) - 1u);
  const int prev_item = __shfl_sync(0xffffffffu, my_item, below ? 31 - __clz(below) : 0);
  uint32_t starts = __ballot_sync(0xffffffffu, my_item >= 0 && (below == 0 || prev_item != my_item));
  while (starts != 0) {
    const int e = __ffs(starts) - 1;
    starts &= starts - 1;
    const uint32_t run = there & ~((1u << e) - 1u) & (starts ? (starts & (0u - starts)) - 1u : 0xffffffffu);
    const Part& a = sh.part[e >> 1][e & 1];
    const int first = a.first, last = a.last, live = a.live;
    const bool split_here = first != last;
    const long long q_row = a.q_row;
    const long long slot = part_slot(p.all_partial, a.item, cta, first == cta) * R;
    int r = warp;  // a split item's row r is always warp r's, which counts its parts below
    if (!split_here) {
      r = (warp - turn) & (W - 1);
      turn += live;
    }
    if (r < live) {
      const bool in = (run >> lane) & 1u;
      const float m_e = in ? sh.part[lane >> 1][lane & 1].m[r] : -INFINITY;
      float mx = m_e;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float f = m_e == -INFINITY ? 0.0f : ptx::ex2(m_e - mx);
      float sum = in ? sh.part[lane >> 1][lane & 1].l[r] * f : 0.0f;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      PartSum s;
      s.clear();
#pragma unroll
      for (int w = 0; w < W; ++w) {  // a warp has at most one part of an item
        const uint32_t which = (run >> (2 * w)) & 3u;
        const float fx = __shfl_sync(0xffffffffu, f, 2 * w + (which >> 1));
        if (which == 0) continue;
        const float* rows = which > 1 ? reinterpret_cast<const float*>(sh.ring[w][0]) : &sh.rest_o[w][0][0];
        s.add(reinterpret_cast<const float4*>(rows)[r * (kHeadDim / 4) + piece(r, lane)], fx);
      }
      s.sum = sum;
      const float4 v = s.normal();
      const float lg = s.log2_total(mx);
      if (!split_here && !p.all_partial) {
        store_row(p.o, p.lse, p.out_bf16, q_row + r, v, lg, lane);
      } else {
        reinterpret_cast<float4*>(p.part_o)[(slot + r) * (kHeadDim / 4) + lane] = v;
        if (lane == 0) p.part_l[slot + r] = lg;
      }
    }
    if (split_here) {
      const Split x{first, last, live, q_row};
      if (first == cta) split[1] = x;
      else split[0] = x;
    }
  }
  if (!p.all_partial && (split[0].last >= 0 || split[1].last >= 0)) {
    // Row r of either item is warp r's.  Asked for once, at the CTA's end: the fence and the counters
    // cost a round trip to L2 each.
    static_assert(R == W, "a row for every warp");
    int done[2] = {-1, -1};
    __threadfence();
    __syncwarp();
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (lane == 0 && split[s].last >= 0 && warp < split[s].live)
        done[s] = atomicAdd(p.counters + split[s].first * R + warp, 1);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int n = __shfl_sync(0xffffffffu, done[s], 0);
      if (n < 0 || n != split[s].last - split[s].first) continue;
      __threadfence();
      if (lane == 0) p.counters[split[s].first * R + warp] = 0;
      join_row(p, split[s].q_row + warp, warp, R, split[s].first, split[s].last, lane);
    }
  }
  if (p.all_partial && blockIdx.x + 1 == gridDim.x) pdl_wait();
}

}  // namespace few

int few_setup() {
  using namespace few;
  const void* kernels[] = {reinterpret_cast<const void*>(few_kernel<false>),
                           reinterpret_cast<const void*>(few_kernel<true>)};
  for (const void* k : kernels)
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(Smem))) != cudaSuccess)
      return BSATTN_E_CUDA;
  return BSATTN_OK;
}

int few_launch(const FewCall& c, cudaStream_t stream) {
  using namespace few;
  // The tokens of a page and head lie side by side.
  const int packed = c.c.k_tok == kHeadDim * 2 && c.c.v_tok == kHeadDim * 2;
  // The calls of a buffer take its two halves by turns, and clear the one that they do not use.  Buffers
  // that share a place here only take their turns in another order.
  static std::atomic<uint8_t> turns[1024];
  constexpr int kHalf = kMaxSms * kFewRows;
  const uint64_t place = (reinterpret_cast<uintptr_t>(c.counters) >> 4) * 0x9E3779B97F4A7C15ull >> 54;
  const int turn = turns[place].fetch_add(1, std::memory_order_relaxed) & 1;
  const Params p{c.c,        c.rule,        c.q,    c.o,   c.lse,    c.rows,   c.row_tiles, c.scale_log2,
                 c.out_bf16, c.all_partial, packed, c.cum, c.part_o, c.part_l,
                 c.counters + turn * kHalf, c.counters + (1 - turn) * kHalf};
  return launch(c.in_bf16 ? few_kernel<true> : few_kernel<false>, dim3(static_cast<unsigned>(c.ctas)),
                kThreads, sizeof(Smem), stream, p);
}

}  // namespace paged
}  // namespace bsattn

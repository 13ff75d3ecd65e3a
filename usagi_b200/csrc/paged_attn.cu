// paged_attn.cu -- attention over a paged K/V cache: the calls, which kernels they take, and the joins
// of partial results.
//
// Rows of q that share a K/V head (G = Hq / Hkv query heads, Tq tokens) go together:
//   * up to 8 rows, and more in small calls: the few-row kernel (paged_few.cu), which is bound by memory;
//   * else the many-row kernel (paged_tile.cu), tiles of 128 rows on the tensor cores;
//   * behind a shared prefix: the prefix's keys by the many-row kernel, over the stacked rows of the
//     whole batch, the sequences' own keys by the few-row kernel beside it, and a join of both.
#include <algorithm>
#include <mutex>

#include "paged_few.cuh"
#include "paged_tile.cuh"
#include "sm100_ptx.cuh"

namespace bsattn {
namespace paged {

// Joins behind a shared prefix: every row of the call, over the parts of the prefix in the order of its
// line, then over those of its own keys: o = sum_i o_i 2^(l_i - l), l = log2 sum 2^l_i.
struct RowJoin {
  int Hkv, rows, groups; // rows = G * Tq; groups = B * Hkv
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

// Four rows of partial results in a warp: lane l has row l % 4 and the 16-byte pieces l / 4 + 8 i.
struct Quad {
  float4 acc[4];
  float sum, mx;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    sum = 0.0f;
    mx = -INFINITY;
  }
  // Parts in their order: their pieces and log2 sums.
  template <int N>
  __device__ __forceinline__ void add(const float4 (&y)[N][4], const float (&lg)[N]) {
    float top = mx;
#pragma unroll
    for (int c = 0; c < N; ++c) top = fmaxf(top, lg[c]);
    if (top == -INFINITY) return;
    scale(ptx::ex2(mx - top));
    mx = top;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const float w = ptx::ex2(lg[c] - top);
      sum += w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[i].x += y[c][i].x * w;
        acc[i].y += y[c][i].y * w;
        acc[i].z += y[c][i].z * w;
        acc[i].w += y[c][i].w * w;
      }
    }
  }
  __device__ __forceinline__ void scale(float f) {
    sum *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc[i] = make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f);
  }
  // Every W-th part from `from` on, of `n`: part c's log2 sum at l[c * l_step], the lane's first piece
  // of it at o[c * o_step], the others `step` apart.  Four at once, so that their loads overlap.
  __device__ __forceinline__ void add_all(const float* l, long long l_step, const float4* o,
                                          long long o_step, int step, int from, int n, int W) {
    for (int c0 = from; c0 < n; c0 += 4 * W) {
      float4 y[4][4];
      float lg[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const long long x = c0 + c * W;
        lg[c] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[c][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (x < n) {
          lg[c] = __ldcg(l + x * l_step);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[c][i] = __ldcg(o + x * o_step + i * step);
        }
      }
      add(y, lg);
    }
  }
  __device__ __forceinline__ void store(void* o, float* lse, int out_bf16, long long row, int piece) const {
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint2*>(o)[row * (kHeadDim / 4) + piece + 8 * i] =
          make_uint2(pack_out(acc[i].x * inv, acc[i].y * inv, out_bf16),
                     pack_out(acc[i].z * inv, acc[i].w * inv, out_bf16));
    if (lse != nullptr && piece == 0)
      lse[row] = sum > 0.0f ? (mx + log2f(sum)) * 0.69314718055994531f : -INFINITY;
  }
};

// The rows of a (sequence, K/V head) go four by four; W warps share a quad when it has many parts.
template <int W>
__global__ void __launch_bounds__(kJoinWarps * 32) join_rows_kernel(const __grid_constant__ RowJoin p) {
  __shared__ float4 so[W > 1 ? kJoinWarps : 1][4][32];
  __shared__ float sl[kJoinWarps][4], sm[kJoinWarps][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quads = (p.rows + 3) >> 2;
  const long long quad = W == 1 ? static_cast<long long>(blockIdx.x) * kJoinWarps + warp : blockIdx.x;
  if (quad >= static_cast<long long>(p.groups) * quads) return;
  const int bh = static_cast<int>(quad / quads);
  const int rr = static_cast<int>(quad - static_cast<long long>(bh) * quads) * 4 + (lane & 3);
  const int piece = lane >> 2;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int hr = h * p.row_tiles + rr / p.R, r = rr % p.R;
  const int heads = p.Hkv * p.row_tiles;
  const long long item_p = static_cast<long long>(b / p.n_b) * p.Hkv + h;
  const int rp = (b % p.n_b) * p.rows + rr;
  const long long sp = item_p * p.tiles_p;
  const int first_p = static_cast<int>(sp / p.quota_p);
  const int pre = static_cast<int>((sp + p.tiles_p - 1) / p.quota_p) - first_p + 1;
  pdl_wait();
  pdl_trigger();
  // The prefix's parts first: where the own ones lie has to be read.
  const int c0 = p.cum[b], n = p.cum[b + 1] - c0;
  const Line ln{p.cum[p.B + 1], p.cum[p.B + 2]};
  const bool live = rr < p.rows;
  const int from = W == 1 ? 0 : warp;
  Quad x;
  x.clear();
  if (live) {
    const long long at_p = item_p + first_p;
    x.add_all(p.pre_l + at_p * 128 + rp, 128,
              reinterpret_cast<const float4*>(p.pre_o) + (at_p * (kHeadDim / 4) + piece) * 128 + rp,
              128 * (kHeadDim / 4), 8 * 128, from, pre, W);
    const int s = c0 * heads + hr * n;
    const int first = s / ln.quota, own = last_cta(ln, s, n) - first + 1;
    const long long at = (static_cast<long long>(b) * heads + hr + first) * p.R + r;
    x.add_all(p.part_l + at, p.R, reinterpret_cast<const float4*>(p.part_o) + at * (kHeadDim / 4) + piece,
              static_cast<long long>(p.R) * (kHeadDim / 4), 8, from, own, W);
  }
  if (W > 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) so[W > 1 ? warp : 0][i][lane] = x.acc[i];
    if (piece == 0) {
      sl[warp][lane & 3] = x.sum;
      sm[warp][lane & 3] = x.mx;
    }
    __syncthreads();
    if (warp != 0) return;
    float top = x.mx;
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, sm[w][lane & 3]);
    x.scale(top > -INFINITY ? ptx::ex2(x.mx - top) : 0.0f);
    x.mx = top;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float f = sm[w][lane & 3] > -INFINITY ? ptx::ex2(sm[w][lane & 3] - top) : 0.0f;
      x.sum += sl[w][lane & 3] * f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 y = so[W > 1 ? w : 0][i][lane];
        x.acc[i].x += y.x * f;
        x.acc[i].y += y.y * f;
        x.acc[i].z += y.z * f;
        x.acc[i].w += y.w * f;
      }
    }
  }
  if (live)
    x.store(p.o, p.lse, p.out_bf16, static_cast<long long>(bh) * p.rows + rr, piece);
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
  const int r = (blockIdx.y * kJoinWarps + warp) * 4 + (lane & 3), piece = lane >> 2;
  const int first = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  // The piece that begins the item lies in slot 2 first + 1, the others in 2 (first + 1), + 2, ...: the first
  // two are asked for before it is known whether there is an item.
  constexpr int kSlot = 128 * (kHeadDim / 4);
  const float* l = p.part_l + (2ll * first + 1) * 128 + r;
  const float4* o = reinterpret_cast<const float4*>(p.part_o) + (2ll * first + 1) * kSlot + piece * 128 + r;
  float4 y[2][4];
  float lg[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const bool there = first + c < static_cast<int>(gridDim.x);
    lg[c] = there ? __ldcg(l + c * 128) : -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      y[c][i] = there ? __ldcg(o + c * kSlot + i * (8 * 128)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  const TileCut cut = p.cuts[first];
  if (cut.v < 0) return;
  const int b = cut.v / p.rt.per_seq;
  const int g = r / p.rt.n_t, t = (cut.v - b * p.rt.per_seq) * p.rt.n_t + r - g * p.rt.n_t;
  if (g >= p.rt.G || t >= p.Tq) return;
  Quad x;
  x.clear();
  x.add(y, lg);
  x.add_all(l + 3 * 128, 256, o + 3 * kSlot, 2 * kSlot, 8 * 128, 0, cut.pieces - 2, 1);
  x.store(p.o, p.lse, p.out_bf16, ((static_cast<long long>(b) * p.Hkv + cut.h) * p.rt.G + g) * p.Tq + t, piece);
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
    int rc2 = few_setup();
    if (rc2 == BSATTN_OK) rc2 = tile_setup();
    if (rc2 != BSATTN_OK) return rc2;
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

// More than 8 rows go to the few-row kernel as well, eight at a time over the same keys, when every such
// item has a CTA of its own, there are no more than kSmallTiles for a K/V head, and a cache as large as the
// page table allows is read in no more than kSmallBytes: it starts 3 us sooner and needs no join kernel.
// Few-row and many-row kernel within that: 32 query heads on 8, 8 tokens, 1,000 keys (16 MB) 12.9 and 14.3
// us; 64 on 8, 3 tokens, 4 sequences of 512 keys (24 MB) 12.1 and 16.0; 64 on 4, 8,192 keys (32 MB) 16.3 and
// 22.3.  Outside: 32 on 8, 5 tokens, 4 sequences of 1,000 keys (48 MB) 18.1 and 17.4; 32 on 2, 16 tokens, 600
// keys (32 for a head) 13.5 and 12.9; 32 on 8, 64 tokens, 200 keys (256 items) 16.6 and 13.3.
// At 8 rows (64 on 8) the few-row kernel is ahead at any size: 8,192 keys 16.9 and 22.1, 32 sequences of
// 4,096 keys 96.5 and 97.4.
constexpr int kSmallTiles = 16;
constexpr long long kSmallBytes = 32ll << 20;
// More rows of one sequence fill a tile without its neighbours.  At 64 rows (32 sequences of 16 tokens, 32
// heads on 8, behind 8,192 tokens) stacked 97 us, one sequence after the other 154.
constexpr int kStackedRows = 64;
// A prefix is read once when that saves at least this much reading; below, three launches and a join
// cost more than the bytes, which L2 serves.  Measured, one pass over everything against prefix once,
// 32 query heads on 8: 8 sequences behind 4,096 tokens (117 MB saved) 24.5 and 23.4 us, 16 behind 4,096
// (252 MB) 36.4 and 26.2, 64 behind 1,024 (264 MB) 38.4 and 26.3, 16 behind 1,024 (63 MB) 15.8 and 19.5.
constexpr long long kSharedBytes = 128ll << 20;

static int shape_of(int B, int Hq, int Hkv, int Tq, int max_pages, int page_size, int prefix_len,
                    int sms, Shape* s) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 || Tq < 1) return BSATTN_E_SHAPE;
  const int G = Hq / Hkv;
  const long long rows = static_cast<long long>(G) * Tq;
  if (rows * B * Hkv > (1ll << 31) - 1) return BSATTN_E_SHAPE;
  s->rows = static_cast<int>(rows);
  const long long saved = static_cast<long long>(B - 1) * prefix_len * Hkv * (4 * kHeadDim);
  s->prefix = prefix_len > 0 && rows <= kStackedRows && saved >= kSharedBytes;
  const long long row_tiles = (rows + kFewRows - 1) / kFewRows;
  const bool small = row_tiles <= kSmallTiles && row_tiles * B * Hkv <= sms &&
                     row_tiles * B * Hkv * max_pages * page_size * (4 * kHeadDim) <= kSmallBytes;
  s->few = s->prefix || rows <= kFewRows || small || G > 128;
  s->k0 = s->prefix ? prefix_len : 0;
  s->all_partial = s->prefix;
  // Most tiles one item can have.
  const int step = s->few ? kSlice : kTileKeys;
  const long long tiles = (static_cast<long long>(max_pages) * page_size + step - 1) / step + 1;
  long long items;
  if (s->few) {
    s->R = kFewRows;
    s->row_tiles = static_cast<int>(row_tiles);
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
  if (items * (tiles + 64) > (1ll << 30)) return BSATTN_E_SHAPE;
  s->pieces = static_cast<int>(std::min<long long>(sms, items * tiles));
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

  TileCall t;
  if (s.prefix || !s.few) {
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
  }
  FewCall f;
  if (s.few) {
    f.c = cache;
    f.rule = rule;
    f.q = q;
    f.o = o;
    f.lse = lse;
    f.rows = s.rows;
    f.row_tiles = s.row_tiles;
    f.scale_log2 = scale_log2;
    f.in_bf16 = bf16;
    f.out_bf16 = out_bf16;
    f.all_partial = s.all_partial;
    f.ctas = s.pieces;
    f.cum = reinterpret_cast<int*>(base + s.cum);
    f.part_o = reinterpret_cast<float*>(base + s.part_o);
    f.part_l = reinterpret_cast<float*>(base + s.part_l);
    f.counters = counters;
  }
  // Behind a prefix the few-row kernel takes the SMs as the other leaves them: it does not wait for it
  // to begin with (its inputs are there, the other has waited for them), but its last CTA holds it
  // open until the other has ended, so that the join may wait for it alone.  (Running both from the
  // start, half of each one's CTAs at a time, was measured: 118 us against 108 for 256 sequences behind
  // 8,192 tokens.)
  if ((s.prefix || !s.few) && (rc = tile_launch(t, page_size, stream)) != BSATTN_OK) return rc;
  if (s.few && (rc = few_launch(f, stream)) != BSATTN_OK) return rc;
  if (s.prefix) {
    RowJoin j;
    j.Hkv = cache.Hkv;
    j.rows = s.rows;
    j.groups = cache.B * cache.Hkv;
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
    // Rows of many parts are shared by four warps (18 parts: 70 us for the call against 78; 5 parts: 110
    // against 105).
    const unsigned quads = static_cast<unsigned>(j.groups) * static_cast<unsigned>((s.rows + 3) / 4);
    return s.pieces_p / items_p >= 8
               ? launch(join_rows_kernel<kJoinWarps>, dim3(quads), kJoinWarps * 32, 0, stream, j)
               : launch(join_rows_kernel<1>, dim3((quads + kJoinWarps - 1) / kJoinWarps),
                        kJoinWarps * 32, 0, stream, j);
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
    return launch(join_cuts_kernel, dim3(static_cast<unsigned>(s.pieces), groups), kJoinWarps * 32, 0,
                  stream, j);
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

int bsattn_paged_counters(void) { return 2 * kMaxSms * kFewRows; }

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
  // More global blocks than the table holds are the same as all of them, whose keys 32 bits can count.
  const long long cap = static_cast<long long>(call->max_pages) * call->page_size;
  const int blocks = static_cast<int>((cap + kTileKeys - 1) / kTileKeys);
  const Rule rule{0, window, std::min(global_blocks, blocks)};
  return launch_paged(q, c, rule, prefix_len, call->Hq, scale, call->dtype_flags, call->page_size, o,
                      lse, scratch, scratch_bytes, counters, static_cast<cudaStream_t>(call->stream));
}

}  // extern "C"

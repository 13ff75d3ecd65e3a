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
//   * Work: an item is (sequence, K/V head, tile of rows), a tile is 128 keys.  The tiles of all
//     items form one line that is cut into equal pieces, one per CTA, so a long sequence is split
//     over many CTAs and a short one shares a CTA with others.  The lengths are on the device:
//     each CTA adds them up itself, in a few microseconds at most, and no host copy is needed.
//   * A CTA is eight warps on their own: warp w owns keys 16w .. 16w+15 of every tile, loads them
//     with cp.async into a private ring (16-byte pieces swizzled so that ldmatrix reads without
//     bank conflicts) and keeps its own running maximum, sum and output.  No barrier is met until
//     a piece of an item ends; the ring runs across item borders.
//   * Keys are the M dimension of the warp MMAs (m16n8k16): S^T = K Q^T and O^T = V^T P^T, so eight
//     rows fill an MMA's N and none of it is spent on padding; P^T moves from the accumulator to
//     the operand layout with movmatrix, in registers.
//   * The running maximum moves only when a score passes it by more than 2^8 (then P stays within
//     2^8, far inside fp16 and bf16); the usual step costs one vote instead of a reduction.
//   * At the end of a piece the eight warps' outputs are merged through shared memory in warp
//     order.  A piece that is a whole item writes o and lse; others leave (o, log2 sum) in 32 bits
//     for the join kernel, which adds them in the order of the line: results do not depend on
//     timing.
// Keys past a sequence's end are loaded as zeros, never read: a recycled page may hold anything.
// P is rounded to the type of V, as the tensor cores take it; its sum is of the unrounded values.
#include <algorithm>
#include <mutex>

#include "paged_common.cuh"
#include "paged_tile.cuh"
#include "sm100_ptx.cuh"

namespace bsattn {
namespace paged {

constexpr int kWarps = 8;
constexpr int kThreadsD = kWarps * 32;
constexpr int kStages = 3;
constexpr int kSlice = 16;                        // keys of a tile per warp
constexpr int kSliceBytes = kSlice * kHeadDim * 2;  // 4 KB of K or of V
constexpr int kOPitch = kHeadDim + 4;             // floats between rows of the merge buffer
constexpr float kRescaleLog2 = 8.0f;
static_assert(kWarps * kSlice == kTileKeys, "a tile is one slice per warp");

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
  // Scratch: prefix sums of the tiles per sequence [B + 1], partial outputs and their log2 sums.
  int* cum;
  float* part_o;
  float* part_l;
};

template <int NB>
struct DecodeSmem {
  uint8_t ring[kWarps][kStages][2][kSliceBytes];
  float o[kWarps][8][kOPitch];
  float m[kWarps][8 * NB], l[kWarps][8 * NB];
  int warp_sum[kWarps];
  int found[3];
};

// Where a piece of item `item` that CTA `cta` holds leaves its partial output.  A CTA holds at most
// one piece that begins its item and one other; when whole items are partial too, item + cta
// numbers all pieces, since along the line one of the two always grows.
__device__ __forceinline__ long long part_slot(int all_partial, long long item, int cta, bool head) {
  return all_partial ? item + cta : 2ll * cta + (head ? 1 : 0);
}

// A position on the line of tiles.
struct Cursor {
  int b, h, tile;  // h counts (K/V head, row tile)
  Tiles t;
};

template <bool BF16, int NB>
__global__ void __launch_bounds__(kThreadsD, 1) decode_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  DecodeSmem<NB>& sh = *reinterpret_cast<DecodeSmem<NB>*>(smem_raw);
  constexpr int R = 8 * NB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int per_seq = p.c.Hkv * p.row_tiles;
  pdl_trigger();

  // Where this CTA's piece of the line starts.
  const int chunk = (p.c.B + kThreadsD - 1) / kThreadsD;
  const int b0 = min(static_cast<int>(threadIdx.x) * chunk, p.c.B);
  const int b1 = min(b0 + chunk, p.c.B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles_of(p.c, p.rule, b).n;
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) sh.warp_sum[warp] = incl;
  __syncthreads();
  int total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh.warp_sum[w];
    total += sh.warp_sum[w];
  }
  const int line = total * per_seq;
  const int quota = (line + gridDim.x - 1) / gridDim.x;
  const int begin = min(static_cast<int>(blockIdx.x) * quota, line);
  const int end = min(begin + quota, line);
  for (int b = b0; b < b1; ++b) {
    const int n = tiles_of(p.c, p.rule, b).n;
    if (blockIdx.x == 0) p.cum[b] = before;
    const int rel = begin - before * per_seq;
    if (rel >= 0 && rel < n * per_seq) {
      sh.found[0] = b;
      sh.found[1] = rel / n;
      sh.found[2] = rel % n;
    }
    before += n;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.cum[p.c.B] = total;
  __syncthreads();
  if (begin >= end) {
    pdl_wait();
    return;
  }

  auto seek = [&](Cursor& x) {
    x.b = sh.found[0];
    x.h = sh.found[1];
    x.tile = sh.found[2];
    x.t = tiles_of(p.c, p.rule, x.b);
  };
  auto advance = [&](Cursor& x) {
    if (++x.tile < x.t.n) return;
    x.tile = 0;
    if (++x.h < per_seq) return;
    x.h = 0;
    if (++x.b < p.c.B) x.t = tiles_of(p.c, p.rule, x.b);
  };
  // First key of this warp's slice.
  auto slice_key = [&](const Cursor& x) { return tile_key(x.t, p.rule, x.tile) + warp * kSlice; };
  auto page_at = [&](const Cursor& x) {
    const int key = slice_key(x);
    return key < x.t.len ? __ldg(p.c.table + x.b * p.c.table_stride + (key >> p.c.page_shift)) : 0;
  };

  // Loads.  Lane l moves piece l % 16 of rows l / 16, l / 16 + 2, ...; the page of the next slice
  // is asked for one step ahead.
  const int n_tiles = end - begin;
  Cursor ld, cx;
  seek(ld);
  seek(cx);
  int ld_page = page_at(ld);
  const uint32_t ring = ptx::smem_u32(sh.ring[warp]);
  const int lr = lane >> 4, lc = lane & 15;
  int ld_i = 0;
  auto load_next = [&]() {
    if (ld_i < n_tiles) {
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
      if (ld_i < n_tiles) {
        advance(ld);
        ld_page = page_at(ld);
      }
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

  for (int i = 0; i < n_tiles; ++i) {
    const int row0 = (cx.h % p.row_tiles) * R;
    const int head = cx.h / p.row_tiles;
    const long long q_row = (static_cast<long long>(cx.b) * p.c.Hkv + head) * p.rows + row0;
    if (fresh) {
      fresh = false;
      seg_tile0 = cx.tile;
      min_limit = 0x7fffffff;
      max_lo = 0;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int r = row0 + nb * 8 + g;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q) + (q_row + nb * 8 + g) * (kHeadDim / 2);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qf[nb][kk][0] = r < p.rows ? __ldg(src + kk * 8 + t4) : 0u;
          qf[nb][kk][1] = r < p.rows ? __ldg(src + kk * 8 + t4 + 4) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rr = row0 + nb * 8 + 2 * t4 + e;
          rk[nb][e] = row_keys(cx.t, p.rule, rr % p.c.Tq);
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

    if (cx.tile + 1 == cx.t.n || i + 1 == n_tiles) {
      // The piece ends: join the warps.
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], d);
          if (g == 0) {
            sh.m[warp][nb * 8 + 2 * t4 + c] = m[nb][c];
            sh.l[warp][nb * 8 + 2 * t4 + c] = l[nb][c];
          }
        }
      const bool whole = !p.all_partial && seg_tile0 == 0 && cx.tile + 1 == cx.t.n;
      const long long slot = part_slot(p.all_partial, static_cast<long long>(cx.b) * per_seq + cx.h,
                                       static_cast<int>(blockIdx.x), seg_tile0 == 0);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        __syncthreads();
        // This thread writes row `warp` of the eight; every lane scales two columns.
        float mx = -INFINITY, sum = 0.0f, f[2];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sh.m[w][nb * 8 + warp]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float mw = sh.m[w][nb * 8 + warp];
          sum += mw == -INFINITY ? 0.0f : sh.l[w][nb * 8 + warp] * ptx::ex2(mw - mx);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mc = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) mc = fmaxf(mc, sh.m[w][nb * 8 + 2 * t4 + c]);
          f[c] = m[nb][c] == -INFINITY ? 0.0f : ptx::ex2(m[nb][c] - mc);
        }
#pragma unroll
        for (int a = 0; a < 8; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sh.o[warp][2 * t4 + (e & 1)][a * 16 + g + (e >> 1) * 8] = o[nb][a][e] * f[e & 1];
        __syncthreads();
        const int r = nb * 8 + warp;
        if (row0 + r < p.rows) {
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(&sh.o[w][warp][lane * 4]);
            acc.x += y.x;
            acc.y += y.y;
            acc.z += y.z;
            acc.w += y.w;
          }
          const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
          const float lg = sum > 0.0f ? mx + log2f(sum) : -INFINITY;
          acc.x *= inv;
          acc.y *= inv;
          acc.z *= inv;
          acc.w *= inv;
          if (whole) {
            uint2 w2 = make_uint2(pack_out(acc.x, acc.y, p.out_bf16), pack_out(acc.z, acc.w, p.out_bf16));
            reinterpret_cast<uint2*>(p.o)[(q_row + r) * (kHeadDim / 4) + lane] = w2;
            if (p.lse != nullptr && lane == 0) p.lse[q_row + r] = lg * 0.69314718055994531f;
          } else {
            reinterpret_cast<float4*>(p.part_o)[(slot * R + r) * (kHeadDim / 4) + lane] = acc;
            if (lane == 0) p.part_l[slot * R + r] = lg;
          }
        }
      }
      fresh = true;
    }
    if (i + 1 < n_tiles) advance(cx);
  }
  cp_async_wait<0>();
  // Behind a shared prefix this kernel starts while the prefix's still runs, and must not end
  // before it: the join waits for this kernel only.
  pdl_wait();
}

// Joins the pieces of a row: o = sum_i o_i 2^(l_i - l), l = log2 sum 2^l_i, over the pieces of its
// item in the order of the line, then over those of the shared prefix.  A row whose item is one
// piece is written already.  One block per row; its four warps take every fourth piece and meet in
// shared memory.
constexpr int kJoinWarps = 4;
struct JoinParams {
  int Hkv, G, Tq;
  void* o;
  float* lse;
  int out_bf16;
  // Own keys: virtual sequence = b * v_per_seq + t / v_tok, item = it * heads + head tile, where a
  // K/V head's rows are in tiles of R (few-row kernel) or already one tile (n_t tokens each).
  const int* cum;
  const float* part_o;
  const float* part_l;
  int count, pieces, R, row_tiles, all_partial;
  int n_t, per_seq;  // many-row kernel: tokens per tile of rows; 0: few-row kernel
  // Prefix: n_b sequences per tile of rows, each item tiles_p tiles, pieces_p CTAs.
  const float* pre_o;
  const float* pre_l;
  int n_b, tiles_p, quota_p;
};
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ JoinParams p) {
  __shared__ float4 so[kJoinWarps][32];
  __shared__ float sl[kJoinWarps], sm[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x % p.Tq;
  const int bh = blockIdx.x / p.Tq;
  const int Hq = p.Hkv * p.G;
  const int b = bh / Hq, hq = bh - b * Hq;
  const int h = hq / p.G, g = hq - h * p.G;
  int v, hr, r;
  if (p.n_t > 0) {
    v = b * p.per_seq + t / p.n_t;
    hr = h;
    r = g * p.n_t + t % p.n_t;
  } else {
    const int row = g * p.Tq + t;
    v = b;
    hr = h * p.row_tiles + row / p.R;
    r = row % p.R;
  }
  const int heads = p.Hkv * p.row_tiles;
  pdl_wait();
  const int c0 = p.cum[v], n = p.cum[v + 1] - c0;
  const int line = p.cum[p.count] * heads;
  const int quota = (line + p.pieces - 1) / p.pieces;
  const int s = c0 * heads + hr * n;
  const int first = s / quota, last = (s + n - 1) / quota;
  if (first == last && !p.all_partial) return;
  const long long item = static_cast<long long>(v) * heads + hr;
  int first_p = 0, pre = 0;  // pieces of the prefix
  long long item_p = 0;
  int rp = 0;
  if (p.tiles_p > 0) {
    item_p = static_cast<long long>(b / p.n_b) * p.Hkv + h;
    rp = ((b % p.n_b) * p.G + g) * p.Tq + t;
    const long long sp = item_p * p.tiles_p;
    first_p = static_cast<int>(sp / p.quota_p);
    pre = static_cast<int>((sp + p.tiles_p - 1) / p.quota_p) - first_p + 1;
  }
  const int own = last - first + 1;
  float mx = -INFINITY, sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = warp; i < own + pre; i += kJoinWarps) {
    const float *po, *pl;
    if (i < own) {
      const long long row = part_slot(p.all_partial, item, first + i, i == 0) * p.R + r;
      po = p.part_o + row * kHeadDim;
      pl = p.part_l + row;
    } else {
      const long long row = (item_p + first_p + i - own) * 128 + rp;
      po = p.pre_o + row * kHeadDim;
      pl = p.pre_l + row;
    }
    const float lg = *pl;
    const float4 y = reinterpret_cast<const float4*>(po)[lane];
    if (lg == -INFINITY) continue;
    const float mn = fmaxf(mx, lg);
    const float fa = ptx::ex2(mx - mn), fb = ptx::ex2(lg - mn);
    acc.x = acc.x * fa + y.x * fb;
    acc.y = acc.y * fa + y.y * fb;
    acc.z = acc.z * fa + y.z * fb;
    acc.w = acc.w * fa + y.w * fb;
    sum = sum * fa + fb;
    mx = mn;
  }
  so[warp][lane] = acc;
  if (lane == 0) {
    sl[warp] = sum;
    sm[warp] = mx;
  }
  __syncthreads();
  if (warp != 0) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, sm[w]);
  float total = 0.0f;
  float4 out = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    if (sm[w] == -INFINITY) continue;
    const float f = ptx::ex2(sm[w] - top);
    const float4 y = so[w][lane];
    total += sl[w] * f;
    out.x += y.x * f;
    out.y += y.y * f;
    out.z += y.z * f;
    out.w += y.w * f;
  }
  const float inv = total > 0.0f ? 1.0f / total : 0.0f;
  const long long row = blockIdx.x;
  reinterpret_cast<uint2*>(p.o)[row * (kHeadDim / 4) + lane] =
      make_uint2(pack_out(out.x * inv, out.y * inv, p.out_bf16), pack_out(out.z * inv, out.w * inv, p.out_bf16));
  if (p.lse != nullptr && lane == 0)
    p.lse[row] = total > 0.0f ? (top + log2f(total)) * 0.69314718055994531f : -INFINITY;
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
  size_t cum, part_o, part_l, cum_p, pre_o, pre_l, bytes;  // offsets into the scratch
};

constexpr int kFewRows = 16;     // rows of one tile of the few-row kernel
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
  const long long tiles = (static_cast<long long>(max_pages) * page_size + kTileKeys - 1) / kTileKeys + 1;
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
  if (items * tiles > (1ll << 30)) return BSATTN_E_SHAPE;
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
  s->cum = take(s->count + 1);
  s->part_o = take(s->slots * s->R * kHeadDim);
  s->part_l = take(s->slots * s->R);
  s->cum_p = take(s->prefix ? s->rt.count + 1 : 0);
  s->pre_o = take(s->slots_p * 128 * kHeadDim);
  s->pre_l = take(s->slots_p * 128);
  s->bytes = at;
  return BSATTN_OK;
}

// A launch that may start while its predecessor still runs.
template <class P>
static bool launch_overlapped(void (*kernel)(P), unsigned grid, int threads, size_t smem,
                              cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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
                        void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  if (!q || !o) return BSATTN_E_NULL;
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
    t.cum = reinterpret_cast<int*>(base + (s.prefix ? s.cum_p : s.cum));
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
  JoinParams j;
  j.Hkv = cache.Hkv;
  j.G = Hq / cache.Hkv;
  j.Tq = cache.Tq;
  j.o = o;
  j.lse = lse;
  j.out_bf16 = out_bf16;
  j.cum = reinterpret_cast<const int*>(base + s.cum);
  j.part_o = reinterpret_cast<const float*>(base + s.part_o);
  j.part_l = reinterpret_cast<const float*>(base + s.part_l);
  j.count = s.count;
  j.pieces = s.pieces;
  j.R = s.R;
  j.row_tiles = s.row_tiles;
  j.all_partial = s.all_partial;
  j.n_t = s.few ? 0 : s.rt.n_t;
  j.per_seq = s.few ? 1 : s.rt.per_seq;
  j.pre_o = reinterpret_cast<const float*>(base + s.pre_o);
  j.pre_l = reinterpret_cast<const float*>(base + s.pre_l);
  j.n_b = s.prefix ? s.rt.n_b : 1;
  j.tiles_p = s.tiles_p;
  j.quota_p = 1;
  if (s.prefix) {
    const long long line = static_cast<long long>(s.rt.count) * cache.Hkv * s.tiles_p;
    j.quota_p = static_cast<int>((line + s.pieces_p - 1) / s.pieces_p);
  }
  const unsigned rows = static_cast<unsigned>(static_cast<long long>(cache.B) * Hq * cache.Tq);
  if (!launch_overlapped(join_kernel, rows, kJoinWarps * 32, 0, stream, j)) return BSATTN_E_CUDA;
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

int bsattn_paged_fwd(const bsattn_paged_call* call, const void* q, void* o, float* lse, int window,
                     int global_blocks, int prefix_len, float scale, void* scratch,
                     size_t scratch_bytes) {
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
                      lse, scratch, scratch_bytes, static_cast<cudaStream_t>(call->stream));
}

}  // extern "C"

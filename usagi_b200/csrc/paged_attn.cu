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
  int G, rows, row_tiles;  // rows = G * Tq; row_tiles = ceil(rows / R)
  float scale_log2;
  int out_bf16;
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
  if (begin >= end) return;

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
      const bool whole = seg_tile0 == 0 && cx.tile + 1 == cx.t.n;
      const long long slot = (static_cast<long long>(cx.b) * per_seq + cx.h) + blockIdx.x;
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
}

// Joins the pieces of the items that were split: o = sum_i o_i 2^(l_i - l), l = log2 sum 2^l_i.
// One block per row; its four warps take every fourth piece and meet in shared memory.
constexpr int kJoinWarps = 4;
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ AttnParams p,
                                                               int pieces, int R) {
  __shared__ float4 so[kJoinWarps][32];
  __shared__ float sl[kJoinWarps], sm[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_seq = p.c.Hkv * p.row_tiles;
  const int row = blockIdx.x % p.rows;
  const int bh = blockIdx.x / p.rows;
  const int b = bh / p.c.Hkv;
  const int hr = (bh - b * p.c.Hkv) * p.row_tiles + row / R;
  pdl_wait();
  const int c0 = p.cum[b], n = p.cum[b + 1] - c0;
  const int line = p.cum[p.c.B] * per_seq;
  const int quota = (line + pieces - 1) / pieces;
  const int s = c0 * per_seq + hr * n;
  const int first = s / quota, last = (s + n - 1) / quota;
  if (first == last) return;  // written whole
  const long long slot0 = static_cast<long long>(b) * per_seq + hr;
  const int r = row % R;
  float mx = -INFINITY, sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int c = first + warp; c <= last; c += kJoinWarps) {
    const float lg = p.part_l[(slot0 + c) * R + r];
    const float4 y = reinterpret_cast<const float4*>(p.part_o)[((slot0 + c) * R + r) * (kHeadDim / 4) + lane];
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
  const long long g = static_cast<long long>(bh) * p.rows + row;
  reinterpret_cast<uint2*>(p.o)[g * (kHeadDim / 4) + lane] =
      make_uint2(pack_out(out.x * inv, out.y * inv, p.out_bf16), pack_out(out.z * inv, out.w * inv, p.out_bf16));
  if (p.lse != nullptr && lane == 0)
    p.lse[g] = total > 0.0f ? (top + log2f(total)) * 0.69314718055994531f : -INFINITY;
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
    known[dev] = n;
  }
  *sms = known[dev];
  return BSATTN_OK;
}

int fill_cache(Cache* c, const void* k_pages, const void* v_pages, const int64_t* page_strides,
               const int32_t* block_table, int64_t table_stride, int max_pages, int n_pages,
               int page_size, const int32_t* seq_lens, const int32_t* q_lens, int B, int Hkv,
               int Tq, void* workspace, size_t workspace_bytes) {
  if (!k_pages || !v_pages || !page_strides || !block_table || !seq_lens) return BSATTN_E_NULL;
  if (B < 1 || Hkv < 1 || Tq < 1 || max_pages < 1 || n_pages < 1 || table_stride < 0)
    return BSATTN_E_SHAPE;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
    return BSATTN_E_SHAPE;
  if (static_cast<long long>(max_pages) * page_size > (1ll << 31) - 2 * kTileKeys)
    return BSATTN_E_SHAPE;
  if (!workspace || workspace_bytes < bsattn_workspace_bytes()) return BSATTN_E_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(k_pages) & 15u) != 0 ||
      (reinterpret_cast<uintptr_t>(v_pages) & 15u) != 0)
    return BSATTN_E_ALIGN;
  for (int i = 0; i < 6; ++i)
    if (page_strides[i] < 0 || page_strides[i] % 8 != 0) return BSATTN_E_ALIGN;
  c->k = static_cast<const char*>(k_pages);
  c->v = static_cast<const char*>(v_pages);
  c->k_page = page_strides[0] * 2;
  c->k_head = page_strides[1] * 2;
  c->k_tok = page_strides[2] * 2;
  c->v_page = page_strides[3] * 2;
  c->v_head = page_strides[4] * 2;
  c->v_tok = page_strides[5] * 2;
  c->table = block_table;
  c->table_stride = table_stride;
  c->seq_lens = seq_lens;
  c->q_lens = q_lens;
  c->max_pages = max_pages;
  c->n_pages = n_pages;
  c->page_shift = 0;
  while ((1 << c->page_shift) < page_size) ++c->page_shift;
  c->B = B;
  c->Hkv = Hkv;
  c->Tq = Tq;
  c->err = static_cast<int*>(workspace);
  return BSATTN_OK;
}

// The launch of one call: rows of q per tile of rows, pieces of the line, scratch.
struct Shape {
  int rows, R, row_tiles, pieces;
  long long items, slots;
  size_t cum_bytes, bytes;
};

static int shape_of(int B, int Hq, int Hkv, int Tq, int max_pages, int page_size, int sms,
                    Shape* s) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 || Tq < 1) return BSATTN_E_SHAPE;
  const long long rows = static_cast<long long>(Hq / Hkv) * Tq;
  if (rows * B * Hkv > (1ll << 31) - 1) return BSATTN_E_SHAPE;
  s->rows = static_cast<int>(rows);
  s->R = rows <= 8 ? 8 : 16;
  s->row_tiles = static_cast<int>((rows + s->R - 1) / s->R);
  s->items = static_cast<long long>(B) * Hkv * s->row_tiles;
  // Most tiles a sequence can have; the line is never longer than that for every item.
  const long long tiles = (static_cast<long long>(max_pages) * page_size + kTileKeys - 1) / kTileKeys + 1;
  if (s->items * tiles > (1ll << 30)) return BSATTN_E_SHAPE;
  s->pieces = static_cast<int>(std::min<long long>(sms, s->items * tiles));
  // A piece of an item is numbered item + CTA: along the line one of the two always grows.
  s->slots = s->items + s->pieces;
  s->cum_bytes = (static_cast<size_t>(B + 1) * sizeof(int) + 255) / 256 * 256;
  s->bytes = s->cum_bytes + static_cast<size_t>(s->slots) * s->R * (kHeadDim + 1) * sizeof(float);
  return BSATTN_OK;
}

static int launch_paged(const void* q, const Cache& cache, const Rule& rule, int Hq, float scale,
                        int dtype_flags, int page_size, void* o, float* lse, void* scratch,
                        size_t scratch_bytes, cudaStream_t stream) {
  if (!q || !o) return BSATTN_E_NULL;
  if ((dtype_flags & ~(BSATTN_OUT_BF16 | BSATTN_IN_BF16)) != 0) return BSATTN_E_DTYPE;
  if ((reinterpret_cast<uintptr_t>(q) & 15u) != 0 || (reinterpret_cast<uintptr_t>(o) & 15u) != 0 ||
      (reinterpret_cast<uintptr_t>(scratch) & 15u) != 0)
    return BSATTN_E_ALIGN;
  int sms = 0;
  int rc = device_sms(&sms);
  if (rc != BSATTN_OK) return rc;
  Shape s;
  rc = shape_of(cache.B, Hq, cache.Hkv, cache.Tq, cache.max_pages, page_size, sms, &s);
  if (rc != BSATTN_OK) return rc;
  if (!scratch || scratch_bytes < s.bytes) return BSATTN_E_WORKSPACE;
  AttnParams p;
  p.c = cache;
  p.rule = rule;
  p.q = q;
  p.o = o;
  p.lse = lse;
  p.G = Hq / cache.Hkv;
  p.rows = s.rows;
  p.row_tiles = s.row_tiles;
  const double sc = scale > 0.0f ? static_cast<double>(scale) : 0.08838834764831845;
  p.scale_log2 = static_cast<float>(sc * 1.4426950408889634);
  p.out_bf16 = (dtype_flags & BSATTN_OUT_BF16) != 0;
  p.cum = static_cast<int*>(scratch);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(scratch) + s.cum_bytes);
  p.part_l = p.part_o + s.slots * s.R * kHeadDim;
  const bool bf16 = (dtype_flags & BSATTN_IN_BF16) != 0;
  const unsigned grid = static_cast<unsigned>(s.pieces);
  if (s.R == 8) {
    if (bf16) decode_kernel<true, 1><<<grid, kThreadsD, sizeof(DecodeSmem<1>), stream>>>(p);
    else decode_kernel<false, 1><<<grid, kThreadsD, sizeof(DecodeSmem<1>), stream>>>(p);
  } else {
    if (bf16) decode_kernel<true, 2><<<grid, kThreadsD, sizeof(DecodeSmem<2>), stream>>>(p);
    else decode_kernel<false, 2><<<grid, kThreadsD, sizeof(DecodeSmem<2>), stream>>>(p);
  }
  if (cudaGetLastError() != cudaSuccess) return BSATTN_E_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<long long>(cache.B) * cache.Hkv * s.rows));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, join_kernel, p, s.pieces, s.R) != cudaSuccess) {
    cudaGetLastError();
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
  rc = shape_of(B, Hq, Hkv, Tq, max_pages, page_size, sms, &s);
  if (rc != BSATTN_OK) return rc;
  *bytes = s.bytes;
  return BSATTN_OK;
}

int bsattn_paged_fwd(const void* q, const void* k_pages, const void* v_pages,
                     const int64_t* page_strides, const int32_t* block_table, int64_t table_stride,
                     int max_pages, int n_pages, int page_size, const int32_t* seq_lens,
                     const int32_t* q_lens, void* o, float* lse, int B, int Hq, int Hkv, int Tq,
                     int window, int global_blocks, int prefix_len, float scale, int dtype_flags,
                     void* scratch, size_t scratch_bytes, void* workspace, size_t workspace_bytes,
                     void* stream) {
  Cache c;
  const int rc = fill_cache(&c, k_pages, v_pages, page_strides, block_table, table_stride,
                            max_pages, n_pages, page_size, seq_lens, q_lens, B, Hkv, Tq, workspace,
                            workspace_bytes);
  if (rc != BSATTN_OK) return rc;
  constexpr int kMaxWindow = 1 << 24;
  if (window < 0 || window > kMaxWindow || global_blocks < 0 || global_blocks > kMaxWindow ||
      (window == 0 && global_blocks != 0))
    return BSATTN_E_SHAPE;
  if (prefix_len < 0 || prefix_len % page_size != 0 ||
      static_cast<long long>(prefix_len) > static_cast<long long>(max_pages) * page_size ||
      (prefix_len > 0 && window > 0))
    return BSATTN_E_SHAPE;
  Rule rule;
  rule.k0 = 0;
  rule.window = window;
  rule.glob = global_blocks;
  return launch_paged(q, c, rule, Hq, scale, dtype_flags, page_size, o, lse, scratch,
                      scratch_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

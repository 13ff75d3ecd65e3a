// paged_append.cu -- new tokens into a paged K/V cache, with the position rotation on the way.
//
// For the live rows t < q_lens[b] of every sequence, at position p = seq_lens[b] - q_lens[b] + t:
//   k_pages[page, h, slot] = R(p) k[b, h, t],  v_pages[page, h, slot] = v[b, h, t],
//   q_out[b, h, t] = R(p) q[b, h, t],          page = block_table[b][p / page], slot = p % page.
// R(p) turns pair i, (x_i, x_{i + rot/2}) or (x_2i, x_{2i+1}), by the angle p * inv_freq[i].
//
// The angle is formed in 64 bits and reduced to a fraction of a turn before it is rounded to 32:
// at position 10^6 a 32-bit product would be off by up to 0.03 rad.  The rotation itself is 32-bit
// and rounds once, on the store.
//
// A row is 256 bytes; eight threads take two 16-byte pieces of it each, chosen so that both
// members of every pair are in one thread (which also makes q_out == q safe).  Memory bound: every
// element is read once and written once.  A block takes kTok tokens of one sequence row range: its
// threads first compute the kTok x rot/2 sines and cosines once into shared memory, then walk the
// tokens' q, k and v rows.
#include <algorithm>

#include "paged_common.cuh"

namespace bsattn {
namespace paged {

constexpr int kAppendThreads = 128;
constexpr int kTok = 2;  // tokens per block (16,384 tokens of 48 heads: 54.7 us; one 58.1, four 59.0)

struct AppendParams {
  Cache c;
  char* k_pages;
  char* v_pages;
  const char* q;
  const char* k;
  const char* v;
  char* q_out;
  // byte strides of the inputs over batch, head, token
  long long qs[3], ks[3], vs[3];
  const double* inv_freq;
  int rot, interleaved;
  int Hq;
  int heads_per_block;  // q, k and v rows of a token are split over gridDim.y blocks
};

template <bool BF16>
__device__ __forceinline__ void rotate_pieces(const AppendParams& p, const float2* cs, int j,
                                              uint4& x, uint4& y) {
  uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
  uint32_t* yw = reinterpret_cast<uint32_t*>(&y);
  if (p.interleaved) {
    // pieces 2j and 2j+1: pairs 8j .. 8j+3 and 8j+4 .. 8j+7
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (16 * j < p.rot) {
        const float2 a = unpack16<BF16>(xw[e]), f = cs[8 * j + e];
        xw[e] = pack16<BF16>(a.x * f.x - a.y * f.y, a.y * f.x + a.x * f.y);
        const float2 b = unpack16<BF16>(yw[e]), g = cs[8 * j + 4 + e];
        yw[e] = pack16<BF16>(b.x * g.x - b.y * g.y, b.y * g.x + b.x * g.y);
      }
    }
  } else if (16 * j < p.rot) {
    // pieces j and j + rot/16: pairs 8j .. 8j+7
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = unpack16<BF16>(xw[e]), b = unpack16<BF16>(yw[e]);
      const float2 f = cs[8 * j + 2 * e], g = cs[8 * j + 2 * e + 1];
      xw[e] = pack16<BF16>(a.x * f.x - b.x * f.y, a.y * g.x - b.y * g.y);
      yw[e] = pack16<BF16>(b.x * f.x + a.x * f.y, b.y * g.x + a.y * g.y);
    }
  }
}

template <bool BF16>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ float2 cs[kTok][kHeadDim / 2];
  __shared__ int s_pos[kTok], s_page[kTok], s_b[kTok], s_t[kTok];
  pdl_wait();
  pdl_trigger();
  const long long tok0 = static_cast<long long>(blockIdx.x) * kTok;
  const long long tokens = static_cast<long long>(p.c.B) * p.c.Tq;
  const int half = p.rot / 2;
  for (int i = threadIdx.x; i < kTok * (kHeadDim / 2); i += kAppendThreads) {
    const int u = i / (kHeadDim / 2), f = i % (kHeadDim / 2);
    const long long tok = tok0 + u;
    int pos = -1, b = -1, t = 0;
    if (tok < tokens) {
      b = static_cast<int>(tok / p.c.Tq);
      t = static_cast<int>(tok - static_cast<long long>(b) * p.c.Tq);
      const SeqLen s = seq_len(p.c, b);
      // A forced length or count says where no token belongs: it would go over one that is held.
      if (t < s.rows && s.ok) pos = s.len - s.rows + t;
    }
    if (f == 0) {
      int page = -1;
      if (pos >= 0)
        page = page_checked(p.c, __ldg(p.c.table + b * p.c.table_stride + (pos >> p.c.page_shift)));
      s_pos[u] = pos;
      s_page[u] = page;
      s_b[u] = b;
      s_t[u] = t;
    }
    if (f < half && pos >= 0) {
      // turns = position * inv_freq / 2 pi, reduced to [-1/2, 1/2] in 64 bits
      const double turns = static_cast<double>(pos) * p.inv_freq[f] * 0.15915494309189533577;
      float sn, cn;
      sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cn);
      cs[u][f] = make_float2(cn, sn);
    }
  }
  __syncthreads();

  const int heads = p.Hq + 2 * p.c.Hkv;
  const int h0 = blockIdx.y * p.heads_per_block;
  const int hn = min(p.heads_per_block, heads - h0);
  const int j = threadIdx.x & 7;
  // The two 16-byte pieces of this thread.
  int c0, c1;
  if (p.interleaved) {
    c0 = 2 * j;
    c1 = 2 * j + 1;
  } else if (16 * j < p.rot) {
    c0 = j;
    c1 = j + p.rot / 16;
  } else {
    c0 = p.rot / 8 + 2 * (j - p.rot / 16);
    c1 = c0 + 1;
  }
  const int off0 = c0 * 16, off1 = c1 * 16;
  for (int r = threadIdx.x >> 3; r < hn * kTok; r += kAppendThreads / 8) {
    const int u = r / hn;
    int h = h0 + r - u * hn;
    const int b = s_b[u], pos = s_pos[u];
    if (b < 0) continue;
    const long long t = s_t[u];
    const char* src;
    char* dst;
    bool turn = true;
    if (h < p.Hq) {
      dst = p.q_out + ((static_cast<long long>(b) * p.Hq + h) * p.c.Tq + t) * (kHeadDim * 2);
      if (pos < 0) {  // padding rows of q_out are zero
        *reinterpret_cast<uint4*>(dst + off0) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + off1) = make_uint4(0, 0, 0, 0);
        continue;
      }
      src = p.q + b * p.qs[0] + h * p.qs[1] + t * p.qs[2];
    } else {
      const int page = s_page[u];
      if (page < 0) continue;
      const long long slot = pos & ((1 << p.c.page_shift) - 1);
      h -= p.Hq;
      if (h < p.c.Hkv) {
        src = p.k + b * p.ks[0] + h * p.ks[1] + t * p.ks[2];
        dst = p.k_pages + page * p.c.k_page + h * p.c.k_head + slot * p.c.k_tok;
      } else {
        h -= p.c.Hkv;
        src = p.v + b * p.vs[0] + h * p.vs[1] + t * p.vs[2];
        dst = p.v_pages + page * p.c.v_page + h * p.c.v_head + slot * p.c.v_tok;
        turn = false;
      }
    }
    uint4 x = *reinterpret_cast<const uint4*>(src + off0);
    uint4 y = *reinterpret_cast<const uint4*>(src + off1);
    if (turn) rotate_pieces<BF16>(p, cs[u], j, x, y);
    *reinterpret_cast<uint4*>(dst + off0) = x;
    *reinterpret_cast<uint4*>(dst + off1) = y;
  }
}

}  // namespace paged
}  // namespace bsattn

using namespace bsattn;
using namespace bsattn::paged;

extern "C" int bsattn_paged_append(const bsattn_paged_call* call, const void* q, const void* k,
                                   const void* v, const int64_t* in_strides, void* q_out,
                                   const double* inv_freq, int rot_dim, int interleaved) {
  AppendParams p;
  int rc = fill_cache(&p.c, call);
  if (rc != BSATTN_OK) return rc;
  const int B = call->B, Hq = call->Hq, Hkv = call->Hkv, Tq = call->Tq;
  if (Hq < 0) return BSATTN_E_SHAPE;
  if (!k || !v || !in_strides || (Hq > 0 && (!q || !q_out))) return BSATTN_E_NULL;
  if ((call->dtype_flags & ~BSATTN_IN_BF16) != 0) return BSATTN_E_DTYPE;
  if (inv_freq == nullptr) rot_dim = 0;
  if (rot_dim < 0 || rot_dim > kHeadDim || rot_dim % 16 != 0 || (inv_freq && rot_dim == 0) ||
      (reinterpret_cast<uintptr_t>(inv_freq) & 7u) != 0)
    return BSATTN_E_SHAPE;
  const void* ptrs[] = {Hq > 0 ? q : k, k, v, Hq > 0 ? q_out : k};
  for (const void* x : ptrs)
    if ((reinterpret_cast<uintptr_t>(x) & 15u) != 0) return BSATTN_E_ALIGN;
  for (int i = 0; i < 9; ++i) {
    if (i < 3 && Hq == 0) continue;
    if (in_strides[i] < 0 || in_strides[i] % 8 != 0) return BSATTN_E_ALIGN;
    (i < 3 ? p.qs : i < 6 ? p.ks : p.vs)[i % 3] = in_strides[i] * 2;
  }
  const long long heads = static_cast<long long>(Hq) + 2ll * Hkv;
  const long long tokens = static_cast<long long>(B) * Tq;
  if (heads > 65535 || tokens > (1ll << 31) - 2) return BSATTN_E_SHAPE;
  int sms = 0;
  if ((rc = device_sms(&sms)) != BSATTN_OK) return rc;
  p.k_pages = static_cast<char*>(call->k_pages);
  p.v_pages = static_cast<char*>(call->v_pages);
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.q_out = static_cast<char*>(q_out);
  p.inv_freq = inv_freq;
  p.rot = rot_dim;
  p.interleaved = interleaved ? 1 : 0;
  p.Hq = Hq;
  const long long bx = (tokens + kTok - 1) / kTok;
  // One pass of the block's 16 row slots over kTok tokens covers 8 heads; with few tokens the
  // heads are split over blocks down to that, so that every SM has work (one token of 48 heads: 2.4 us,
  // in one block 3.6).
  long long split = std::min<long long>((heads + 7) / 8, std::max<long long>(1, 4ll * sms / bx));
  p.heads_per_block = static_cast<int>((heads + split - 1) / split);
  const dim3 grid(static_cast<unsigned>(bx),
                  static_cast<unsigned>((heads + p.heads_per_block - 1) / p.heads_per_block));
  return launch((call->dtype_flags & BSATTN_IN_BF16) ? append_kernel<true> : append_kernel<false>, grid,
                kAppendThreads, 0, static_cast<cudaStream_t>(call->stream), p);
}

// paged_few.cuh -- launch interface of the few-row attention over a paged cache (paged_few.cu), and
// the line on which its work is laid out, which the join behind a shared prefix has to know.
#pragma once

#include "paged_common.cuh"

namespace bsattn {
namespace paged {

constexpr int kFewRows = 8;    // rows of a tile of rows
constexpr int kSlice = 16;     // keys a warp takes at a time
constexpr int kMaxSms = 160;   // CTAs of a call at most (a B200 has 148 SMs)

struct FewCall {
  Cache c;
  Rule rule;
  const void* q;
  void* o;
  float* lse;
  int rows, row_tiles;     // rows = G * Tq, in tiles of kFewRows
  float scale_log2;
  int in_bf16, out_bf16;
  int all_partial;         // behind a shared prefix: no piece is a whole result
  int ctas;
  // Scratch: for the join behind a prefix, the sequences' places on the line [B + 1], the line's
  // quota and alignment; partial outputs and their log2 sums, slots of kFewRows rows.
  int* cum;
  float* part_o;
  float* part_l;
  int* counters;           // [2, kMaxSms, kFewRows], zero between calls
};

int few_setup();
int few_launch(const FewCall& call, cudaStream_t stream);

// The line.  An item is (sequence, K/V head, tile of rows): its slices of 16 keys, one unit each, and
// kItemUnits for what its end costs.  The line of all items is cut into pieces of `quota` units, one
// per CTA, and those into equal shares for its warps; a warp takes the slices that begin in its share.
// When there are CTAs enough for every item to have its own, that may be better than equal pieces
// (align > 0: items are rounded up to whole pieces of that many units, and no CTA holds two).
constexpr int kItemUnits = 1;
struct Line {
  int quota, align;
};
// Units of an item of n slices.
__device__ __forceinline__ int units_of(int n, int align) {
  return align > 0 ? (n + align - 1) / align * align : n + kItemUnits;
}
// Last CTA that holds a slice of the item that begins at unit `at`.
__device__ __forceinline__ int last_cta(const Line& x, int at, int units) {
  return (x.align > 0 ? at + units - 1 : at + units - kItemUnits - 1) / x.quota;
}

// Where the part of an item that a CTA holds is left.  A CTA holds at most one item that begins in it
// and goes on, and one that began before; when whole items are partial too (behind a prefix), item +
// cta numbers all parts, since along the line one of the two always grows.
__host__ __device__ __forceinline__ long long part_slot(int all_partial, long long item, int cta,
                                                        bool head) {
  return all_partial ? item + cta : 2ll * cta + (head ? 1 : 0);
}

__device__ __forceinline__ void store_row(void* o, float* lse, int out_bf16, long long row, float4 v,
                                          float lg, int lane) {
  reinterpret_cast<uint2*>(o)[row * (kHeadDim / 4) + lane] =
      make_uint2(pack_out(v.x, v.y, out_bf16), pack_out(v.z, v.w, out_bf16));
  if (lse != nullptr && lane == 0) lse[row] = lg * 0.69314718055994531f;
}

// A weighted sum of partial rows.  Rows in global memory are read past L1: other SMs may have written
// them while the kernel ran.
struct PartSum {
  float4 acc;
  float sum;
  __device__ __forceinline__ void clear() {
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    sum = 0.0f;
  }
  __device__ __forceinline__ void scale(float f) {
    acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
    sum *= f;
  }
  __device__ __forceinline__ void add(float4 y, float w) {
    acc.x += y.x * w;
    acc.y += y.y * w;
    acc.z += y.z * w;
    acc.w += y.w * w;
    sum += w;
  }
  __device__ __forceinline__ float4 normal() const {
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    return make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  }
  __device__ __forceinline__ float log2_total(float mx) const {
    return sum > 0.0f ? mx + log2f(sum) : -INFINITY;
  }
};
__device__ __forceinline__ float4 part_row(const float* po, long long row, int lane) {
  return __ldcg(reinterpret_cast<const float4*>(po) + row * (kHeadDim / 4) + lane);
}

}  // namespace paged
}  // namespace bsattn

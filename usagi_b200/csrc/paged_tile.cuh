// paged_tile.cuh -- launch interface of the many-row attention over a paged cache (paged_tile.cu).
#pragma once

#include "paged_common.cuh"

namespace bsattn {
namespace paged {

// How the rows of q fill tiles of 128: a tile holds n_t tokens of G query heads of n_b sequences,
// row = (b * G + g) * n_t + t.  A virtual sequence is one tile of rows over one list of keys.
struct RowTiles {
  int G, n_t, n_b;
  int per_seq;  // virtual sequences per sequence (n_b == 1), or 1
  int count;    // virtual sequences of the call
};

// What CTA c leaves for the join: the item that begins in it and goes on in the next ones, and in
// how many CTAs it lies (v < 0: none).  Its pieces are slots 2 c + 1, then 2 (c + 1), 2 (c + 2), ...
struct TileCut {
  int v, h, pieces, unused;
};

struct TileCall {
  Cache c;
  Rule rule;       // k0 is 0
  RowTiles rt;
  int prefix_len;  // > 0: the keys are the first prefix_len tokens of sequence 0, for every row
  const void* q;
  void* o;
  float* lse;
  int Hq;
  float scale_log2;
  int in_bf16, out_bf16;
  int pieces;      // CTAs
  long long slots; // partial outputs of 128 rows
  TileCut* cuts;   // [pieces], without a prefix
  float* part_o;   // [slots][32 pieces of four columns][128 rows]
  float* part_l;   // [slots, 128], log2
};

// Registers the kernels need per thread at launch, checked once per device.
int tile_setup();
int tile_launch(const TileCall& call, int page_size, cudaStream_t stream);

}  // namespace paged
}  // namespace bsattn

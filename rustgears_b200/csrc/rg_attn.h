// rg_attn.h -- what the paged-attention kernels share: launch parameters and the rule that
// picks between them.
#pragma once
#include "rg_serving.h"

namespace rg {

struct AttnParams {
  PagedAttnArgs p;
  FastDiv page, group;
  float scale2;  // scale * log2(e)
  // A kernel takes the sequences with min_rows < rows <= max_rows (rows: tokens times the heads
  // that share a key head): a batch may mix decoding sequences and chunks.
  int32_t min_rows, max_rows;
  // A sequence's keys may be split over blocks: their partial rows (not normalised; maximum and
  // sum) go to the workspace, split s of row (token, head) at s * tokens * heads + token * heads
  // + head, and k_attn_join adds them.
  int32_t splits;
  float* part_o;
  float2* part_ml;
};

// Which of a sequence's key tiles a split takes.  The same function serves the kernels and the
// join, so all agree on how many splits have work.
struct KeySplit {
  int32_t tiles, per, active;  // key tiles seen, tiles of a split, splits that have any (1 at least)
  __device__ __forceinline__ KeySplit(int seen, int key_tile, int splits) {
    tiles = (seen + key_tile - 1) / key_tile;
    per = max(1, (tiles + splits - 1) / splits);
    active = max(1, (tiles + per - 1) / per);
  }
};

// A launch's shape of tiles.
struct TileShape {
  int32_t rows, keys, splits;
};
struct JoinParams {
  AttnParams A;
  TileShape few, many;  // of the sequences with at most / more than `limit` rows
  int32_t limit;
};

// The tcgen05 kernel (k_attn_tc.cu): head_dim 64 or 128, page sizes of 8 to 64 tokens that are
// powers of two, or multiples of 128.
bool attention_tc_takes(const PagedAttnArgs& p);
constexpr int kTcRows = 256, kTcKeys = 128;  // its tiles
// `beside`: the launch before it is the kernel for few rows, which it does not depend on.
rg_status launch_attention_tc(const AttnParams& P, bool beside, cudaStream_t st);

}  // namespace rg

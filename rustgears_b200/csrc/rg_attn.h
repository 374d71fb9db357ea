// rg_attn.h -- what the paged-attention kernels share: launch parameters and the rule that
// picks between them.
#pragma once
#include "rg_serving.h"

namespace rg {

// n / d for 0 <= n < 2^31 by multiplication (Granlund and Montgomery, PLDI 1994):
// m = floor(2^32 (2^l - d) / d) + 1, l = ceil(log2 d).
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t v = 1) : d(v) {
    uint32_t l = 0;
    while ((1ull << l) < v) ++l;
    m = (uint32_t)(((1ull << 32) * ((1ull << l) - v)) / v + 1);
    s = l;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return (uint32_t)(((uint64_t)__umulhi(n, m) + n) >> s);
  }
};

struct AttnParams {
  PagedAttnArgs p;
  FastDiv page, group;
  float scale2;  // scale * log2(e)
  // A kernel takes the sequences with min_rows < rows <= max_rows (rows: tokens times the heads
  // that share a key head): a batch may mix decoding sequences and chunks.
  int32_t min_rows, max_rows;
};

// The tcgen05 kernel (k_attn_tc.cu): head_dim 64 or 128, page sizes of 8 to 64 tokens that are
// powers of two, or multiples of 128.
bool attention_tc_takes(const PagedAttnArgs& p);
rg_status launch_attention_tc(const AttnParams& P, cudaStream_t st);

}  // namespace rg

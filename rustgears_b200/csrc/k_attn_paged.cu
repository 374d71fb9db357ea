// k_attn_paged.cu -- attention of a chunk of new tokens over a paged cache.
//
// Query i of sequence b (of q_len, with kv_len keys) sees keys j <= kv_len - q_len + i:
//   o = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s),  s_j = scale * q . k_j,
// one pass over the keys with the running maximum and sum; a row without keys is zeros.
#include "rg_serving.h"

namespace rg {
namespace {

// One warp per query row (token, head); lane l holds dimensions l, l + 32, ...
template <typename T, int D>
__global__ void __launch_bounds__(128) k_attn_rows(const PagedAttnArgs p) {
  const rg_kv_cache& c = p.c;
  const rg_paged_attention_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1];
  const int kv = a.kv_len[b];
  if (q0 < 0 || q1 < q0 || q1 > a.tokens || q1 - q0 > a.max_q_len || kv < 0 || kv > a.max_kv_len) {
    if (threadIdx.x == 0) p.err[1] = 1;
    return;
  }
  const int ql = (int)(q1 - q0);
  if (i >= ql) return;
  const int hk = h / (a.heads / c.kv_heads);
  constexpr int N = D / 32;
  float q[N], o[N];
  const T* qp = static_cast<const T*>(a.q) + (q0 + i) * a.q_token_stride + h * a.q_head_stride;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    q[j] = ElemOf<T>::to(qp[lane + 32 * j]) * a.scale;
    o[j] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;
  const int last = a.causal ? min(kv, kv - ql + i + 1) : kv;  // keys seen
  for (int key = 0; key < last; ++key) {
    const int page = a.block_table[(int64_t)b * a.block_table_stride + key / c.page_size];
    const bool ok = page >= 0 && page < c.pages;
    if (!ok && lane == 0) p.err[1] = 1;
    const int64_t at = ok ? page * c.page_stride + (key % c.page_size) * c.token_stride + hk * c.head_stride : 0;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j)
      s = fmaf(q[j], ok ? ElemOf<T>::to(static_cast<const T*>(c.k)[at + lane + 32 * j]) : 0.0f, s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float m = fmaxf(top, s);
    const float keep = m == -INFINITY ? 1.0f : expf(top - m);
    const float e = m == -INFINITY ? 0.0f : expf(s - m);
    sum = fmaf(sum, keep, e);
    top = m;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float v = ok ? ElemOf<T>::to(static_cast<const T*>(c.v)[at + lane + 32 * j]) : 0.0f;
      o[j] = fmaf(o[j], keep, e * v);
    }
  }
  T* op = static_cast<T*>(a.out) + (q0 + i) * a.out_token_stride + h * a.out_head_stride;
#pragma unroll
  for (int j = 0; j < N; ++j) op[lane + 32 * j] = ElemOf<T>::from(sum > 0.0f ? o[j] / sum : 0.0f);
}

template <typename T>
rg_status go(const PagedAttnArgs& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.a.max_q_len + 3) / 4), (unsigned)p.a.heads, (unsigned)p.a.batch);
  switch (p.c.head_dim) {
    case 64: k_attn_rows<T, 64><<<grid, 128, 0, st>>>(p); break;
    case 96: k_attn_rows<T, 96><<<grid, 128, 0, st>>>(p); break;
    case 128: k_attn_rows<T, 128><<<grid, 128, 0, st>>>(p); break;
    default: k_attn_rows<T, 256><<<grid, 128, 0, st>>>(p); break;
  }
  return RG_OK;
}

}  // namespace

int64_t attention_paged_workspace(const PagedAttnArgs&) { return 0; }

rg_status launch_attention_paged(const PagedAttnArgs& p, cudaStream_t st) {
  return p.c.dtype == RG_DTYPE_F16 ? go<__half>(p, st) : go<__nv_bfloat16>(p, st);
}

}  // namespace rg

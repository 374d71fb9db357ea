// k_attn_paged.cu -- attention of a chunk of new tokens over a paged cache: the kernel for
// few rows (decoding), and for the shapes the tcgen05 kernel does not take.
//
// Query i of sequence b (of q_len, with kv_len keys) sees keys j <= kv_len - q_len + i:
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j,  m = max s_j,
// one pass over the keys with the running maximum and sum; a row without keys is zeros.
//
// Rows: the heads / kv_heads query heads that share a key head are rows of one matrix
// product, row r = token r / group, head r % group, so a key is read once for all of them.
// A block takes 16 WR rows of one (sequence, key head) and a share of its keys; its warps
// are WR row groups x WK key groups, each 16 rows x its keys of every tile, with its
// own maximum, sum and output (registers), joined once at the end.
//
// Bound: memory for few rows (keys and values are read once: 4 head_dim bytes per key and
// key head; 16 rows fill one m16n8k16 fragment, whose rate is far above what the loads
// need).  A three-stage ring of cp.async tiles keeps two tiles in flight per block, two blocks
// per SM.  Few (sequence, head) pairs leave SMs idle, so a sequence's keys are split over
// blocks whose partial rows a second, overlapped launch joins in a fixed order.  (A cluster
// of up to 16 blocks joining through distributed shared memory was slower: the blocks of a
// cluster start together, which costs a wait for 16 free places; 16.2 against 11.3 us at one
// token over 4001 keys.)
//
// Measured (32 query heads on 8 of 128, bf16): one token over 4001 keys 11.2 us (16.4 MB, half of
// it launches and the join); over 131072 keys 94 us (5.7 TB/s); 64 sequences of up to 6144 keys
// 183 us (5.6 TB/s).
#include <algorithm>
#include <climits>

#include "rg_attn.h"
#include "rg_mma16.cuh"

namespace rg {
namespace {

using namespace mma16;

constexpr int kStages = 3;
constexpr float kLog2e = 1.44269504088896340736f;

constexpr int few_keys(int d) { return d <= 128 ? 64 : 32; }

template <int D, int WR, int WK>
struct Shape {
  static constexpr int KT = few_keys(D);           // keys of a tile: two blocks' rings fit an SM
  static constexpr int kWarps = WR * WK, kThreads = 32 * kWarps, kRows = 16 * WR;
  static constexpr int kKeys = KT / WK;            // keys of a warp in a tile
  static constexpr int kPitch = D * 2 + 16;        // odd multiple of 16 bytes: ldmatrix without conflicts
  static constexpr int kTile = KT * kPitch;
  static constexpr int kStage = 2 * kTile;         // keys, values
  static constexpr int kQ = kRows * kPitch;
  static constexpr int kOffs = (kStages + 1) * KT * 8;
  static constexpr int kSmem = kQ + kStages * kStage + kOffs;
  static constexpr bool kQRegs = D <= 128;         // query fragments stay in registers
  // the join reuses the ring: kRows x (D + 4) outputs, then per-warp maxima and sums
  static constexpr int kOPitch = D + 4;
  static_assert(kRows * kOPitch * 4 + 2 * (kWarps + 1) * 16 * WR * 4 <= kStages * kStage, "join fits the ring");
};

template <typename T, int D, int WR, int WK>
__global__ void __launch_bounds__(32 * WR * WK) k_attn_few(const AttnParams P) {
  using S = Shape<D, WR, WK>;
  constexpr int KT = S::KT;
  extern __shared__ __align__(16) uint8_t smem[];
  const rg_kv_cache& c = P.p.c;
  const rg_paged_attention_args& a = P.p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = warp % WR, wk = warp / WR;
  const int split = blockIdx.x % P.splits, tile = blockIdx.x / P.splits;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int group = P.group.d;

  uint8_t* sq = smem;
  uint8_t* ring = smem + S::kQ;
  int64_t* offs = reinterpret_cast<int64_t*>(ring + kStages * S::kStage);  // [kStages + 1][KT], -1: zeros

  grid_dependency_wait();
  const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1];
  const int kv = a.kv_len[b];
  if (q0 < 0 || q1 < q0 || q1 > a.tokens || q1 - q0 > a.max_q_len || kv < 0 || kv > a.max_kv_len) {
    if (tid == 0) P.p.err[1] = 1;
    return;
  }
  const int ql = (int)(q1 - q0), rows = ql * group, row0 = tile * S::kRows;
  if (row0 >= rows || rows <= P.min_rows || rows > P.max_rows) return;
  // keys seen by the tile's last row
  const int last_tok = (int)P.group.div((uint32_t)(min(row0 + S::kRows, rows) - 1));
  const int seen = a.causal ? max(0, min(kv, kv - ql + last_tok + 1)) : kv;
  const KeySplit ks(seen, KT, P.splits);
  if (split >= ks.active) return;
  const int t0 = split * ks.per, t1 = min(t0 + ks.per, ks.tiles);

  // ---- queries: rows past the last one are zeros ----
  for (int i = tid; i < S::kRows * (D / 8); i += S::kThreads) {
    const int r = i / (D / 8), ch = i % (D / 8), row = row0 + r;
    const bool ok = row < rows;
    const int tok = (int)P.group.div((uint32_t)(ok ? row : 0)), h = hk * group + (ok ? row : 0) - tok * group;
    cp_async16(saddr(sq + r * S::kPitch + ch * 16),
               static_cast<const T*>(a.q) + (q0 + tok) * a.q_token_stride + h * a.q_head_stride + ch * 8, ok);
  }
  cp_async_commit();

  // ---- key addresses: thread r < KT looks tile t's key r up, one tile ahead of its loads ----
  const int32_t* table = a.block_table + (int64_t)b * a.block_table_stride;
  constexpr int kNone = INT_MIN;  // no such key
  const auto look = [&](int t) -> int {
    const int key = t * KT + tid;
    return tid < KT && t < t1 && key < seen ? table[P.page.div((uint32_t)key)] : kNone;
  };
  const auto offset = [&](int t, int page) -> int64_t {
    if (page < 0 || page >= c.pages) {
      if (page != kNone) P.p.err[1] = 1;
      return -1;
    }
    const int key = t * KT + tid;
    return page * c.page_stride + (int64_t)(key - P.page.div((uint32_t)key) * c.page_size) * c.token_stride +
           hk * c.head_stride;
  };
  const auto load = [&](int t) {  // tile t into its stage
    const int stage = (t - t0) % kStages;
    const int64_t* off = offs + ((t - t0) % (kStages + 1)) * KT;
    const uint32_t base = saddr(ring + stage * S::kStage);
#pragma unroll 4
    for (int i = tid; i < KT * (D / 8); i += S::kThreads) {
      const int r = i / (D / 8), ch = i % (D / 8);
      const int64_t o = off[r];
      const bool ok = o >= 0;
      const int64_t at = ok ? o + ch * 8 : 0;
      cp_async16(base + r * S::kPitch + ch * 16, static_cast<const T*>(c.k) + at, ok);
      cp_async16(base + S::kTile + r * S::kPitch + ch * 16, static_cast<const T*>(c.v) + at, ok);
    }
  };
  int ahead;
  {
    int page[kStages];
#pragma unroll
    for (int s = 0; s < kStages; ++s) page[s] = look(t0 + s);
    ahead = look(t0 + kStages);
    if (tid < KT)
#pragma unroll
      for (int s = 0; s < kStages; ++s) offs[s * KT + tid] = offset(t0 + s, page[s]);
  }
  __syncthreads();
  for (int s = 0; s < kStages - 1; ++s) {
    if (t0 + s < t1) load(t0 + s);
    cp_async_commit();
  }

  // ---- main loop ----
  const int g = lane >> 2, t4 = lane & 3;
  int limit[2];  // keys seen by this thread's two rows (g, g + 8)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = row0 + wr * 16 + g + 8 * i;
    limit[i] = row >= rows ? 0 : a.causal ? min(kv, kv - ql + (int)P.group.div((uint32_t)row) + 1) : kv;
  }
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
  uint32_t qf[S::kQRegs ? D / 16 : 1][4];
  const uint32_t q_addr = saddr(sq + (wr * 16 + (lane & 15)) * S::kPitch + (lane >> 4) * 16);

  for (int t = t0; t < t1; ++t) {
    cp_async_wait<kStages - 2>();
    if (tid < KT) {
      offs[((t - t0 + kStages) % (kStages + 1)) * KT + tid] = offset(t + kStages, ahead);
      ahead = look(t + kStages + 1);
    }
    __syncthreads();  // tile t has landed, and everyone is done with tile t - 1's stage
    if (t + kStages - 1 < t1) load(t + kStages - 1);
    cp_async_commit();
    if constexpr (S::kQRegs) {
      if (t == t0)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) ldmatrix4(qf[d], q_addr + d * 32);
    }
    const uint32_t kb = saddr(ring + ((t - t0) % kStages) * S::kStage) + wk * S::kKeys * S::kPitch;
    const uint32_t vb = kb + S::kTile;
    // scores: fragments of 8 keys
    float s[S::kKeys / 8][4];
#pragma unroll
    for (int j = 0; j < S::kKeys / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][i] = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      if constexpr (!S::kQRegs) ldmatrix4(qf[0], q_addr + d * 32);
#pragma unroll
      for (int j = 0; j < S::kKeys / 16; ++j) {
        uint32_t kf[4];  // keys 16 j .. + 7 (dims 0-7, 8-15), then the next 8 keys
        ldmatrix4(kf, kb + (j * 16 + (lane & 7) + ((lane >> 4) << 3)) * S::kPitch + d * 32 + ((lane >> 3) & 1) * 16);
        mma<T>(s[2 * j], qf[S::kQRegs ? d : 0], kf[0], kf[1]);
        mma<T>(s[2 * j + 1], qf[S::kQRegs ? d : 0], kf[2], kf[3]);
      }
    }
    const int key0 = t * KT + wk * S::kKeys + 2 * t4;
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int j = 0; j < S::kKeys / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = s[j][i] * P.scale2;
        s[j][i] = key0 + j * 8 + (i & 1) < limit[i >> 1] ? v : -INFINITY;
        top[i >> 1] = fmaxf(top[i >> 1], s[j][i]);
      }
    float base[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      base[i] = top[i] == -INFINITY ? 0.0f : top[i];  // no key yet: 2^(-inf - 0) = 0
    }
    if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
      const float f0 = ex2(m[0] - base[0]), f1 = ex2(m[1] - base[1]);
      l[0] *= f0;
      l[1] *= f1;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= f0;
        o[j][1] *= f0;
        o[j][2] *= f1;
        o[j][3] *= f1;
      }
      m[0] = top[0];
      m[1] = top[1];
    }
#pragma unroll
    for (int j = 0; j < S::kKeys / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[j][i] = ex2(s[j][i] - base[i >> 1]);
        l[i >> 1] += s[j][i];
      }
    // output: the probabilities, rounded to the cache's type, times the values.  (The matrix
    // instructions take both operands in one 16-bit type; the rounding adds at most half a step of
    // that type, relative, to a sum that is rounded to it at the end: 1.2 to 1.4 times the error
    // of f32 probabilities.  The row sum adds them unrounded.)
#pragma unroll
    for (int j = 0; j < S::kKeys / 16; ++j) {
      const uint32_t pf[4] = {pack<T>(s[2 * j][0], s[2 * j][1]), pack<T>(s[2 * j][2], s[2 * j][3]),
                              pack<T>(s[2 * j + 1][0], s[2 * j + 1][1]), pack<T>(s[2 * j + 1][2], s[2 * j + 1][3])};
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t vf[4];  // dims 16 d .. + 7 (keys 0-7, 8-15), then the next 8 dims
        ldmatrix4_trans(vf, vb + (j * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * S::kPitch + d * 32 + (lane >> 4) * 16);
        mma<T>(o[2 * d], pf, vf[0], vf[1]);
        mma<T>(o[2 * d + 1], pf, vf[2], vf[3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }

  grid_launch_dependents();  // (earlier, the next launch's blocks would sit unevenly among these)

  // ---- join the key groups: every warp scales to the rows' common maximum, adds in order ----
  cp_async_wait<0>();
  __syncthreads();
  float* jo = reinterpret_cast<float*>(ring);          // [kRows][kOPitch]
  float* jm = jo + S::kRows * S::kOPitch;              // [WK][kRows], then the joined [kRows]
  float* jl = jm + (S::kWarps + 1) * 16 * WR;
  const int r0 = wr * 16 + g;
  if (t4 == 0)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      jm[wk * S::kRows + r0 + 8 * i] = m[i];
      jl[wk * S::kRows + r0 + 8 * i] = l[i];
    }
  __syncthreads();
  float f[2], M[2], L[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    M[i] = -INFINITY;
    L[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < WK; ++w) M[i] = fmaxf(M[i], jm[w * S::kRows + r0 + 8 * i]);
    const float base = M[i] == -INFINITY ? 0.0f : M[i];
#pragma unroll
    for (int w = 0; w < WK; ++w) L[i] += jl[w * S::kRows + r0 + 8 * i] * ex2(jm[w * S::kRows + r0 + 8 * i] - base);
    f[i] = ex2(m[i] - base);
  }
  for (int w = 0; w < WK; ++w) {
    if (wk == w)
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2* dst = reinterpret_cast<float2*>(jo + (r0 + 8 * i) * S::kOPitch + j * 8 + 2 * t4);
          float2 v = w == 0 ? make_float2(0.0f, 0.0f) : *dst;
          v.x += o[j][2 * i] * f[i];
          v.y += o[j][2 * i + 1] * f[i];
          *dst = v;
        }
    __syncthreads();
  }
  float* fm = jm + WK * S::kRows;  // the block's maxima and sums
  float* fl = jl + WK * S::kRows;
  if (wk == 0 && t4 == 0)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fm[r0 + 8 * i] = M[i];
      fl[r0 + 8 * i] = L[i];
    }

  // ---- store: the rows, or what this split has of them ----
  __syncthreads();
  const int64_t part = (int64_t)split * a.tokens * a.heads;
  for (int i = tid; i < S::kRows * (D / 8); i += S::kThreads) {
    const int r = i / (D / 8), ch = i % (D / 8), row = row0 + r;
    if (row >= rows) break;
    const int tok = (int)P.group.div((uint32_t)row), h = hk * group + row - tok * group;
    float v[8];
    Pack<float, 8>::load(jo + r * S::kOPitch + ch * 8, v);
    if (ks.active > 1) {
      const int64_t at = part + (q0 + tok) * a.heads + h;
      Pack<float, 8>::store(P.part_o + at * D + ch * 8, v);
      if (ch == 0) P.part_ml[at] = make_float2(fm[r], fl[r]);
    } else {
      const float inv = 1.0f / fl[r];
#pragma unroll
      for (int x = 0; x < 8; ++x) v[x] = fl[r] == 0.0f ? 0.0f : v[x] * inv;  // no key: zeros
      Pack<T, 8>::store(static_cast<T*>(a.out) + (q0 + tok) * a.out_token_stride + h * a.out_head_stride + ch * 8, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Joins the splits' partial rows, in a fixed order: W of a block's 8 warps per row, each adding
// every W-th split (few rows and many splits are a matter of latency: their loads are all in
// flight at once).  Launched beside the end of the kernels before it (its blocks wait for them).
// ---------------------------------------------------------------------------
template <typename T, int D, int W>
__global__ void __launch_bounds__(256) k_attn_join(const JoinParams J) {
  const AttnParams& P = J.A;
  const rg_paged_attention_args& a = P.p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hk = blockIdx.y, b = blockIdx.z, group = P.group.d;
  const int row = blockIdx.x * (8 / W) + warp / W, w = warp % W;
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1];
  const int kv = a.kv_len[b];
  if (q0 < 0 || q1 < q0 || q1 > a.tokens || q1 - q0 > a.max_q_len || kv < 0 || kv > a.max_kv_len) return;
  const int ql = (int)(q1 - q0), rows = ql * group;
  if (row >= rows) return;
  const TileShape& sh = rows <= J.limit ? J.few : J.many;
  const int last = min(row / sh.rows * sh.rows + sh.rows, rows) - 1;  // of the row's tile
  const int seen = a.causal ? max(0, min(kv, kv - ql + (int)P.group.div((uint32_t)last) + 1)) : kv;
  const KeySplit ks(seen, sh.keys, sh.splits);
  if (ks.active == 1) return;  // stored by its block
  const int tok = (int)P.group.div((uint32_t)row), h = hk * group + row - tok * group;
  const int64_t at = (q0 + tok) * a.heads + h, step = a.tokens * a.heads;
  float top = -INFINITY;
  for (int s = lane; s < ks.active; s += 32) top = fmaxf(top, P.part_ml[at + s * step].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  const float base = top == -INFINITY ? 0.0f : top;
  constexpr int N = D / 32;  // dimensions N lane .. + N - 1
  float v[N], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
#pragma unroll 4
  for (int s = w; s < ks.active; s += W) {
    const float2 ml = P.part_ml[at + s * step];
    float o[N];
    const float* src = P.part_o + (at + s * step) * D + lane * N;
    if constexpr (N % 2 == 0) {
      Pack<float, N>::load(src, o);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = src[i];
    }
    const float e = ex2(ml.x - base);
    sum += e * ml.y;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += e * o[i];
  }
  if constexpr (W > 1) {
    __shared__ float add[8][33 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) add[warp][lane * N + i] = v[i];
    if (lane == 0) add[warp][32 * N] = sum;
    __syncthreads();
    if (w != 0) return;
    for (int x = 1; x < W; ++x) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += add[warp + x][lane * N + i];
      sum += add[warp + x][32 * N];
    }
  }
  const float inv = 1.0f / sum;
  T* dst = static_cast<T*>(a.out) + (q0 + tok) * a.out_token_stride + h * a.out_head_stride + lane * N;
#pragma unroll
  for (int i = 0; i < N; ++i) dst[i] = ElemOf<T>::from(sum == 0.0f ? 0.0f : v[i] * inv);
}

template <typename T, int D, int WR, int WK>
rg_status go(const AttnParams& A, cudaStream_t st) {
  using S = Shape<D, WR, WK>;
  const auto kernel = k_attn_few<T, D, WR, WK>;
  static DeviceOnce once;
  once.run([&] { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem); });
  const int64_t rows = std::min<int64_t>((int64_t)std::max(A.p.a.max_q_len, 1) * A.group.d, A.max_rows);
  const int64_t tiles = (rows + S::kRows - 1) / S::kRows;
  if (tiles * A.splits > INT_MAX) return RG_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)(tiles * A.splits), (unsigned)A.p.c.kv_heads, (unsigned)A.p.a.batch);
  launch_early(kernel, grid, S::kThreads, S::kSmem, st, A);
  return RG_OK;
}

// Rows of a block: 16 (one fragment, all warps on the keys), or 64 where rows come in numbers.
// Beside chunks the sequences of this kernel are decoding ones, mostly of few rows.
inline int few_rows(const AttnParams& A) {
  return (int64_t)A.p.a.max_q_len * A.group.d <= 16 || A.max_rows < INT_MAX ? 16 : 64;
}
template <typename T, int D>
rg_status go_rows(const AttnParams& A, cudaStream_t st) {
  return few_rows(A) == 16 ? go<T, D, 1, (D <= 128 ? 4 : 2)>(A, st) : go<T, D, 4, 2>(A, st);
}

template <typename T>
rg_status go_dim(const AttnParams& A, cudaStream_t st) {
  switch (A.p.c.head_dim) {
    case 64: return go_rows<T, 64>(A, st);
    case 96: return go_rows<T, 96>(A, st);
    case 128: return go_rows<T, 128>(A, st);
    default: return go_rows<T, 256>(A, st);
  }
}

rg_status launch_few(const AttnParams& A, cudaStream_t st) {
  return A.p.c.dtype == RG_DTYPE_F16 ? go_dim<__half>(A, st) : go_dim<__nv_bfloat16>(A, st);
}

template <typename T, int W>
void launch_join(const JoinParams& J, int64_t rows, cudaStream_t st) {
  const dim3 grid((unsigned)((rows * W + 7) / 8), (unsigned)J.A.p.c.kv_heads, (unsigned)J.A.p.a.batch);
  switch (J.A.p.c.head_dim) {
    case 64: launch_early(k_attn_join<T, 64, W>, grid, 256, 0, st, J); break;
    case 96: launch_early(k_attn_join<T, 96, W>, grid, 256, 0, st, J); break;
    case 128: launch_early(k_attn_join<T, 128, W>, grid, 256, 0, st, J); break;
    default: launch_early(k_attn_join<T, 256, W>, grid, 256, 0, st, J); break;
  }
}
template <typename T>
void launch_join(const JoinParams& J, int64_t rows, cudaStream_t st) {
  // a block per row where the rows do not fill the SMs by themselves
  if (rows * J.A.p.c.kv_heads * J.A.p.a.batch <= 148 * 8 && std::max(J.few.splits, J.many.splits) > 4)
    launch_join<T, 8>(J, rows, st);
  else launch_join<T, 1>(J, rows, st);
}

// How a launch's time depends on its splits, in microseconds (measured): a block's start, a key
// tile, `slots` blocks at once.
struct Pace {
  int slots;
  double start, tile;
};

// Splits of `blocks` blocks of at most `tiles` key tiles.  Blocks that all run at once take as
// long as the longest; more of them take their sum over the slots, and half a longest block
// until the last one ends: the host knows the longest sequence only, so the others of a batch
// count as 0.6 of it.  The join costs about 2 us, and join_us a split for the partial rows.
int split_keys(int64_t blocks, int64_t tiles, bool one_sequence, const Pace& pace, int min_tiles, double join_us) {
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= 64 && (s == 1 || (tiles + s - 1) / s >= min_tiles); ++s) {
    const int64_t per = (tiles + s - 1) / s, n = blocks * s;
    const double one = pace.start + pace.tile * (double)per;
    double t = one;
    if (n > pace.slots)
      t = one_sequence ? (double)((n + pace.slots - 1) / pace.slots) * one
                       : (double)n / pace.slots * (pace.start + 0.6 * pace.tile * (double)per) + 0.5 * one;
    if (s > 1) t += 2.0 + s * join_us;
    if (t < 0.97 * least) {
      least = t;
      best = s;
    }
  }
  return best;
}

// Up to so many rows (tokens times the heads that share a key head) a sequence takes the kernel
// for few rows: one block's; beside chunks one fragment's, so that a sequence of the batch costs
// one block of that launch and not four of which three find nothing.
constexpr int kFewRows = 64, kFewRowsBeside = 16;

struct Plan {
  AttnParams A;
  bool few, many;
  TileShape few_shape, many_shape;
  int64_t rows;
  int64_t part_rows;  // rows of partial results, all splits
};

rg_status make_plan(const PagedAttnArgs& p, Plan& L) {
  AttnParams& A = L.A;
  A.p = p;
  A.page = FastDiv((uint32_t)p.c.page_size);
  A.group = FastDiv((uint32_t)(p.a.heads / p.c.kv_heads));
  A.scale2 = p.a.scale * kLog2e;
  A.splits = 1;
  A.part_o = nullptr;
  A.part_ml = nullptr;
  // (max_q_len 0: one block per sequence and head reports those that have tokens)
  L.rows = (int64_t)std::max(p.a.max_q_len, 1) * A.group.d;
  if (L.rows > INT_MAX || p.c.kv_heads > 65535) return RG_ERR_UNSUPPORTED;
  // Chunks go to the tensor-core kernel.  Where the batch may hold shorter sequences too (the
  // tokens are fewer than batch times the longest), those take the kernel for few rows.
  L.many = p.a.max_q_len > 0 && L.rows > kFewRows && attention_tc_takes(p);
  L.few = !L.many || (p.a.batch > 1 && p.a.tokens < (int64_t)p.a.batch * p.a.max_q_len);
  A.min_rows = 0;
  A.max_rows = L.many ? kFewRowsBeside : INT_MAX;
  const int d = p.c.head_dim;
  const double row_us = 8.0 * d * (double)p.a.tokens * p.a.heads / 5e6;  // partial rows written and read
  const int64_t seqs = (int64_t)p.c.kv_heads * p.a.batch;
  L.few_shape = {few_rows(A), few_keys(d), 1};
  L.many_shape = {kTcRows, kTcKeys, 1};
  if (L.few && p.a.max_q_len > 0) {
    // (beside chunks: taken as one block for every other sequence)
    const int64_t blocks = L.many ? (seqs + 1) / 2 : seqs * ((L.rows + L.few_shape.rows - 1) / L.few_shape.rows);
    // blocks an SM holds at once (Shape::kSmem)
    const int keys = L.few_shape.keys, smem = (L.few_shape.rows + 6 * keys) * (2 * d + 16) + 4 * keys * 8;
    const Pace pace = {148 * std::min(3, 227 * 1024 / smem), 2.5, d <= 64 ? 0.6 : d <= 96 ? 0.8 : 1.1};
    L.few_shape.splits = split_keys(blocks, (p.a.max_kv_len + L.few_shape.keys - 1) / L.few_shape.keys,
                                    p.a.batch == 1, pace, 2, row_us);
  }
  if (L.many) {
    // blocks with work: what the tokens fill, and half a block for every sequence's rest
    const int64_t most = seqs * ((L.rows + kTcRows - 1) / kTcRows);
    const int64_t blocks = std::min<int64_t>(
        most, (p.a.tokens * A.group.d / kTcRows + (p.a.batch + 1) / 2 + 1) * (int64_t)p.c.kv_heads);
    const Pace pace = {148, 4.0, d <= 64 ? 1.6 : 1.9};
    L.many_shape.splits = split_keys(blocks, (p.a.max_kv_len + kTcKeys - 1) / kTcKeys, p.a.batch == 1, pace, 2, row_us);
  }
  const int most = std::max(L.few ? L.few_shape.splits : 1, L.many ? L.many_shape.splits : 1);
  L.part_rows = most > 1 ? most * p.a.tokens * p.a.heads : 0;
  return RG_OK;
}

}  // namespace

int64_t attention_paged_workspace(const PagedAttnArgs& p) {
  Plan L;
  if (make_plan(p, L) != RG_OK) return 0;
  return L.part_rows * (p.c.head_dim * 4 + 8);
}

rg_status launch_attention_paged(const PagedAttnArgs& p, cudaStream_t st) {
  Plan L;
  rg_status s = make_plan(p, L);
  if (s != RG_OK) return s;
  AttnParams& A = L.A;
  A.part_o = static_cast<float*>(p.workspace);
  A.part_ml = reinterpret_cast<float2*>(A.part_o + L.part_rows * p.c.head_dim);
  if (L.few) {
    A.splits = L.few_shape.splits;
    s = launch_few(A, st);
    if (s != RG_OK) return s;
  }
  if (L.many) {
    A.splits = L.many_shape.splits;
    A.min_rows = L.few ? kFewRowsBeside : 0;
    A.max_rows = INT_MAX;
    s = launch_attention_tc(A, L.few, st);
    if (s != RG_OK) return s;
  }
  if (L.part_rows) {
    JoinParams J;
    J.A = A;
    J.few = L.few_shape;
    J.many = L.many_shape;
    J.limit = !L.many ? INT_MAX : L.few ? kFewRowsBeside : 0;
    // unsplit chunks have nothing to join: then the rows of the others only
    const int64_t rows = L.many && L.many_shape.splits == 1 ? std::min<int64_t>(L.rows, J.limit) : L.rows;
    if (p.c.dtype == RG_DTYPE_F16) launch_join<__half>(J, rows, st);
    else launch_join<__nv_bfloat16>(J, rows, st);
  }
  return RG_OK;
}

}  // namespace rg

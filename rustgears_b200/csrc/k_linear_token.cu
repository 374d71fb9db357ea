// k_linear_token.cu -- i8 x i8 product with one scale per token and one per output channel:
//   sa[r] = absmax(x[r]) < 1e-12 ? 1 : absmax / 127,  q = clamp(round(x / sa)),
//   out[r, c] = act(f32(sum_k q[r,k] w[c,k]) * (sa[r] * sw[c]) + bias[c]).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <cstring>

#include "rg_f32x2.cuh"
#include "rg_math.cuh"
#include "rg_mma16.cuh"
#include "rg_serving.h"
#include "rg_sm100_pair.cuh"

namespace rg {

PFN_cuTensorMapEncodeTiled_v12000 tma_encode_fn();  // k_gemm_tc.cu

namespace {

constexpr int kQuantThreads = 256;

// ---------------------------------------------------------------------------
// Row quantizer.  Bound: memory (x read once, q and the scales written once).  One block
// per row; the row stays in registers, as it was read, between its absmax and its rounding
// (32 values a thread, 8192 a row); longer rows are read again, from L1 or L2.  16384 x 8192: bf16
// 76 us (5.3 TB/s), f32 97 us (6.9 TB/s).  (A block looping over rows with the next one read
// ahead: 86 us for bf16: its registers leave four blocks on an SM instead of six.)
// ---------------------------------------------------------------------------
// The low bytes of four integers.
__device__ __forceinline__ uint32_t pack_i8(int32_t a, int32_t b, int32_t c, int32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
template <typename T>
__device__ __forceinline__ T from_bits(uint16_t v);
template <>
__device__ __forceinline__ __half from_bits<__half>(uint16_t v) { return __ushort_as_half(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_bits<__nv_bfloat16>(uint16_t v) { return __ushort_as_bfloat16(v); }
// Largest magnitude, NaN ignored; 16-bit values two at a time (their maximum is exact).
template <typename T>
struct AbsMax;
template <>
struct AbsMax<float> {
  float m = 0.0f;
  __device__ __forceinline__ void fold(float a, float b) { m = fmaxf(m, fmaxf(fabsf(a), fabsf(b))); }
  __device__ __forceinline__ float value() const { return m; }
};
template <>
struct AbsMax<__half> {
  __half2 m = __half2half2(__ushort_as_half(0));
  __device__ __forceinline__ void fold(__half a, __half b) { m = __hmax2(m, __habs2(__halves2half2(a, b))); }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct AbsMax<__nv_bfloat16> {
  __nv_bfloat162 m = __bfloat162bfloat162(__ushort_as_bfloat16(0));
  __device__ __forceinline__ void fold(__nv_bfloat16 a, __nv_bfloat16 b) {
    m = __hmax2(m, __habs2(__halves2bfloat162(a, b)));
  }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(m), __high2float(m)); }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 2 ? 6 : 4)
    k_quantize_token(const T* x, int64_t k, int64_t ldx, int8_t* q, int64_t ldq, float* scale) {
  constexpr int E = VEC ? 16 / (int)sizeof(T) : 4;  // values a thread handles at once
  constexpr int NREG = 32 / E;
  // A chunk as it was read: 32-bit words, taken apart where they are used (16-bit values would be
  // unpacked behind each load, which then waits for it).
  constexpr int W = E * (int)sizeof(T) / 4;
  struct Raw {
    uint32_t w[W];
    __device__ __forceinline__ T at(int j) const {
      if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
      else return from_bits<T>((uint16_t)(w[j / 2] >> (j % 2 * 16)));
    }
  };
  __shared__ float red[kQuantThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int chunks = (int)(ldq / E);
  const auto read = [&](int64_t r, int c) {
    Raw v;
    const int64_t at = (int64_t)c * E;
    const T* src = x + r * ldx;
    if (VEC && at + E <= k) {
      const uint4 u = *reinterpret_cast<const uint4*>(src + at);
      v.w[0] = u.x; v.w[1] = u.y; v.w[2] = u.z; v.w[3] = u.w;
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < E; ++j) v.w[j] = at + j < k ? __float_as_uint(src[at + j]) : 0u;
    } else {
      const uint16_t* bits = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int j = 0; j < E; j += 2)
        v.w[j / 2] = (at + j < k ? bits[at + j] : 0u) | (at + j + 1 < k ? (uint32_t)bits[at + j + 1] << 16 : 0u);
    }
    return v;
  };
  const int64_t r = blockIdx.x;
  Raw keep[NREG];
#pragma unroll
  for (int i = 0; i < NREG; ++i) {
    const int c = threadIdx.x + i * kQuantThreads;
    if (c < chunks) keep[i] = read(r, c);
  }
  {
    AbsMax<T> peak;
    const auto fold = [&](const Raw& v) {
#pragma unroll
      for (int j = 0; j < E; j += 2) peak.fold(v.at(j), v.at(j + 1));
    };
#pragma unroll
    for (int i = 0; i < NREG; ++i)
      if (threadIdx.x + i * kQuantThreads < chunks) fold(keep[i]);
    for (int c = threadIdx.x + NREG * kQuantThreads; c < chunks; c += kQuantThreads) fold(read(r, c));
    float amax = peak.value();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQuantThreads / 32; ++i) amax = fmaxf(amax, red[i]);
    const float sc = quant_scale(amax), inv = quant_inv(sc);
    if (threadIdx.x == 0) scale[r] = sc;
    const auto write = [&](int c, const Raw& v) {
      struct alignas(E) Out {
        uint32_t w[E / 4];
      } u;
#pragma unroll
      for (int j = 0; j < E; j += 4)
        u.w[j / 4] = pack_i8(quant1_bounded(ElemOf<T>::to(v.at(j)), inv), quant1_bounded(ElemOf<T>::to(v.at(j + 1)), inv),
                             quant1_bounded(ElemOf<T>::to(v.at(j + 2)), inv),
                             quant1_bounded(ElemOf<T>::to(v.at(j + 3)), inv));
      *reinterpret_cast<Out*>(q + r * ldq + (int64_t)c * E) = u;
    };
#pragma unroll
    for (int i = 0; i < NREG; ++i) {
      const int c = threadIdx.x + i * kQuantThreads;
      if (c < chunks) write(c, keep[i]);
    }
    for (int c = threadIdx.x + NREG * kQuantThreads; c < chunks; c += kQuantThreads) write(c, read(r, c));
  }
}

template <typename T>
void quantize(const void* x, int64_t rows, int64_t k, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
              cudaStream_t st) {
  const bool vec = (((uintptr_t)x | (uintptr_t)(ldx * (int64_t)sizeof(T))) & 15) == 0;
  const T* p = static_cast<const T*>(x);
  const dim3 grid((unsigned)rows);
  if (vec) launch_early(k_quantize_token<T, true>, grid, kQuantThreads, 0, st, p, k, ldx, q, ldq, scale);
  else launch_early(k_quantize_token<T, false>, grid, kQuantThreads, 0, st, p, k, ldx, q, ldq, scale);
}

// ---------------------------------------------------------------------------
// Product on the tensor cores: tcgen05 kind::i8 on CTA pairs.
//
// A pair's tile is 256 rows x BN columns: each CTA holds 128 rows of A, BN / 2 rows of W and
// the sums of its 128 rows (TMEM, two accumulators, so that one tile's epilogue runs beside
// the next tile's products).  Bound: the tensor pipe for many rows; against one CTA per tile
// a pair halves the bytes of W that each SM writes to and reads from shared memory per
// product, which is what held the single-CTA form at 0.6 of the rate (128 x 256 x 32 moves
// 96 bytes a clock in and 96 out, of 128).  For few rows it is the stream of W: rows of A past
// m are filled with zeros without traffic, and narrow tiles spread W over all SMs.
// Measured alone: 16384 x 8192 x 8192 660 us = 3330 TOPS, 4096 x 8192 x 8192 163 us = 3380 (tensor
// pipe 91 % active); 2048 x 4096 x 14336 + GELU to f16 about 88 us (448 tiles on 74 pairs: seven
// rounds where 6.05 have work).
//   warp 0      TMA producer of its own CTA's operands, completing on the even CTA's barrier
//   warp 1      of the even CTA: issues the products for both
//   warps 2-9   epilogue: scale, bias, activation, rounding, a 64-byte-wide tile staged in
//               shared memory and written by TMA (or by row, where rows are not 16-byte aligned)
// Every wait is bounded; a CTA that gives up sets the caller's error word.
// ---------------------------------------------------------------------------
using namespace sm100;

constexpr int kBK = 128;  // bytes of K per stage: one 128-byte swizzle row
constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 64 + 32 * kEpiWarps;
constexpr uint64_t kWaitNs = 2000000000ull, kDrainNs = 200000000ull;

constexpr int kRing = 192 * 1024;            // operand stages
constexpr int kMaxStages = 24;
constexpr int kStaging = kEpiWarps * 4096;   // two 2 KB tiles per epilogue warp
constexpr int kGemmSmem = 1024 + kRing + kStaging + 512;
static_assert(kGemmSmem <= 227 * 1024, "shared memory per CTA");

struct PairParams {
  TokenGemmArgs g;
  int32_t tiles_m, tiles_n, num_kb, group_m;
  // Rows of A a CTA loads (128; fewer when m is, and then the odd CTA loads none: a short
  // stage leaves room for more of W in flight).  The products read 128 rows all the same;
  // what lies behind the loaded ones only reaches rows that are not stored.
  int32_t a_rows, a_ctas, stages, stage_bytes;
  int32_t tma_store;
  uint64_t wait_ns;
  int32_t starve;
};

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Activation of N pre-activation values.  f32 results follow the framework's restatements
// bit for bit.  For 16-bit results GELU and SiLU are x / (1 + 2^a) on the hardware's exponent
// and reciprocal: 8 instructions a value instead of about 90, which would outlast the products
// of a 4096-long reduction.  Relative error: 2^-20 where the result is of x's size, and with
// the f32 rounding of a about 2^-22 |a| more where it vanishes (GELU 2^-17.4 at x = -7,
// 2^-16 at -10; SiLU 2^-19 at -40, 2^-18 at -87), under 1/16 of the types' half steps of 2^-9 and
// 2^-12; bf16's subnormal results are within one of their steps.
template <bool GELU>
__device__ __forceinline__ float smooth16(float x) {
  // GELU: 0.5 x (1 + tanh u) = x / (1 + e^(-2u)), u = sqrt(2 / pi) (x + 0.044715 x^3).  (x x may
  // overflow: the exponent is infinite then, of the right sign.)  Numerator and denominator are
  // taken times 2^-14: 1 + 2^a has a normal reciprocal up to a = 126 only, but x / (1 + 2^a) is a
  // bf16 number up to a = 140.
  constexpr float c1 = GELU ? -2.0f * 0.7978846f * 1.44269504f : -1.44269504f, c3 = c1 * 0.044715f;
  const float a = fmaf(x, GELU ? fmaf(x * x, c3, c1) : c1, -14.0f);
  return (x * 0x1p-14f) * rcp_approx(0x1p-14f + mma16::ex2(a));
}

template <typename T, int N>
__device__ __forceinline__ void activate(float (&y)[N], int32_t act, float param) {
  if (act == ACT_NONE) return;
  if (act == ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = fmaxf(y[j], 0.0f);
    return;
  }
  if (sizeof(T) == 2 && act == ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = smooth16<true>(y[j]);
    return;
  }
  if (sizeof(T) == 2 && act == ACT_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = smooth16<false>(y[j]);
    return;
  }
  if (act == ACT_GELU) {
    // Two values per packed instruction on the restatement's common range; the others (an
    // argument of 7.5 and more, tiny or not finite) one at a time with the general one.
    float t[N];
    uint32_t redo = 0;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const f32x2 u = gelu_arg_x2(pack2(y[j], y[j + 1]));
      tanh_f32_common_x2(lo2(u), hi2(u), t[j], t[j + 1]);
      redo |= (uint32_t)!tanh_common_range(lo2(u)) << j;
      redo |= (uint32_t)!tanh_common_range(hi2(u)) << (j + 1);
    }
    while (__any_sync(0xffffffffu, redo != 0)) {
      const int jr = redo ? __ffs(redo) - 1 : 0;
      float x = y[0];
#pragma unroll
      for (int j = 1; j < N; ++j) x = jr == j ? y[j] : x;
      const float tr = tanh_f32(gelu_arg(x));
#pragma unroll
      for (int j = 0; j < N; ++j) t[j] = (redo && jr == j) ? tr : t[j];
      redo &= redo - 1;
    }
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const f32x2 g = gelu_from_tanh_x2(pack2(y[j], y[j + 1]), pack2(t[j], t[j + 1]));
      y[j] = lo2(g);
      y[j + 1] = hi2(g);
    }
    return;
  }
#pragma unroll 1
  for (int j0 = 0; j0 < N; j0 += 4) {  // rolled: one copy of the long restatements
    float t[4];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if ((j & ~3) == j0) t[j & 3] = y[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = act_apply(act, param, t[j]);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if ((j & ~3) == j0) y[j] = t[j & 3];
  }
}

// Tiles in groups of group_m row tiles that sweep all column tiles: the group's rows of A stay
// in L2 while W streams past.
__device__ __forceinline__ void pair_tile(int tile, const PairParams& p, int& mb, int& nb) {
  const int per = p.group_m * p.tiles_n;
  const int first = tile / per * p.group_m;
  const int gm = min(p.group_m, p.tiles_m - first);
  const int in = tile - tile / per * per;
  mb = first + in % gm;
  nb = in / gm;
}

template <int BN, typename T>
__global__ void __launch_bounds__(kGemmThreads, 1) __cluster_dims__(2, 1, 1)
    k_gemm_token_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                      const __grid_constant__ CUtensorMap map_o, const PairParams p) {
  constexpr int kBBytes = BN / 2 * kBK;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + kRing;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kStaging);  // used in the even CTA
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;   // [2]
  uint64_t* tempty = tfull + 2;           // [2], used in the even CTA
  uint64_t* done = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int num_tiles = p.tiles_m * p.tiles_n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * kEpiWarps);
    }
    mbar_init(done, 1);
    *abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_w);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 2 * BN);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    const uint32_t ring = smem_addr(smem);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int issued = 0;
    if (!p.g.after_quantizer) grid_dependency_wait();  // else only what the quantizer writes is waited for
    for (int tile = pair; tile < num_tiles && ok; tile += pairs) {
      int mb, nb;
      pair_tile(tile, p, mb, nb);
      for (int kb = 0; kb < p.num_kb; ++kb) {
        if (!warp_wait(&empty[stage], phase ^ 1, abort, p.wait_ns)) { ok = false; break; }
        if (!p.starve) {
          const uint32_t sa = ring + stage * p.stage_bytes;
          if (rank == 0) expect_tx_elect(&full[stage], (uint32_t)(p.a_ctas * p.a_rows * kBK + 2 * kBBytes));
          const uint32_t bar = cluster_addr(&full[stage], 0);
          tma_load_2d_pair_elect(sa + p.a_rows * kBK, &map_w, bar, kb * kBK, nb * BN + (int)rank * (BN / 2));
          if ((int)rank < p.a_ctas) {
            if (issued == 0) grid_dependency_wait();  // W may be read before the quantizer is done, A not
            tma_load_2d_pair_elect(sa, &map_a, bar, kb * kBK, mb * 256 + (int)rank * 128);
          }
          ++issued;
        }
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
    // Drain: the products that read the last stages arrive on `empty` here, so no copy or
    // arrival is on its way to this CTA when it leaves.
    volatile int never = 0;
    for (int s = 0; s < p.stages && s < issued; ++s) {
      stage = stage == 0 ? p.stages - 1 : stage - 1;
      if (stage == p.stages - 1) phase ^= 1;
      warp_wait(&empty[stage], phase, &never, kDrainNs);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_i8(256, BN);
      const uint32_t ring = smem_addr(smem);
      int stage = 0, iter = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += pairs, ++iter) {
        const int buf = iter & 1;
        if (!warp_wait(&tempty[buf], ((iter >> 1) & 1) ^ 1, abort, p.wait_ns)) break;
        tc_fence_after();
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!warp_wait(&full[stage], phase, abort, p.wait_ns)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = ring + stage * p.stage_bytes;
          const uint64_t da = desc_kmajor_sw128(sa), db = desc_kmajor_sw128(sa + p.a_rows * kBK);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)  // 32 bytes on: 2 in the descriptors' 16-byte units
            mma_i8_pair_elect(tmem + (uint32_t)(buf * BN), da + 2 * kk, db + 2 * kk, idesc, (kb | kk) != 0);
          commit_pair_elect(&empty[stage]);
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
        if (ok) commit_pair_elect(&tfull[buf]);
      }
      commit_pair_elect(done);
    }
  } else {
    const int q = warp & 3;               // TMEM lane quadrant this warp may access
    const int half = (warp - 2) >> 2;     // which half of the columns
    uint8_t* stg = staging + (warp - 2) * 4096;
    constexpr int kCols = BN / 2;
    constexpr int kBox = 64 / (int)sizeof(T);  // columns of a staged tile
    const TokenGemmArgs& g = p.g;
    int iter = 0, turn = 0;
    grid_dependency_wait();  // the row scales come from the quantizer
    grid_launch_dependents();
    for (int tile = pair; tile < num_tiles; tile += pairs, ++iter) {
      int mb, nb;
      pair_tile(tile, p, mb, nb);
      const int64_t row0 = (int64_t)mb * 256 + rank * 128 + q * 32, row = row0 + lane;
      const float sa = row < g.m ? g.a_scale[row] : 0.0f;
      const int buf = iter & 1;
      const bool got = mbar_wait_tight(&tfull[buf], (iter >> 1) & 1, abort, p.wait_ns);
      if (!__all_sync(0xffffffffu, got)) { *abort = 1; break; }
      tc_fence_after();
#pragma unroll 1
      for (int c0 = half * kCols; c0 < (half + 1) * kCols; c0 += 32) {
        const int64_t col0 = (int64_t)nb * BN + c0;
        if (col0 >= g.n || row0 >= g.m) break;  // warp-uniform
        uint32_t v[32];
        tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + c0), v);
        // lane j holds column col0 + j's scale and bias: one load each, broadcast by shuffles
        const bool in = col0 + lane < g.n;
        const float sw = in ? g.w_scale[col0 + lane] : 0.0f;
        const float bi = in && g.bias ? g.bias[col0 + lane] : 0.0f;
        tmem_ld_wait();
        float y[32];
#pragma unroll
        for (int j = 0; j < 32; ++j)
          y[j] = dequant((int32_t)v[j], __fmul_rn(sa, __shfl_sync(0xffffffffu, sw, j)),
                         __shfl_sync(0xffffffffu, bi, j));
        activate<T, 32>(y, g.act, g.act_param);
        if (p.tma_store) {
#pragma unroll
          for (int bx = 0; bx < 32 / kBox; ++bx) {
            if (col0 + bx * kBox >= g.n) break;
            // two staged tiles in turn: the store before the latest has finished reading
            uint8_t* st = stg + (turn & 1) * 2048;
            ++turn;
            if (lane == 0) bulk_wait_read_1();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // 16-byte chunk j of row `lane`, 64-byte swizzle
              uint4 w;
              if constexpr (sizeof(T) == 4) {
                w = make_uint4(__float_as_uint(y[bx * 16 + 4 * j]), __float_as_uint(y[bx * 16 + 4 * j + 1]),
                               __float_as_uint(y[bx * 16 + 4 * j + 2]), __float_as_uint(y[bx * 16 + 4 * j + 3]));
              } else {
                w = make_uint4(mma16::pack<T>(y[8 * j], y[8 * j + 1]), mma16::pack<T>(y[8 * j + 2], y[8 * j + 3]),
                               mma16::pack<T>(y[8 * j + 4], y[8 * j + 5]), mma16::pack<T>(y[8 * j + 6], y[8 * j + 7]));
              }
              *reinterpret_cast<uint4*>(st + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = w;
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d_evict_first(&map_o, st, (int32_t)col0 + bx * kBox, (int32_t)row0);
              bulk_commit();
            }
          }
        } else {
          // rows not 16-byte aligned: turned in shared memory, 8 columns of 32 rows at a time,
          // so that a row's columns are written together
          float* ft = reinterpret_cast<float*>(stg);
#pragma unroll
          for (int c8 = 0; c8 < 32; c8 += 8) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) ft[lane * 9 + j] = y[c8 + j];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3), cc = lane & 7;
              if (row0 + r < g.m && col0 + c8 + cc < g.n)
                static_cast<T*>(g.out)[(row0 + r) * g.ldo + col0 + c8 + cc] = ElemOf<T>::from(ft[r * 9 + cc]);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(&tempty[buf], 0));
    }
    if (p.tma_store && lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    // every product has completed (and this CTA's copy of the arrival has landed)
    volatile int never = 0;
    mbar_wait(done, 0, &never, p.wait_ns + kDrainNs);
    if (*abort) atomicExch(p.g.err, 1);
  }
  __syncwarp();
  cluster_sync();  // neither CTA leaves, or frees TMEM, while the other still uses it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * BN);
  }
}

// ---------------------------------------------------------------------------
// Product for few tokens: the roles turned, so that a tile is 128 rows of W by all the
// tokens, and K split over a cluster of `splits` CTAs.
//
// Bound: the stream of W, then latency.  A pair's 64-column tile takes 4 KB of W per copy and
// walks all of K: 16.0 us at 64 x 4096 x 4096, 12.5 here, where a copy brings 16 KB of W and the
// splits share K.  The splits' i32 sums are exact in any
// order; they meet in distributed shared memory, where CTA r of the cluster adds and
// finishes its share of the tokens, four of W's rows a thread: a token's outputs are neighbours.
//   warp 0  TMA producer: W (before the quantizer is done), then the tokens
//   warp 1  issues the products
//   warps 2-5  sums, scale, bias, activation, stores
// ---------------------------------------------------------------------------
constexpr int kFewThreads = 192, kFewStages = 12;

struct FewParams {
  TokenGemmArgs g;
  int32_t splits, num_kb;
  int32_t box_rows, n_cols, stages, stage_bytes, ring, tmem_cols;
  int32_t vec_out;  // four neighbouring outputs may be written at once
  uint64_t wait_ns;
  int32_t starve;
};

__device__ __forceinline__ int4 ld_cluster4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads)
    k_gemm_token_few(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                     const FewParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.ring);
  uint64_t* empty = full + kFewStages;
  uint64_t* tfull = empty + kFewStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const TokenGemmArgs& g = p.g;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.splits;
  const int64_t n0 = (int64_t)(blockIdx.x / p.splits) * 128;
  const int tokens = (int)g.m;
  const int kb0 = (int)((int64_t)p.num_kb * split / p.splits), kb1 = (int)((int64_t)p.num_kb * (split + 1) / p.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    *abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_a);
  }
  if (warp == 1) tmem_alloc(tmem_slot, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    if (p.starve != 1) {
      if (!g.after_quantizer) grid_dependency_wait();  // else only what the quantizer writes is waited for
      const uint32_t ring = smem_addr(smem);
      const uint32_t bytes = (uint32_t)(128 + p.box_rows) * kBK;
      const int first = min(p.stages, kb1 - kb0);
      for (int s = 0; s < first; ++s) {
        expect_tx_elect(&full[s], bytes);
        tma_load_2d_elect(ring + s * p.stage_bytes, &map_w, &full[s], (kb0 + s) * kBK, (int)n0);
      }
      grid_dependency_wait();
      for (int s = 0; s < first; ++s)
        tma_load_2d_elect(ring + s * p.stage_bytes + 128 * kBK, &map_a, &full[s], (kb0 + s) * kBK, 0);
      int stage = 0, issued = first;
      uint32_t phase = 0;  // of the use before: its product empties the stage
      for (int kb = kb0 + first; kb < kb1; ++kb, ++issued) {
        if (!warp_wait(&empty[stage], phase, abort, p.wait_ns)) break;
        const uint32_t sw = ring + stage * p.stage_bytes;
        expect_tx_elect(&full[stage], bytes);
        tma_load_2d_elect(sw, &map_w, &full[stage], kb * kBK, (int)n0);
        tma_load_2d_elect(sw + 128 * kBK, &map_a, &full[stage], kb * kBK, 0);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      // Drain: every stage's last copies land before the CTA leaves, whoever gave up and when (after
      // the last copy was issued, too).  Where nobody did, the products wait for them anyway.
      volatile int never = 0;
      for (int s = 0; s < first; ++s) {
        const int op = issued - 1 - s;
        warp_wait(&full[op % p.stages], (uint32_t)(op / p.stages) & 1, &never, kDrainNs);
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(128, p.n_cols), ring = smem_addr(smem);
    int stage = 0;
    uint32_t phase = 0;
    if (p.starve == 2) *abort = 1;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (p.starve == 2 || !warp_wait(&full[stage], phase, abort, p.wait_ns)) break;
      tc_fence_after();
      const uint32_t sw = ring + stage * p.stage_bytes;
      const uint64_t dw = desc_kmajor_sw128(sw), dx = desc_kmajor_sw128(sw + 128 * kBK);
#pragma unroll
      for (int kk = 0; kk < kBK / 32; ++kk)  // 32 bytes on: 2 in the descriptors' 16-byte units
        mma_i8_elect(tmem, dw + 2 * kk, dx + 2 * kk, idesc, (kb - kb0) | kk);
      commit_elect(&empty[stage]);
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    commit_elect(tfull);
    volatile int never = 0;  // all products have completed before TMEM is freed
    warp_wait(tfull, 0, &never, p.wait_ns + kDrainNs);
  } else {
    // The warp's result, not the lane's: what follows it (tcgen05.ld, the activations' votes) takes
    // whole warps.  After a give-up, here or of the products, there are no sums to read.
    const bool got = __all_sync(0xffffffffu, mbar_wait_tight(tfull, 0, abort, p.wait_ns) && !*abort);
    if (!got) *abort = 1;
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;  // of the tile: this thread's TMEM lane
    const uint32_t lanes = tmem + ((uint32_t)(row & ~31) << 16);
    grid_dependency_wait();  // the row scales come from the quantizer
    grid_launch_dependents();
    if (p.splits == 1) {
      const int64_t n = n0 + row;
      const bool row_ok = n < g.n;
      const float sw = row_ok ? g.w_scale[n] : 0.0f;
      const float bi = row_ok && g.bias ? g.bias[n] : 0.0f;
#pragma unroll 1
      for (int t = 0; t < tokens && got; t += 8) {
        uint32_t v[8];
        float y[8];
        tmem_ld8(lanes + t, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          y[j] = dequant((int32_t)v[j], __fmul_rn(t + j < tokens ? g.a_scale[t + j] : 0.0f, sw), bi);
        activate<T, 8>(y, g.act, g.act_param);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (t + j < tokens && row_ok) static_cast<T*>(g.out)[(t + j) * g.ldo + n] = ElemOf<T>::from(y[j]);
      }
    } else {
      int32_t* part = reinterpret_cast<int32_t*>(smem);  // [tokens][128], over the operands
#pragma unroll 1
      for (int t = 0; t < tokens && got; t += 8) {
        uint32_t v[8];
        tmem_ld8(lanes + t, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (t + j < tokens) part[(t + j) * 128 + row] = (int32_t)v[j];
      }
    }
    tc_fence_before();
  }
  if (p.splits > 1) {
    __syncwarp();
    cluster_sync();  // every split's sums are in place
    grid_dependency_wait();
    const int per = (tokens + p.splits - 1) / p.splits;
    const int lo = min(split * per, tokens), items = (min(lo + per, tokens) - lo) * 32;
    // an item: four neighbouring rows of one token; kItems of them in flight per thread
    constexpr int kItems = 4;
    const int row = (threadIdx.x & 31) * 4;
    const int64_t n = n0 + row;
    float sw[4], bi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sw[j] = n + j < g.n ? g.w_scale[n + j] : 0.0f;
      bi[j] = n + j < g.n && g.bias ? g.bias[n + j] : 0.0f;
    }
    const bool whole = n + 4 <= g.n && p.vec_out;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < items; i0 += kItems * kFewThreads) {
      int4 v[kItems];
#pragma unroll
      for (int u = 0; u < kItems; ++u) v[u] = make_int4(0, 0, 0, 0);
      for (int s = 0; s < p.splits; ++s) {
        const uint32_t from = cluster_addr(smem, s) + (uint32_t)(lo * 128 + row) * 4;
#pragma unroll
        for (int u = 0; u < kItems; ++u) {
          const int i = i0 + u * kFewThreads;
          if (i < items) {
            const int4 x = ld_cluster4(from + (uint32_t)(i >> 5) * 512);
            v[u].x += x.x;
            v[u].y += x.y;
            v[u].z += x.z;
            v[u].w += x.w;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const int i = i0 + u * kFewThreads;
        if (i - lane >= items) break;  // warp-uniform
        const int64_t t = lo + min(i, items - 1) / 32;
        const float sa = g.a_scale[t];
        float y[4] = {dequant(v[u].x, __fmul_rn(sa, sw[0]), bi[0]), dequant(v[u].y, __fmul_rn(sa, sw[1]), bi[1]),
                      dequant(v[u].z, __fmul_rn(sa, sw[2]), bi[2]), dequant(v[u].w, __fmul_rn(sa, sw[3]), bi[3])};
        activate<T, 4>(y, g.act, g.act_param);
        T* dst = static_cast<T*>(g.out) + t * g.ldo + n;
        if (whole) {
          Pack<T, 4>::store(dst, y);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < g.n) dst[j] = ElemOf<T>::from(y[j]);
        }
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while another reads its sums
  }
  __syncthreads();
  if (threadIdx.x == 0 && *abort) atomicExch(g.err, 1);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

// ---------------------------------------------------------------------------
// Up to 8 tokens in one launch.  Bound: latency, and the stream of W for wide layers.  Every
// block quantizes the tokens itself (m k values, from L2) while its first loads of W are under
// way, then multiplies its 16 rows of W with mma.sync m16n8k32: W goes from memory to the
// product's registers directly.  A thread's 16 bytes of a row feed two products whose K order is
// permuted the same way on both sides (sums of integers: any order).  The block's 8 warps take
// 64-byte steps of K in turn, and their sums meet in shared memory.
//   The quantizer and the split-K product as two launches take 6.1 us for one token through
// 1024 -> 2816 where this takes 3.8.
// ---------------------------------------------------------------------------
constexpr int kSkinnyTokens = 8, kSkinnyThreads = 256, kSkinnyWarps = 8;
// Measured against the two launches: 3.8 / 6.1 us at 1 x 1024 x 2816, 7.7 / 9.7 at 1 x 4096 x 4096,
// 9.3 / 10 at 2 x 4096 x 4096, 11.8 / 10.3 at 4 x 4096 x 4096 (every block quantizes), 21.7 / 17.1 at
// 1 x 4096 x 14336 (more tiles than blocks at once).
constexpr int64_t kSkinnyValues = 8192;  // m * ld
constexpr int kSkinnyBlocks = 148 * 3;

struct SkinnyParams {
  TokenGemmArgs g;
  const void* x;
  int64_t ldx;
  int32_t k, m, pitch, vec;
};

__device__ __forceinline__ void mma_i8_16832(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename TX, typename TO>
__global__ void __launch_bounds__(kSkinnyThreads, 3) k_linear_skinny(const SkinnyParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int32_t part[kSkinnyWarps][16][kSkinnyTokens];
  __shared__ float peak[kSkinnyWarps], scales[kSkinnyTokens];
  const TokenGemmArgs& g = p.g;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, t4 = lane & 3;
  const int ld = (int)g.ld;
  const int steps = (ld + 63) / 64;  // of K; this warp takes steps warp, warp + 8, ...
  constexpr int U = 4;               // steps in flight
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const auto load_w = [&](int64_t row, int s) {  // 16 bytes of a row at step s
    const int at = s * 64 + t4 * 16;
    return row < g.n && at < ld ? *reinterpret_cast<const uint4*>(g.w + row * ld + at) : zero;
  };
  uint4 w0[U], w1[U];
  const int tile = blockIdx.x;
  grid_dependency_wait();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    w0[u] = load_w((int64_t)tile * 16 + gr, warp + u * kSkinnyWarps);
    w1[u] = load_w((int64_t)tile * 16 + gr + 8, warp + u * kSkinnyWarps);
  }

  // ---- quantize: 8 / (m rounded to a power of two) warps per token ----
  {
    int slots = 1;
    while (slots < p.m) slots *= 2;
    const int per = kSkinnyWarps / slots, token = warp / per, share = (warp % per) * 32 + lane, step = per * 32;
    constexpr int E = 16 / (int)sizeof(TX);
    const TX* x = static_cast<const TX*>(p.x) + token * p.ldx;
    const int chunks = ld / E;  // ld: a multiple of 16
    const auto read = [&](int c, float (&f)[E]) {
      const int at = c * E;
      if (p.vec && at + E <= p.k) {
        Pack<TX, E>::load(x + at, f);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = at + j < p.k ? ElemOf<TX>::to(x[at + j]) : 0.0f;
      }
    };
    float amax = 0.0f;
    if (token < p.m)
      for (int c = share; c < chunks; c += step) {
        float f[E];
        read(c, f);
#pragma unroll
        for (int j = 0; j < E; ++j) amax = fmaxf(amax, fabsf(f[j]));
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) peak[warp] = amax;
    __syncthreads();
    for (int i = 0; i < per; ++i) amax = fmaxf(amax, peak[token * per + i]);
    const float sc = quant_scale(amax), inv = quant_inv(sc);
    if (warp % per == 0 && lane == 0) scales[token] = sc;
    uint8_t* q = smem + token * p.pitch;
    for (int c = share; c < chunks; c += step) {
      struct alignas(E) Out {
        int8_t b[E];
      } u;
      float f[E];
      if (token < p.m) {
        read(c, f);
#pragma unroll
        for (int j = 0; j < E; ++j) u.b[j] = (int8_t)quant1_bounded(f[j], inv);
        *reinterpret_cast<Out*>(q + c * E) = u;
      }
    }
  }
  __syncthreads();

  const uint8_t* xq = smem + min(gr, p.m - 1) * p.pitch + t4 * 16;
  const bool has = gr < p.m;
  {
    const int64_t row0 = (int64_t)tile * 16 + gr;
    int32_t d[4] = {0, 0, 0, 0};
    for (int s = warp; s < steps; s += U * kSkinnyWarps) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int now = s + u * kSkinnyWarps;
        const uint4 a = w0[u], b = w1[u];
        const int then = now + U * kSkinnyWarps;  // the step that takes these registers next
        if (then < steps) {
          w0[u] = load_w(row0, then);
          w1[u] = load_w(row0 + 8, then);
        }
        if (now * 64 < ld) {
          const uint4 v = has && now * 64 + t4 * 16 < ld ? *reinterpret_cast<const uint4*>(xq + now * 64) : zero;
          mma_i8_16832(d, a.x, b.x, a.y, b.y, v.x, v.y);
          mma_i8_16832(d, a.z, b.z, a.w, b.w, v.z, v.w);
        }
      }
    }
    // Not before: blocks of a launch placed among these would sit unevenly on the SMs (one token
    // through 4096 -> 4096 back to back: 11.1 us with the trigger at the start, 8.3 here).
    grid_launch_dependents();
    // d: rows gr and gr + 8, tokens 2 t4 and 2 t4 + 1
    *reinterpret_cast<int2*>(&part[warp][gr][2 * t4]) = make_int2(d[0], d[1]);
    *reinterpret_cast<int2*>(&part[warp][gr + 8][2 * t4]) = make_int2(d[2], d[3]);
    __syncthreads();
    if (tid < 128) {
      const int r = tid & 15, t = tid >> 4;
      const int64_t n = (int64_t)tile * 16 + r;
      if (t < p.m && n < g.n) {
        int32_t sum = 0;
#pragma unroll
        for (int i = 0; i < kSkinnyWarps; ++i) sum += part[i][r][t];
        const float y = dequant(sum, __fmul_rn(scales[t], g.w_scale[n]), g.bias ? g.bias[n] : 0.0f);
        static_cast<TO*>(g.out)[t * g.ldo + n] =
            ElemOf<TO>::from(sizeof(TO) == 2 && g.act == ACT_GELU   ? smooth16<true>(y)
                             : sizeof(TO) == 2 && g.act == ACT_SILU ? smooth16<false>(y)
                                                                    : act_apply(g.act, g.act_param, y));
      }
    }
  }
}

template <typename TX, typename TO>
rg_status go_skinny(const TokenGemmArgs& a, const void* x, int64_t k, int64_t ldx, cudaStream_t st) {
  SkinnyParams p;
  p.g = a;
  p.x = x;
  p.ldx = ldx;
  p.k = (int32_t)k;
  p.m = (int32_t)a.m;
  p.pitch = (int32_t)a.ld + 16;
  p.vec = (((uintptr_t)x | (uintptr_t)(ldx * (int64_t)sizeof(TX))) & 15) == 0;
  launch_early(k_linear_skinny<TX, TO>, dim3((unsigned)((a.n + 15) / 16)), kSkinnyThreads, p.m * p.pitch, st, p);
  return RG_OK;
}

template <typename TX>
rg_status go_skinny_out(const TokenGemmArgs& a, const void* x, int64_t k, int64_t ldx, cudaStream_t st) {
  if (a.out_dtype == RG_DTYPE_F32) return go_skinny<TX, float>(a, x, k, ldx, st);
  return a.out_dtype == RG_DTYPE_F16 ? go_skinny<TX, __half>(a, x, k, ldx, st)
                                     : go_skinny<TX, __nv_bfloat16>(a, x, k, ldx, st);
}

bool operand_map(CUtensorMap* map, const void* base, int64_t rows, int64_t ld, int box_rows) {
  const auto fn = tma_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)ld, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
bool output_map(CUtensorMap* map, const TokenGemmArgs& a) {
  const auto fn = tma_encode_fn();
  if (!fn || ((uintptr_t)a.out & 15) || (a.ldo * (int64_t)sizeof(T)) & 15) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)a.n, (cuuint64_t)a.m}, strides[1] = {(cuuint64_t)a.ldo * sizeof(T)};
  const cuuint32_t box[2] = {64 / sizeof(T), 32}, one[2] = {1, 1};
  const auto type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  return fn(map, type, 2, a.out, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, typename T>
rg_status go_pair(const TokenGemmArgs& a, cudaStream_t st) {
  const auto kernel = k_gemm_token_pair<BN, T>;
  static DeviceOnce once;
  once.run([&] { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem); });
  CUtensorMap ma, mw, mo;
  PairParams p;
  p.a_rows = a.m >= 128 ? 128 : (int32_t)((a.m + 7) / 8 * 8);
  p.a_ctas = a.m > 128 ? 2 : 1;
  p.stage_bytes = (p.a_rows + BN / 2) * kBK;
  p.stages = std::min(kMaxStages, kRing / p.stage_bytes);
  if (!operand_map(&ma, a.a, a.m, a.ld, p.a_rows) || !operand_map(&mw, a.w, a.n, a.ld, BN / 2)) return RG_ERR_CUDA;
  memset(&mo, 0, sizeof mo);
  p.g = a;
  p.tma_store = output_map<T>(&mo, a);
  const int64_t tm = (a.m + 255) / 256, tn = (a.n + BN - 1) / BN;
  if (tm * tn > INT_MAX) return RG_ERR_UNSUPPORTED;
  p.tiles_m = (int32_t)tm;
  p.tiles_n = (int32_t)tn;
  p.num_kb = (int32_t)((a.ld + kBK - 1) / kBK);
  p.group_m = 16;
  p.wait_ns = a.wait_ns ? a.wait_ns : kWaitNs;
  p.starve = a.starve == 1;
  const int pairs = (int)std::min<int64_t>(tm * tn, 74);
  launch_early(kernel, dim3(2 * pairs), kGemmThreads, kGemmSmem, st, ma, mw, mo, p);
  return RG_OK;
}

template <typename T>
rg_status go_few(const TokenGemmArgs& a, cudaStream_t st) {
  const int tokens = (int)a.m;
  const auto kernel = k_gemm_token_few<T>;
  static DeviceOnce once;
  once.run([&] { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024); });
  FewParams p;
  p.g = a;
  p.box_rows = (tokens + 7) / 8 * 8;
  p.n_cols = (tokens + 15) / 16 * 16;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.n_cols) p.tmem_cols *= 2;
  p.stage_bytes = (128 + p.box_rows) * kBK;
  // up to 64 tokens two CTAs share an SM, beyond one has it alone; 1 KB behind the ring is read
  // (not used) by a product whose tokens are no multiple of 16
  const int slots = tokens <= 64 ? 2 * 148 : 148;
  p.stages = std::min(kFewStages, (tokens <= 64 ? 96 : 192) * 1024 / p.stage_bytes);
  p.ring = p.stages * p.stage_bytes + 1024;
  p.num_kb = (int32_t)((a.ld + kBK - 1) / kBK);
  const int64_t tn = (a.n + 127) / 128;
  p.splits = 1;  // as many as find an SM, each with two steps of K at least
  while (p.splits < 8 && tn * p.splits * 2 <= slots && p.num_kb >= p.splits * 4) p.splits *= 2;
  if (tn * p.splits > INT_MAX) return RG_ERR_UNSUPPORTED;
  p.wait_ns = a.wait_ns ? a.wait_ns : kWaitNs;
  p.starve = a.starve;
  p.vec_out = (((uintptr_t)a.out | (uintptr_t)(a.ldo * (int64_t)sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
  CUtensorMap mw, ma;
  if (!operand_map(&mw, a.w, a.n, a.ld, 128) || !operand_map(&ma, a.a, a.m, a.ld, p.box_rows)) return RG_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tn * p.splits));
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = 1024 + p.ring + 512;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (p.splits > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = p.splits;
    attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
    ++na;
  }
  attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[na].val.programmaticStreamSerializationAllowed = 1;
  ++na;
  cfg.attrs = attr;
  cfg.numAttrs = na;
  cudaLaunchKernelEx(&cfg, kernel, mw, ma, p);
  return RG_OK;
}

// Narrower tiles where wider ones would leave SMs idle: the time of a launch is the number of
// rounds over the 74 pairs times the tile's width.
template <typename T>
rg_status go_gemm(const TokenGemmArgs& a, cudaStream_t st) {
  // Few tokens against pairs, us: 10.1 / 15.7 at 17 x 4096 x 4096, 12.5 / 16.0 at 64, 14.6 / 17.3 at 128;
  // 18.6 / 20.8 at 64 x 4096 x 14336, 24.6 / 22.2 at 128; 10.3 / 8.1 at 128 x 1024 x 1024.  One limit
  // for all widths: above it wide and short layers gain, layers like 4096 x 4096 lose (11.9 us at 96
  // tokens, 16.5 at 97).
  if (a.m <= 96) return go_few<T>(a, st);
  const auto cost = [&](int64_t bn) { return ((a.m + 255) / 256 * ((a.n + bn - 1) / bn) + 73) / 74 * (bn + 96); };
  if (cost(256) <= cost(128) && cost(256) <= cost(64)) return go_pair<256, T>(a, st);
  return cost(128) <= cost(64) ? go_pair<128, T>(a, st) : go_pair<64, T>(a, st);
}

}  // namespace

void launch_quantize_token(const void* x, int32_t dtype, int64_t rows, int64_t k, int64_t ldx, int8_t* q, int64_t ldq,
                           float* scale, cudaStream_t st) {
  if (dtype == RG_DTYPE_F32) quantize<float>(x, rows, k, ldx, q, ldq, scale, st);
  else if (dtype == RG_DTYPE_F16) quantize<__half>(x, rows, k, ldx, q, ldq, scale, st);
  else quantize<__nv_bfloat16>(x, rows, k, ldx, q, ldq, scale, st);
}

bool linear_skinny_takes(int64_t m, int64_t n, int64_t ld) {
  return m <= kSkinnyTokens && m * ld <= kSkinnyValues && n <= 16 * kSkinnyBlocks;
}

rg_status launch_linear_skinny(const TokenGemmArgs& a, const void* x, int32_t dtype, int64_t k, int64_t ldx,
                               cudaStream_t st) {
  if (dtype == RG_DTYPE_F32) return go_skinny_out<float>(a, x, k, ldx, st);
  return dtype == RG_DTYPE_F16 ? go_skinny_out<__half>(a, x, k, ldx, st)
                               : go_skinny_out<__nv_bfloat16>(a, x, k, ldx, st);
}

rg_status launch_gemm_token(const TokenGemmArgs& a, cudaStream_t st) {
  if (a.out_dtype == RG_DTYPE_F32) return go_gemm<float>(a, st);
  return a.out_dtype == RG_DTYPE_F16 ? go_gemm<__half>(a, st) : go_gemm<__nv_bfloat16>(a, st);
}

}  // namespace rg

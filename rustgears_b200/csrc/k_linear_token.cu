// k_linear_token.cu -- i8 x i8 product with one scale per token and one per output channel:
//   sa[r] = absmax(x[r]) < 1e-12 ? 1 : absmax / 127,  q = clamp(round(x / sa)),
//   out[r, c] = act(f32(sum_k q[r,k] w[c,k]) * (sa[r] * sw[c]) + bias[c]).
#include <climits>

#include "rg_math.cuh"
#include "rg_serving.h"

namespace rg {
namespace {

constexpr int kQuantThreads = 256;

// ---------------------------------------------------------------------------
// Row quantizer.  Bound: memory (x read once, q and the scales written once).  One block
// per row; the row stays in registers between its absmax and its rounding (up to 32
// values a thread, 8192 a row), longer rows are read again, from L1 or L2.
// ---------------------------------------------------------------------------
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads)
    k_quantize_token(const T* __restrict__ x, int64_t k, int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                     float* __restrict__ scale) {
  constexpr int E = VEC ? 16 / (int)sizeof(T) : 4;  // values a thread handles at once
  constexpr int NREG = 32 / E;
  __shared__ float red[kQuantThreads / 32];
  const int64_t r = blockIdx.x;
  x += r * ldx;
  q += r * ldq;
  const int64_t chunks = ldq / E;
  float keep[NREG][E];
  const auto read = [&](int64_t c, float (&f)[E]) {
    const int64_t at = c * E;
    if (VEC && at + E <= k) {
      Pack<T, E>::load(x + at, f);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = at + j < k ? ElemOf<T>::to(x[at + j]) : 0.0f;
    }
  };
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < NREG; ++i) {
    const int64_t c = threadIdx.x + (int64_t)i * kQuantThreads;
    if (c < chunks) {
      read(c, keep[i]);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) keep[i][j] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < NREG; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) amax = fmaxf(amax, fabsf(keep[i][j]));
  for (int64_t c = threadIdx.x + (int64_t)NREG * kQuantThreads; c < chunks; c += kQuantThreads) {
    float f[E];
    read(c, f);
#pragma unroll
    for (int j = 0; j < E; ++j) amax = fmaxf(amax, fabsf(f[j]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantThreads / 32; ++i) amax = fmaxf(amax, red[i]);
  const float sc = quant_scale(amax), inv = quant_inv(sc);
  if (threadIdx.x == 0) scale[r] = sc;
  const auto write = [&](int64_t c, const float (&f)[E]) {
    union {
      int8_t b[E];
      uint32_t w[E / 4];
    } u;
#pragma unroll
    for (int j = 0; j < E; ++j) u.b[j] = (int8_t)quant1_bounded(f[j], inv);
#pragma unroll
    for (int j = 0; j < E / 4; ++j) reinterpret_cast<uint32_t*>(q + c * E)[j] = u.w[j];
  };
#pragma unroll
  for (int i = 0; i < NREG; ++i) {
    const int64_t c = threadIdx.x + (int64_t)i * kQuantThreads;
    if (c < chunks) write(c, keep[i]);
  }
  for (int64_t c = threadIdx.x + (int64_t)NREG * kQuantThreads; c < chunks; c += kQuantThreads) {
    float f[E];
    read(c, f);
    write(c, f);
  }
}

template <typename T>
void quantize(const void* x, int64_t rows, int64_t k, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
              cudaStream_t st) {
  const bool vec = (((uintptr_t)x | (uintptr_t)(ldx * (int64_t)sizeof(T))) & 15) == 0;
  const T* p = static_cast<const T*>(x);
  if (vec) k_quantize_token<T, true><<<(unsigned)rows, kQuantThreads, 0, st>>>(p, k, ldx, q, ldq, scale);
  else k_quantize_token<T, false><<<(unsigned)rows, kQuantThreads, 0, st>>>(p, k, ldx, q, ldq, scale);
}

// ---------------------------------------------------------------------------
// Product: 64 x 64 tiles on the CUDA cores (dp4a), any size.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void put(void* out, int64_t i, float v) {
  static_cast<T*>(out)[i] = ElemOf<T>::from(v);
}

template <typename T>
__global__ void __launch_bounds__(256) k_gemm_token(const TokenGemmArgs p) {
  __shared__ int32_t sa[64][17], sw[64][17];  // 64 bytes of K
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  int32_t acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.ld; k0 += 64) {
    const int r = threadIdx.x >> 2, c = threadIdx.x & 3;
    const bool in_k = k0 + c * 16 < p.ld;
    const int4 z = make_int4(0, 0, 0, 0);
    const int4 va = in_k && m0 + r < p.m ? *reinterpret_cast<const int4*>(p.a + (m0 + r) * p.ld + k0 + c * 16) : z;
    const int4 vw = in_k && n0 + r < p.n ? *reinterpret_cast<const int4*>(p.w + (n0 + r) * p.ld + k0 + c * 16) : z;
    __syncthreads();
    sa[r][c * 4] = va.x; sa[r][c * 4 + 1] = va.y; sa[r][c * 4 + 2] = va.z; sa[r][c * 4 + 3] = va.w;
    sw[r][c * 4] = vw.x; sw[r][c * 4 + 1] = vw.y; sw[r][c * 4 + 2] = vw.z; sw[r][c * 4 + 3] = vw.w;
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sa[ty + 16 * i][kk], sw[tx + 16 * j][kk], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = m0 + ty + 16 * i;
    if (r >= p.m) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = n0 + tx + 16 * j;
      if (c >= p.n) continue;
      const float cs = __fmul_rn(p.a_scale[r], p.w_scale[c]);
      put<T>(p.out, r * p.ldo + c, epilogue(acc[i][j], cs, p.bias ? p.bias[c] : 0.0f, p.act, p.act_param));
    }
  }
}

}  // namespace

void launch_quantize_token(const void* x, int32_t dtype, int64_t rows, int64_t k, int64_t ldx, int8_t* q, int64_t ldq,
                           float* scale, cudaStream_t st) {
  if (dtype == RG_DTYPE_F32) quantize<float>(x, rows, k, ldx, q, ldq, scale, st);
  else if (dtype == RG_DTYPE_F16) quantize<__half>(x, rows, k, ldx, q, ldq, scale, st);
  else quantize<__nv_bfloat16>(x, rows, k, ldx, q, ldq, scale, st);
}

rg_status launch_gemm_token(const TokenGemmArgs& a, cudaStream_t st) {
  const int64_t gy = (a.m + 63) / 64, gx = (a.n + 63) / 64;
  if (gy > 65535 || gx > INT_MAX) return RG_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (a.out_dtype == RG_DTYPE_F32) k_gemm_token<float><<<grid, 256, 0, st>>>(a);
  else if (a.out_dtype == RG_DTYPE_F16) k_gemm_token<__half><<<grid, 256, 0, st>>>(a);
  else k_gemm_token<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  return RG_OK;
}

}  // namespace rg

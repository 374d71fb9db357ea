// rg_serving.h -- launchers of the decoder-serving kernels (internal to librg_npu.so) and
// the element types they share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <utility>

#include "../../include/rg_npu.h"

namespace rg {

// The serving kernels are launched so that each may start while the launch before it ends: its
// blocks are placed and set up early, then wait.  Every kernel begins with grid_dependency_wait
// (before it reads or writes anything another launch may have written or read) and lets the next
// one start only after it, so that whatever ran earlier in the stream is over by then too.  (The
// product that follows its own quantizer reads W before it waits, and the chunk kernel beside the
// one for few rows waits at its end: see there.)
// So a kernel's life begins while what it reads is still being written.  Its loads are therefore
// plain ones: never the read-only path (__ldg, or const __restrict__ parameters), which promises
// data that is constant for the whole launch and lets a load be moved above the wait.
template <typename... P, typename... A>
inline void launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}
// Waits for the launch before this one and for its writes.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the launch after this one start.
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Runs a kernel's set-up once on every device (a function attribute belongs to the device
// that was current).
class DeviceOnce {
 public:
  template <typename F>
  void run(F f) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev > 63) return f();
    const uint64_t bit = 1ull << dev;
    if (done_.load(std::memory_order_acquire) & bit) return;
    f();
    done_.fetch_or(bit, std::memory_order_release);
  }

 private:
  std::atomic<uint64_t> done_{0};
};

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

inline int dtype_size(int32_t dt) { return dt == RG_DTYPE_F32 ? 4 : 2; }

template <typename T>
struct ElemOf;  // conversions to and from f32, one rounding each (none widening)
template <>
struct ElemOf<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct ElemOf<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct ElemOf<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// N consecutive elements as f32, moved 16 bytes at a time (or all at once when shorter):
// the address is aligned to min(16, N * sizeof(T)).
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = N * (int)sizeof(T);
  static constexpr int kWord = kBytes >= 16 ? 16 : kBytes;
  struct alignas(kWord) Word {
    T e[kWord / (int)sizeof(T)];
  };
  static constexpr int kPer = kWord / (int)sizeof(T);
  static __device__ __forceinline__ void load(const T* p, float (&f)[N]) {
#pragma unroll
    for (int w = 0; w < N / kPer; ++w) {
      const Word v = reinterpret_cast<const Word*>(p)[w];
#pragma unroll
      for (int i = 0; i < kPer; ++i) f[w * kPer + i] = ElemOf<T>::to(v.e[i]);
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[N]) {
#pragma unroll
    for (int w = 0; w < N / kPer; ++w) {
      Word v;
#pragma unroll
      for (int i = 0; i < kPer; ++i) v.e[i] = ElemOf<T>::from(f[w * kPer + i]);
      reinterpret_cast<Word*>(p)[w] = v;
    }
  }
};

// ---- per-token linear (k_linear_token.cu) ---------------------------------------
void launch_quantize_token(const void* x, int32_t dtype, int64_t rows, int64_t k, int64_t ldx, int8_t* q, int64_t ldq,
                           float* scale, cudaStream_t st);
struct TokenGemmArgs {
  const int8_t* a = nullptr;       // [m, ld]
  const float* a_scale = nullptr;  // [m]
  const int8_t* w = nullptr;       // [n, ld]
  const float* w_scale = nullptr;  // [n]
  const float* bias = nullptr;     // [n] or NULL
  int64_t m = 0, n = 0, ld = 0, ldo = 0;
  int32_t act = 0;
  float act_param = 0.0f;
  void* out = nullptr;
  int32_t out_dtype = 0;
  int32_t* err = nullptr;
  uint64_t wait_ns = 0;  // limit of every pipeline wait (0: the default)
  int32_t after_quantizer = 0;  // a and a_scale come from the quantizer launched just before
  int32_t starve = 0;    // test hook: 1 issue no operand loads, so the waits run out; 2 give the products up at once
};
rg_status launch_gemm_token(const TokenGemmArgs& a, cudaStream_t st);
// Quantizer and product in one launch for a few tokens (a, a_scale unused).
bool linear_skinny_takes(int64_t m, int64_t n, int64_t ld);
rg_status launch_linear_skinny(const TokenGemmArgs& a, const void* x, int32_t dtype, int64_t k, int64_t ldx,
                               cudaStream_t st);

// ---- rotary positions and the paged append (k_rope.cu) --------------------------
// Three groups of heads per token: q heads (rotated, stored by strides), then kv_heads
// key heads (rotated, stored in the cache) and kv_heads value heads (copied there).
struct RopeArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr;
  int64_t q_ts = 0, q_hs = 0, k_ts = 0, k_hs = 0, v_ts = 0, v_hs = 0;
  void *q_out = nullptr, *k_out = nullptr, *v_out = nullptr;
  int64_t qo_ts = 0, qo_hs = 0, page_stride = 0, token_stride = 0, head_stride = 0;
  const int32_t* positions = nullptr;
  const float* table = nullptr;
  const int64_t* slots = nullptr;
  int64_t table_rows = 0, tokens = 0, num_slots = 0;
  int32_t heads = 0, kv_heads = 0, head_dim = 0, rot_dim = 0, page_size = 1;
  int32_t in_dtype = 0, out_dtype = 0, interleaved = 0;
  int32_t* err = nullptr;
};
rg_status launch_rope(const RopeArgs& a, cudaStream_t st);
void launch_rope_table(const rg_rope_scaling& s, int64_t positions, int32_t rot_dim, float* table, cudaStream_t st);

// ---- attention over a paged cache (k_attn_paged.cu) ------------------------------
struct PagedAttnArgs {
  rg_kv_cache c;
  rg_paged_attention_args a;
  void* workspace = nullptr;
  int32_t* err = nullptr;
  uint64_t wait_ns = 0;  // as TokenGemmArgs
  int32_t starve = 0;
};
int64_t attention_paged_workspace(const PagedAttnArgs& a);
rg_status launch_attention_paged(const PagedAttnArgs& a, cudaStream_t st);

}  // namespace rg

// k_rope.cu -- rotary positions and the append to a paged key / value cache.
//
// For pair i of a head, with the table row's cosine c and sine s of the token's position:
//   (a, b) -> (a c - b s, b c + a s),
// a and b being dimensions (i, i + rot / 2) or, interleaved, (2 i, 2 i + 1); dimensions
// from rot on are copied.  Sums in f32 (two products, one addition, each rounded), one
// rounding to the output's type.  The append runs the same work over one token's query,
// key and value heads and stores keys and values through the token's slot, so rotating q
// and k and writing the cache is one launch.
//
// Bound: memory (every element is read and written once; a table row of 4 rot bytes per
// token is shared by its heads and stays in L1).  One thread moves P pairs: P elements from
// each of two places (half layout) or 2 P consecutive ones, P elements filling a 16-byte
// access, so a warp's accesses are whole 128-byte lines; resident threads, not unrolling,
// keep the loads in flight.  Measured: 16384 tokens x 32 heads of 128, f32, 64 dimensions rotated
// 87 us (6.2 TB/s of 541 MB); append of 8192 tokens, 16 heads of 64, f32 to f16 27.5 us (5.5 TB/s);
// 64 tokens 2.2 us, one token 1.8 us (a launch).
#include <climits>

#include "rg_serving.h"

namespace rg {
namespace {

constexpr int kThreads = 256;

template <typename TI, typename TO, int P, bool INTER>
__global__ void __launch_bounds__(kThreads)
    k_rope(const RopeArgs a, int32_t tokens_per_block, FastDiv per_token, FastDiv units, FastDiv page_size) {
  // units: work items of one head (rot / 2P rotations, then (head_dim - rot) / 2P copies);
  // per_token: those of all heads
  grid_dependency_wait();
  grid_launch_dependents();
  const int i = blockIdx.y * kThreads + threadIdx.x;
  const int within = (int)per_token.div((uint32_t)i);
  if (within >= tokens_per_block) return;
  const int64_t t = (int64_t)blockIdx.x * tokens_per_block + within;
  if (t >= a.tokens) return;
  const int rem = i - within * (int)per_token.d;
  int h = (int)units.div((uint32_t)rem);
  const int u = rem - h * (int)units.d;

  const TI* src;
  TO* dst;
  int64_t pos = 0;
  if (a.table) {
    pos = a.positions[t];
    if (pos < 0 || pos >= a.table_rows) {
      a.err[1] = 1;
      return;
    }
  }
  bool rotate = u < a.rot_dim / (2 * P);
  if (h < a.heads) {
    src = static_cast<const TI*>(a.q) + t * a.q_ts + h * a.q_hs;
    dst = static_cast<TO*>(a.q_out) + t * a.qo_ts + h * a.qo_hs;
  } else {
    h -= a.heads;
    const int64_t slot = a.slots[t];
    if (slot < 0) return;
    if (slot >= a.num_slots) {
      a.err[1] = 1;
      return;
    }
    const int64_t page = slot <= INT_MAX ? (int64_t)page_size.div((uint32_t)slot) : slot / a.page_size;
    const int64_t off = slot - page * a.page_size;
    const bool value = h >= a.kv_heads;
    if (value) h -= a.kv_heads;
    src = value ? static_cast<const TI*>(a.v) + t * a.v_ts + h * a.v_hs
                : static_cast<const TI*>(a.k) + t * a.k_ts + h * a.k_hs;
    dst = static_cast<TO*>(value ? a.v_out : a.k_out) + page * a.page_stride + off * a.token_stride + h * a.head_stride;
    rotate = rotate && !value;
  }
  // the two groups of P elements this thread moves
  const bool halves = rotate && !INTER;
  const int at0 = halves ? u * P : u * 2 * P;
  const int at1 = halves ? u * P + a.rot_dim / 2 : u * 2 * P + P;
  float x0[P], x1[P];
  Pack<TI, P>::load(src + at0, x0);
  Pack<TI, P>::load(src + at1, x1);
  if (rotate) {
    float c[P], s[P];
    const float* row = a.table + pos * a.rot_dim + u * P;
    Pack<float, P>::load(row, c);
    Pack<float, P>::load(row + a.rot_dim / 2, s);
    if constexpr (INTER) {
      float x[2 * P];
#pragma unroll
      for (int j = 0; j < P; ++j) {
        x[j] = x0[j];
        x[P + j] = x1[j];
      }
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float p = x[2 * j], q = x[2 * j + 1];
        x[2 * j] = p * c[j] - q * s[j];
        x[2 * j + 1] = q * c[j] + p * s[j];
      }
#pragma unroll
      for (int j = 0; j < P; ++j) {
        x0[j] = x[j];
        x1[j] = x[P + j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float p = x0[j], q = x1[j];
        x0[j] = p * c[j] - q * s[j];
        x1[j] = q * c[j] + p * s[j];
      }
    }
  }
  Pack<TO, P>::store(dst + at0, x0);
  Pack<TO, P>::store(dst + at1, x1);
}

// P pairs per thread need: whole units of the rotated and the copied part, and addresses
// aligned to the accesses of P elements in both types.
bool takes(const RopeArgs& a, int P) {
  if (a.rot_dim % (2 * P) || a.head_dim % (2 * P)) return false;
  const int si = dtype_size(a.in_dtype), so = dtype_size(a.out_dtype);
  const auto in_ok = [&](const void* p, int64_t ts, int64_t hs) {
    const int b = P * si < 16 ? P * si : 16;
    return p == nullptr || (((uintptr_t)p | (uintptr_t)(ts * si) | (uintptr_t)(hs * si)) & (b - 1)) == 0;
  };
  const auto out_ok = [&](const void* p, int64_t ts, int64_t hs) {
    const int b = P * so < 16 ? P * so : 16;
    return p == nullptr || (((uintptr_t)p | (uintptr_t)(ts * so) | (uintptr_t)(hs * so)) & (b - 1)) == 0;
  };
  const int tb = P * 4 < 16 ? P * 4 : 16;
  return in_ok(a.q, a.q_ts, a.q_hs) && in_ok(a.k, a.k_ts, a.k_hs) && in_ok(a.v, a.v_ts, a.v_hs) &&
         out_ok(a.q_out, a.qo_ts, a.qo_hs) && out_ok(a.k_out, a.page_stride | a.token_stride, a.head_stride) &&
         out_ok(a.v_out, a.page_stride | a.token_stride, a.head_stride) && ((uintptr_t)a.table & (tb - 1)) == 0;
}

template <typename TI, typename TO, int P>
rg_status go(const RopeArgs& a, cudaStream_t st) {
  const int units = a.head_dim / (2 * P);
  const int64_t per_token = (int64_t)(a.heads + 2 * a.kv_heads) * units;
  if (per_token > (int64_t)kThreads * 65535) return RG_ERR_UNSUPPORTED;
  // short tokens share a block
  const int tpb = per_token >= kThreads ? 1 : (int)(kThreads / per_token);
  const int64_t blocks = (a.tokens + tpb - 1) / tpb;
  if (blocks > INT_MAX) return RG_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks, (unsigned)((tpb * per_token + kThreads - 1) / kThreads));
  const FastDiv by_token((uint32_t)per_token), by_head((uint32_t)units), by_page((uint32_t)a.page_size);
  if (a.interleaved) launch_early(k_rope<TI, TO, P, true>, grid, kThreads, 0, st, a, tpb, by_token, by_head, by_page);
  else launch_early(k_rope<TI, TO, P, false>, grid, kThreads, 0, st, a, tpb, by_token, by_head, by_page);
  return RG_OK;
}

template <typename TI, typename TO>
rg_status go_types(const RopeArgs& a, cudaStream_t st) {
  if constexpr (sizeof(TI) == 2)
    if (takes(a, 8)) return go<TI, TO, 8>(a, st);
  if (takes(a, 4)) return go<TI, TO, 4>(a, st);
  return go<TI, TO, 1>(a, st);
}

// Angles in 64 bits: at position 10^5 the f32 product position * freq is off by up to 2^-8.
__global__ void k_rope_table(const rg_rope_scaling s, int64_t positions, int32_t rot, float* table) {
  const int half = rot / 2;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= positions * half) return;
  const int64_t p = i / half;
  const int d = (int)(i - p * half);
  double f = pow(s.base, -2.0 * d / rot);
  if (s.kind == RG_ROPE_LINEAR) {
    f /= s.factor;
  } else if (s.kind == RG_ROPE_BANDS) {
    // the dimension that turns n times within old_context: base^(-2 d / rot) old_context = 2 pi n
    const double pi = 3.14159265358979323846, lb = 2.0 * log(s.base);
    const double lo = fmax(0.0, floor(rot * log(s.old_context / (s.fast_turns * 2.0 * pi)) / lb));
    const double hi = fmin(rot - 1.0, ceil(rot * log(s.old_context / (s.slow_turns * 2.0 * pi)) / lb));
    const double ramp = fmin(1.0, fmax(0.0, (d - lo) / fmax(hi - lo, 1e-3)));
    f = f / s.factor * ramp + f * (1.0 - ramp);
  }
  double sn, cs;
  sincos((double)p * f, &sn, &cs);
  table[p * rot + d] = (float)(cs * s.gain);
  table[p * rot + half + d] = (float)(sn * s.gain);
}

}  // namespace

rg_status launch_rope(const RopeArgs& a, cudaStream_t st) {
  if (a.in_dtype == RG_DTYPE_F32) {
    if (a.out_dtype == RG_DTYPE_F32) return go_types<float, float>(a, st);
    if (a.out_dtype == RG_DTYPE_F16) return go_types<float, __half>(a, st);
    return go_types<float, __nv_bfloat16>(a, st);
  }
  if (a.in_dtype == RG_DTYPE_F16) return go_types<__half, __half>(a, st);
  return go_types<__nv_bfloat16, __nv_bfloat16>(a, st);
}

void launch_rope_table(const rg_rope_scaling& s, int64_t positions, int32_t rot_dim, float* table, cudaStream_t st) {
  const int64_t n = positions * (rot_dim / 2);
  k_rope_table<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(s, positions, rot_dim, table);
}

}  // namespace rg

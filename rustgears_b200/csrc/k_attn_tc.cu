// k_attn_tc.cu -- attention of a chunk of new tokens over a paged cache on the 5th-generation
// tensor cores (the formulas: k_attn_paged.cu), for sequences of many rows.
//
// A block takes 256 rows (two groups of 128) of one (sequence, key head), row r = token
// r / group, head r % group, and walks the sequence's keys in tiles of 128:
//   S_g = Q_g K^T   tcgen05, both operands in shared memory, S in TMEM (128 columns a group)
//   P_g = 2^(S_g scale2 - m), rounded to the cache's type (both operands of a product have
//                   one type; the row sum adds P unrounded), written over S_g in TMEM
//   O_g += P_g V    tcgen05, P from TMEM, V from shared memory as it was loaded (keys are the
//                   product's K dimension: V is the "transposed" operand), O in TMEM
// One thread per row does the softmax, so a row's maximum and sum need no exchange; its 128
// scores take 224 registers, which the control warps give up.  (Two threads per row on half the
// keys each, 16 warps: 498 against 474 us at D = 128, 454 against 478 at D = 64.)  While one
// group's exponentials run, the tensor cores work on the other group.  A new maximum rescales
// O only when it exceeds the one in use by 2^8 (the sums stay exact: numerator and denominator
// use the same m; 2^8 fits every type here), so O is almost never read back.
//
// Bound: per 128 x 128 tile and group 2 x 128 x 128 x D products (1024 clocks of the tensor
// pipe at D = 128) against 16384 exponentials (1024 clocks of the SM's 16 a clock): both pipes
// are full at once at best, 2048 clocks for both groups.  Measured 3300: a group's chain of load
// (95 clocks), maximum (320), exponentials (1430), store and arrival (150), then its products, is
// longer than twice the tensor time.  2048 new tokens over 16384 keys, 32 query heads on 8 of 128:
// 478 to 509 us from run to run, 1077 to 1013 TFLOP/s (the power cap; 256 blocks on 148 SMs: two
// rounds where 1.73 have work).  Every fourth
// pair of exponentials as a polynomial on the FMA pipes: 545 us, not kept.
//   warp 0     TMA: a page's part of a tile is one box per 64 dimensions (page sizes that
//              divide 128 or are multiples of it), so a tile arrives swizzled whatever its pages
//   warp 1     issues the products
//   warp 2     zeroes V rows past the last key (a probability of 0 times NaN is NaN)
//   warps 4-11 softmax and output, one warp per 32 TMEM lanes of a group
// Every wait is bounded.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cfloat>
#include <climits>
#include <cstring>

#include "rg_attn.h"
#include "rg_f32x2.cuh"
#include "rg_mma16.cuh"
#include "rg_sm100_pair.cuh"

namespace rg {

PFN_cuTensorMapEncodeTiled_v12000 tma_encode_fn();  // k_gemm_tc.cu

namespace {

using namespace sm100;

constexpr int kThreads = 384;
constexpr int kTile = kTcKeys;  // keys of a tile, rows of a group
constexpr uint64_t kWaitNs = 2000000000ull, kDrainNs = 200000000ull;
constexpr float kLazy = 8.0f;

template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;                  // 128-byte wide sub-tiles
  static constexpr int kOperand = kTile * D * 2;          // bytes of a K, V or Q tile
  static constexpr int kSub = kTile * 128;                // bytes of a sub-tile
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kSmem = 1024 + 2 * kOperand + kStages * kOperand + 512;
  static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
};

struct TcParams {
  AttnParams P;
  int32_t page_log2;      // page size as a power of two, or -1: a multiple of 128
  int32_t box;            // tokens of a box: min(page size, 128)
  float scale2;           // |scale| log2(e); a negative scale turns Q's signs
  uint32_t flip;          // sign bits to flip in a pair of Q's values
  uint64_t wait_ns;
  int32_t starve;
  // The launch before is the kernel for few rows, which this one does not depend on: it waits
  // for it at its end only.  (That kernel's blocks waited until whatever ran before the call was
  // over, and this launch starts when all of them have come further.  This one has not waited
  // itself, so nothing it reads comes through L1, which might be older: TMA, and __ldcg.)
  int32_t beside;
};

// Instruction descriptor of tcgen05.mma kind::f16: f32 sums, A and B of one 16-bit type, B
// K-major or (b_mn) MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_16(int m, int n, bool b_mn) {
  const uint32_t f = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
// MN-major operand in the 128-byte swizzle layout: 64 MN-elements x 8 K-rows per 1024-byte
// atom, the next 8 K-rows 1024 bytes on, the next 64 MN-elements `mn_stride` bytes on.
__device__ __forceinline__ uint64_t desc_mnmajor_sw128(uint32_t saddr, uint32_t mn_stride) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(mn_stride >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    k_attn_tc(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TcParams p) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * C::kOperand;  // behind the two groups' queries
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + C::kStages * C::kOperand);
  uint64_t* empty = full + C::kStages;
  uint64_t* s_full = empty + C::kStages;  // [2] S (and every earlier product) done
  uint64_t* p_ready = s_full + 2;         // [2] P written, S read
  uint64_t* q_ready = p_ready + 2;
  uint64_t* v_here = q_ready + 1;   // the last V tile has landed
  uint64_t* v_fixed = v_here + 1;   // ... and its rows past the last key are zeros
  uint64_t* done = v_fixed + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const rg_kv_cache& c = p.P.p.c;
  const rg_paged_attention_args& a = p.P.p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int hk = blockIdx.y, b = blockIdx.z, group = (int)p.P.group.d;
  if (!p.beside) grid_dependency_wait();
  grid_launch_dependents();

  const int64_t q0 = __ldcg(a.cu_q + b), q1 = __ldcg(a.cu_q + b + 1);
  const int kv = __ldcg(a.kv_len + b);
  if (q0 < 0 || q1 < q0 || q1 > a.tokens || q1 - q0 > a.max_q_len || kv < 0 || kv > a.max_kv_len) {
    if (threadIdx.x == 0) p.P.p.err[1] = 1;
    grid_dependency_wait();
    return;
  }
  const int ql = (int)(q1 - q0), rows = ql * group;
  // the last rows see the most keys: they start first
  const int turned = (int)(gridDim.x - 1 - blockIdx.x);
  const int row0 = turned / p.P.splits * 2 * kTile, split = turned % p.P.splits;
  if (row0 >= rows || rows <= p.P.min_rows) {
    grid_dependency_wait();
    return;
  }
  const int groups = rows - row0 > kTile ? 2 : 1;
  const auto keys_of = [&](int row) {  // keys that a row sees
    return a.causal ? max(0, min(kv, kv - ql + (int)p.P.group.div((uint32_t)row) + 1)) : kv;
  };
  const int seen = keys_of(min(row0 + groups * kTile, rows) - 1);
  const KeySplit ks(seen, kTile, p.P.splits);
  if (split >= ks.active) {
    grid_dependency_wait();
    return;
  }
  // this split's tiles t0 .. t0 + tiles - 1, called 0 .. tiles - 1 below
  const int t0 = split * ks.per, tiles = min(t0 + ks.per, ks.tiles) - t0;
  const bool tail = (t0 + tiles) * kTile > kv;  // the last tile has rows past the last key

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_ready[g], 4);
    }
    mbar_init(q_ready, 4 * groups);
    mbar_init(v_here, 1);
    mbar_init(v_fixed, 1);
    mbar_init(done, 1);
    *abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  // S_g (and P_g over its first 64 columns) at 128 g, O_g at 256 + D g

  // A softmax thread holds its row's 128 scores.  The launch gives 384 x 168 = 64512 registers;
  // 128 x 56 + 256 x 224 is the same sum.
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == 0) {
    // ---------------- loads ----------------
    const int per_tile = p.page_log2 >= 0 ? kTile >> p.page_log2 : 1;  // pages of a tile
    const int32_t* table = a.block_table + (int64_t)b * a.block_table_stride;
    const auto look = [&](int n) -> int {  // lane i: the page of tile n's i-th box
      if (lane >= per_tile || n >= tiles) return 0;
      const int key = (t0 + n) * kTile + lane * p.box;
      if (key >= kv) return 0;
      const int page = __ldcg(table + p.P.page.div((uint32_t)key));
      if (page >= 0 && page < c.pages) return page;
      p.P.p.err[1] = 1;
      return (int)c.pages;  // past the last page: the copy fills zeros
    };
    int next = look(0);
    int op = 0;
    bool ok = p.starve != 1;
    for (int n = 0; n < tiles && ok; ++n) {
      const int page = next;
      next = look(n + 1);
      const int key0 = (t0 + n) * kTile;
      const int pages = p.page_log2 >= 0 ? min(per_tile, (kv - key0 + p.box - 1) >> p.page_log2) : 1;
      const int tok0 = p.page_log2 >= 0 ? 0 : key0 - (int)p.P.page.div((uint32_t)key0) * c.page_size;
      for (int which = 0; which < 2; ++which, ++op) {
        const int st = op % C::kStages;
        ok = warp_wait(&empty[st], ((op / C::kStages) & 1) ^ 1, abort, p.wait_ns);
        if (!ok) break;
        expect_tx_elect(&full[st], (uint32_t)(pages * p.box * 128 * C::kHalves));
        const uint32_t dst = smem_addr(ring) + st * C::kOperand;
        for (int j = 0; j < pages; ++j) {
          const int pg = __shfl_sync(0xffffffffu, page, j);
#pragma unroll
          for (int half = 0; half < C::kHalves; ++half)
            tma_load_4d_elect(dst + half * C::kSub + j * p.box * 128, which ? &map_v : &map_k, &full[st], half * 64,
                              tok0, hk, pg);
        }
      }
    }
    // Every stage's last copies land before the CTA leaves, whoever gave up and when (after the last
    // copy was issued, too).  Where nobody did, the products wait for them anyway.
    volatile int never = 0;
    for (int s = 0; s < C::kStages && s < op; ++s) {
      const int o = op - 1 - s;
      warp_wait(&full[o % C::kStages], (o / C::kStages) & 1, &never, kDrainNs);
    }
  } else if (warp == 1) {
    // ---------------- products ----------------
    if (tiles > 0) {
      constexpr uint32_t id_s = idesc_16<T>(kTile, kTile, false), id_o = idesc_16<T>(kTile, D, true);
      const uint32_t sq = smem_addr(smem), sr = smem_addr(ring);
      const auto wait_op = [&](int op) {
        return warp_wait(&full[op % C::kStages], (op / C::kStages) & 1, abort, p.wait_ns);
      };
      const auto scores = [&](int g, int op) {
        const uint64_t q = desc_kmajor_sw128(sq + g * C::kOperand);
        const uint64_t k = desc_kmajor_sw128(sr + (op % C::kStages) * C::kOperand);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {  // 16 dimensions on: in the descriptors' 16-byte units
          const int at = (i >> 2) * (C::kSub >> 4) + (i & 3) * 2;
          mma_16_ss_elect(tmem + g * kTile, q + at, k + at, id_s, i != 0);
        }
      };
      if (p.starve == 2) *abort = 1;
      bool ok = p.starve != 2 && warp_wait(q_ready, 0, abort, p.wait_ns) && wait_op(0);
      if (ok) {
        tc_fence_after();
        for (int g = 0; g < groups; ++g) {
          scores(g, 0);
          commit_elect(&s_full[g]);
        }
        commit_elect(&empty[0]);
      }
      for (int n = 0; n < tiles && ok; ++n) {
        const int vop = 2 * n + 1, kop = 2 * n + 2;
        const bool more = n + 1 < tiles;
        ok = wait_op(vop);
        if (ok && !more && tail) {
          arrive_elect(v_here);
          ok = warp_wait(v_fixed, 0, abort, p.wait_ns);
        }
        const uint64_t v = desc_mnmajor_sw128(sr + (vop % C::kStages) * C::kOperand, C::kSub);
        for (int g = 0; g < groups && ok; ++g) {
          ok = warp_wait(&p_ready[g], n & 1, abort, p.wait_ns);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < kTile / 16; ++i)  // 16 keys on: two 1024-byte atoms
            mma_16_ts_elect(tmem + 256 + g * D, tmem + g * kTile + i * 8, v + i * 128, id_o, (n | i) != 0);
          if (more) {
            if (g == 0) {
              ok = wait_op(kop);
              if (!ok) break;
              tc_fence_after();
            }
            scores(g, kop);
          }
          commit_elect(&s_full[g]);
        }
        if (ok) {
          commit_elect(&empty[vop % C::kStages]);
          if (more) commit_elect(&empty[kop % C::kStages]);
        }
      }
      commit_elect(done);
      volatile int never = 0;  // all products have completed before TMEM is freed
      warp_wait(done, 0, &never, kDrainNs);
    }
  } else if (warp == 2) {
    // ---------------- V past the last key ----------------
    if (tiles > 0 && tail) {
      const int op = 2 * (tiles - 1) + 1;
      const bool ok = mbar_wait(v_here, 0, abort, p.wait_ns);
      if (__all_sync(0xffffffffu, ok)) {
        uint8_t* v = ring + (op % C::kStages) * C::kOperand;
        const int first = kv - (t0 + tiles - 1) * kTile;  // whole rows: the swizzle stays inside a row
        for (int h = 0; h < C::kHalves; ++h)
          for (int i = first * 8 + lane; i < kTile * 8; i += 32)
            *reinterpret_cast<uint4*>(v + h * C::kSub + i * 16) = make_uint4(0, 0, 0, 0);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_fixed);
      }
    }
  }
  } else {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
  if ((warp - 4) / 4 < groups) {
    // ---------------- softmax ----------------
    const int g = (warp - 4) / 4;
    const int tr = (warp & 3) * 32 + lane;  // row of the group, and its TMEM lane
    const int row = row0 + g * kTile + tr;
    const bool real = row < rows;
    const int tok = (int)p.P.group.div((uint32_t)(real ? row : 0));
    const int head = hk * group + (real ? row - tok * group : 0);
    {
      // this row's query into the swizzled K-major tile: 16-byte chunk c of a 128-byte row r
      // lies at chunk c ^ (r & 7)
      const T* src = static_cast<const T*>(a.q) + (q0 + tok) * a.q_token_stride + head * a.q_head_stride;
      uint8_t* dst = smem + g * C::kOperand + tr * 128;
#pragma unroll
      for (int ch = 0; ch < D / 8; ++ch) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (real) w = __ldcg(reinterpret_cast<const uint4*>(src) + ch);
        w.x ^= p.flip; w.y ^= p.flip; w.z ^= p.flip; w.w ^= p.flip;
        *reinterpret_cast<uint4*>(dst + (ch >> 3) * C::kSub + (((ch & 7) ^ (tr & 7)) << 4)) = w;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = lanes + g * kTile, to = lanes + 256 + g * D;
    const int limit = real ? keys_of(row) : 0;
    const int all_see = keys_of(row0 + g * kTile);  // keys that every row of the group sees
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int n = 0; n < tiles; ++n) {
      ok = __all_sync(0xffffffffu, mbar_wait_tight(&s_full[g], n & 1, abort, p.wait_ns));
      if (!ok) break;
      tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld32(ts + i * 32, v[i]);
      tmem_ld_wait();
      if ((t0 + n + 1) * kTile > all_see) {
        const int left = limit - (t0 + n) * kTile;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) v[i][j] = i * 32 + j < left ? v[i][j] : 0xff800000u;
      }
      float top[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top[i] = fmaxf(u2f(v[i][0]), u2f(v[i][1]));
#pragma unroll
        for (int j = 2; j < 32; j += 2) top[i] = fmaxf(top[i], fmaxf(u2f(v[i][j]), u2f(v[i][j + 1])));
      }
      const float raw = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      const float now = raw == -INFINITY ? -INFINITY : raw * p.scale2;
      const bool grow = now - m > kLazy;  // (also from -inf)
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? mma16::ex2(m - now) : 1.0f;
        if (grow) m = now;
        l *= f;
        if (n > 0) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tmem_ld32(to + i * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = f2u(u2f(o[j]) * f);
            tmem_st32(to + i * 32, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.0f : m;  // no key yet: 2^(-inf) = 0
      const f32x2 sc = splat2(p.scale2), nb = splat2(-base);
      f32x2 sum = splat2(0.0f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t pk[32];
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          const uint32_t x = v[2 * i + (j >> 5)][j & 31], y = v[2 * i + (j >> 5)][(j & 31) + 1];
          const f32x2 e = fma2(pack2(u2f(x), u2f(y)), sc, nb);
          const float e0 = mma16::ex2(lo2(e)), e1 = mma16::ex2(hi2(e));
          sum = add2(sum, pack2(e0, e1));
          pk[j >> 1] = mma16::pack<T>(e0, e1);
        }
        tmem_st32(ts + i * 32, pk);
      }
      l += lo2(sum) + hi2(sum);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[g]);
    }
    if (tiles > 0 && ok) {
      ok = __all_sync(0xffffffffu, mbar_wait_tight(&s_full[g], tiles & 1, abort, p.wait_ns));
      tc_fence_after();
    }
    if (!ok) *abort = 1;
    T* dst = static_cast<T*>(a.out) + (q0 + tok) * a.out_token_stride + head * a.out_head_stride;
    const int64_t part = ((int64_t)split * a.tokens + q0 + tok) * a.heads + head;
    if (ok && real && ks.active > 1) p.P.part_ml[part] = make_float2(m, l);
    const float inv = 1.0f / l;
    if (ok) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        __syncwarp();
        if (tiles > 0) {
          tmem_ld32(to + i * 32, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int j = 0; j < 32 && real; j += 8) {
          float y[8];
          if (ks.active > 1) {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = u2f(o[j + k]);
            Pack<float, 8>::store(p.P.part_o + part * D + i * 32 + j, y);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = l == 0.0f ? 0.0f : u2f(o[j + k]) * inv;  // no key: zeros
            Pack<T, 8>::store(dst + i * 32 + j, y);
          }
        }
      }
    }
    tc_fence_before();
  }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort) atomicExch(p.P.p.err, 1);
  grid_dependency_wait();  // when this launch ends, so has the one it ran beside
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T>
bool cache_map(CUtensorMap* map, void* base, const rg_kv_cache& c, int box) {
  const auto fn = tma_encode_fn();
  if (!fn) return false;
  // a dimension of one has no stride of its own
  const auto bytes = [](int64_t n, int64_t s) { return (cuuint64_t)(n > 1 ? s * 2 : 16); };
  const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads,
                              (cuuint64_t)c.pages};
  const cuuint64_t strides[3] = {bytes(c.page_size, c.token_stride), bytes(c.kv_heads, c.head_stride),
                                 bytes(c.pages, c.page_stride)};
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, one[4] = {1, 1, 1, 1};
  const auto type = sizeof(T) == 2 && __is_same(T, __half) ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return fn(map, type, 4, base, dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
rg_status go(const AttnParams& P, bool beside, cudaStream_t st) {
  using C = Cfg<D>;
  const auto kernel = k_attn_tc<T, D>;
  static DeviceOnce once;
  once.run([&] { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem); });
  TcParams p;
  p.P = P;
  const rg_kv_cache& c = P.p.c;
  p.box = c.page_size < kTile ? c.page_size : kTile;
  p.page_log2 = -1;
  if (c.page_size < kTile)
    for (p.page_log2 = 3; (1 << p.page_log2) < c.page_size;) ++p.page_log2;
  // a hidden score is -inf before the scale: a scale of 0 becomes the smallest normal number
  p.scale2 = fmaxf(fabsf(P.scale2), FLT_MIN);
  p.flip = P.scale2 < 0.0f ? 0x80008000u : 0u;
  p.wait_ns = P.p.wait_ns ? P.p.wait_ns : kWaitNs;
  p.starve = P.p.starve;
  CUtensorMap mk, mv;
  if (!cache_map<T>(&mk, c.k, c, p.box) || !cache_map<T>(&mv, c.v, c, p.box)) return RG_ERR_CUDA;
  const int64_t rows = (int64_t)P.p.a.max_q_len * P.group.d, blocks = (rows + kTcRows - 1) / kTcRows * P.splits;
  if (blocks > INT_MAX) return RG_ERR_UNSUPPORTED;
  p.beside = beside;
  const dim3 grid((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)P.p.a.batch);
  launch_early(kernel, grid, kThreads, C::kSmem, st, mk, mv, p);
  return RG_OK;
}

}  // namespace

bool attention_tc_takes(const PagedAttnArgs& p) {
  const int page = p.c.page_size;
  if (p.c.head_dim != 64 && p.c.head_dim != 128) return false;
  if (page < kTile ? page < 8 || (page & (page - 1)) : page % kTile) return false;
  // tensor map limits: strides below 2^40 bytes
  const int64_t most = (int64_t)1 << 39;
  return p.c.page_stride < most && p.c.token_stride < most && p.c.head_stride < most;
}

rg_status launch_attention_tc(const AttnParams& P, bool beside, cudaStream_t st) {
  if (P.p.c.dtype == RG_DTYPE_F16) return P.p.c.head_dim == 64 ? go<__half, 64>(P, beside, st) : go<__half, 128>(P, beside, st);
  return P.p.c.head_dim == 64 ? go<__nv_bfloat16, 64>(P, beside, st) : go<__nv_bfloat16, 128>(P, beside, st);
}

}  // namespace rg

// serving.cu -- C entry points of the decoder-serving operators: argument checks, and the
// launch.  Everything a host can see is checked here before any device work; the kernels
// check what only the device can (positions, slots, pages, lengths).
#include <cuda_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <climits>

#include "../../include/rg_npu.h"
#include "rg_kernels.h"
#include "rg_serving.h"

namespace {

using namespace rg;

rg_status refuse(rg_status st, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_last_error(st, buf);
}

// The launch's own error, if any; an error that was pending before belongs to someone else
// and is reported as such by the first call that meets it.
rg_status launched(const char* what, rg_status st) {
  if (st == RG_ERR_CUDA) return refuse(st, "%s: TMA descriptor encoding failed", what);
  if (st != RG_OK) return refuse(st, "%s: the sizes exceed the launch limits", what);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? RG_OK : refuse(RG_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool is_dtype(int32_t dt) { return dt == RG_DTYPE_F32 || dt == RG_DTYPE_F16 || dt == RG_DTYPE_BF16; }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

rg_status check_rows(const char* f, const void* x, int32_t dt, int64_t rows, int64_t k, int64_t ldx, int64_t ldq) {
  if (!is_dtype(dt)) return refuse(RG_ERR_INVALID_ARG, "%s: unknown x dtype %d", f, dt);
  if (rows < 0 || rows > INT_MAX || k <= 0 || ldx < k || ldq < k || (ldq & 15))
    return refuse(RG_ERR_INVALID_ARG,
                  "%s: rows %lld, k %lld, ldx %lld, ld %lld (ldx >= k, ld >= k and a multiple of 16 wanted)", f,
                  (long long)rows, (long long)k, (long long)ldx, (long long)ldq);
  if (rows > 0 && !x) return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (rows > 0 && !aligned(x, dtype_size(dt))) return refuse(RG_ERR_INVALID_ARG, "%s: x must be aligned to its type", f);
  return RG_OK;
}

rg_status check_gemm(const char* f, const int8_t* w, const float* w_scale, int64_t m, int64_t n, int64_t ld,
                     const float* bias, int32_t act, const void* out, int32_t out_dtype, int64_t ldo,
                     const int32_t* err) {
  if (!is_dtype(out_dtype)) return refuse(RG_ERR_INVALID_ARG, "%s: unknown output dtype %d", f, out_dtype);
  if (act < RG_ACT_NONE || act > RG_ACT_SILU) return refuse(RG_ERR_INVALID_ARG, "%s: unknown activation %d", f, act);
  if (m < 0 || m > INT_MAX || n <= 0 || n > INT_MAX || ld <= 0 || (ld & 15) || ldo < n)
    return refuse(RG_ERR_INVALID_ARG, "%s: m %lld, n %lld, ld %lld, ldo %lld (ld a multiple of 16, ldo >= n wanted)", f,
                  (long long)m, (long long)n, (long long)ld, (long long)ldo);
  // |sum| <= 127 * 128 * ld has to fit 32 bits
  if (ld > INT_MAX / (127 * 128)) return refuse(RG_ERR_UNSUPPORTED, "%s: ld %lld exceeds the i32 sums", f, (long long)ld);
  if (m == 0) return RG_OK;
  if (!w || !w_scale || !out || !err) return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (!aligned(w, 16) || !aligned(w_scale, 4) || !aligned(bias, 4) || !aligned(out, dtype_size(out_dtype)) ||
      !aligned(err, 4))
    return refuse(RG_ERR_INVALID_ARG, "%s: w must be 16-byte aligned, the others aligned to their types", f);
  return RG_OK;
}

// Whether any of m rows of `a` bytes, `as` bytes apart, shares memory with one of m rows of `b`
// bytes, `bs` bytes apart (m is small).
bool rows_overlap(const void* x, int64_t a, int64_t as, const void* y, int64_t b, int64_t bs, int64_t m) {
  const uintptr_t px = reinterpret_cast<uintptr_t>(x), py = reinterpret_cast<uintptr_t>(y);
  if (px + (uintptr_t)((m - 1) * as + a) <= py || py + (uintptr_t)((m - 1) * bs + b) <= px) return false;
  for (int64_t i = 0; i < m; ++i)
    for (int64_t j = 0; j < m; ++j) {
      const uintptr_t u = px + (uintptr_t)(i * as), v = py + (uintptr_t)(j * bs);
      if (u < v + (uintptr_t)b && v < u + (uintptr_t)a) return true;
    }
  return false;
}

#define RG_CHECK(expr)                \
  do {                                \
    const rg_status st_ = (expr);     \
    if (st_ != RG_OK) return st_;     \
  } while (0)

__global__ void k_take_words(int32_t* words, int32_t* taken) { taken[threadIdx.x] = atomicExch(words + threadIdx.x, 0); }

rg_status check_cache(const char* f, const rg_kv_cache* c) {
  if (!c) return refuse(RG_ERR_INVALID_ARG, "%s: null cache", f);
  if (c->dtype != RG_DTYPE_F16 && c->dtype != RG_DTYPE_BF16)
    return refuse(RG_ERR_UNSUPPORTED, "%s: the cache is f16 or bf16", f);
  if (c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0 || c->pages <= 0 || c->pages > INT_MAX)
    return refuse(RG_ERR_INVALID_ARG, "%s: pages %lld of %d tokens, %d heads of %d", f, (long long)c->pages,
                  c->page_size, c->kv_heads, c->head_dim);
  if (!c->k || !c->v) return refuse(RG_ERR_INVALID_ARG, "%s: null cache tensor", f);
  if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
    return refuse(RG_ERR_INVALID_ARG, "%s: negative cache stride", f);
  if (!aligned(c->k, 2) || !aligned(c->v, 2)) return refuse(RG_ERR_INVALID_ARG, "%s: misaligned cache", f);
  return RG_OK;
}

rg_status check_rotation(const char* f, const int32_t* positions, const float* table, int64_t rows, int32_t rot,
                         int32_t head_dim) {
  if (rot <= 0 || (rot & 1) || rot > head_dim)
    return refuse(RG_ERR_INVALID_ARG, "%s: rot_dim %d has to be even and at most head_dim %d", f, rot, head_dim);
  if (!positions || !table || rows <= 0) return refuse(RG_ERR_INVALID_ARG, "%s: null or empty table", f);
  if (!aligned(positions, 4) || !aligned(table, 4)) return refuse(RG_ERR_INVALID_ARG, "%s: misaligned table", f);
  return RG_OK;
}

}  // namespace

extern "C" {

rg_status rg_take_error_words(int32_t* error_words, int32_t* taken, void* stream) {
  const char* f = "rg_take_error_words";
  if (!error_words || !taken) return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (!aligned(error_words, 4) || !aligned(taken, 4)) return refuse(RG_ERR_INVALID_ARG, "%s: misaligned words", f);
  k_take_words<<<1, 2, 0, (cudaStream_t)stream>>>(error_words, taken);
  return launched(f, RG_OK);
}

rg_status rg_quantize_token_i8(const void* x, int32_t x_dtype, int64_t rows, int64_t k, int64_t ldx, int8_t* q,
                               int64_t ldq, float* scale, void* stream) {
  const char* f = "rg_quantize_token_i8";
  RG_CHECK(check_rows(f, x, x_dtype, rows, k, ldx, ldq));
  if (rows == 0) return RG_OK;
  if (!q || !scale) return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (!aligned(q, 16) || !aligned(scale, 4))
    return refuse(RG_ERR_INVALID_ARG, "%s: the i8 rows must be aligned to 16 bytes", f);
  launch_quantize_token(x, x_dtype, rows, k, ldx, q, ldq, scale, (cudaStream_t)stream);
  return launched(f, RG_OK);
}

rg_status rg_gemm_i8_token(const int8_t* a, const float* a_scale, const int8_t* w, const float* w_scale, int64_t m,
                           int64_t n, int64_t ld, const float* bias, int32_t act, float act_param, void* out,
                           int32_t out_dtype, int64_t ldo, int32_t* error_words, void* stream) {
  const char* f = "rg_gemm_i8_token";
  RG_CHECK(check_gemm(f, w, w_scale, m, n, ld, bias, act, out, out_dtype, ldo, error_words));
  if (m == 0) return RG_OK;
  if (!a || !a_scale) return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (!aligned(a, 16) || !aligned(a_scale, 4)) return refuse(RG_ERR_INVALID_ARG, "%s: a must be 16-byte aligned", f);
  TokenGemmArgs g;
  g.a = a; g.a_scale = a_scale; g.w = w; g.w_scale = w_scale; g.bias = bias;
  g.m = m; g.n = n; g.ld = ld; g.ldo = ldo; g.act = act; g.act_param = act_param;
  g.out = out; g.out_dtype = out_dtype; g.err = error_words;
  tc_wait_hook(&g.wait_ns, &g.starve);
  return launched(f, launch_gemm_token(g, (cudaStream_t)stream));
}

int64_t rg_linear_i8_token_workspace_size(int64_t m, int64_t n, int64_t ld) {
  if (m <= 0 || n <= 0 || ld <= 0 || linear_skinny_takes(m, n, ld)) return 0;
  return round_up(m * ld, 256) + round_up(m * (int64_t)sizeof(float), 256);
}

rg_status rg_linear_i8_token(const rg_linear_token_args* p, void* workspace, int32_t* error_words, void* stream) {
  const char* f = "rg_linear_i8_token";
  if (!p) return refuse(RG_ERR_INVALID_ARG, "%s: null arguments", f);
  RG_CHECK(check_gemm(f, p->w, p->w_scale, p->m, p->n, p->ld, p->bias, p->act, p->out, p->out_dtype, p->ldo,
                      error_words));
  const bool skinny = linear_skinny_takes(p->m, p->n, p->ld);
  if (p->m > 0 && !skinny && (!workspace || !aligned(workspace, 256)))
    return refuse(RG_ERR_INVALID_ARG, "%s: the workspace must be given and 256-byte aligned", f);
  int8_t* q = static_cast<int8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(static_cast<char*>(workspace) + round_up(p->m * p->ld, 256));
  RG_CHECK(check_rows(f, p->x, p->x_dtype, p->m, p->k, p->ldx, p->ld));
  if (p->m == 0) return RG_OK;
  // every block of the one launch reads all of x, also after others have stored their outputs
  const int64_t sx = dtype_size(p->x_dtype), so = dtype_size(p->out_dtype);
  if (skinny && rows_overlap(p->x, p->k * sx, p->ldx * sx, p->out, p->n * so, p->ldo * so, p->m))
    return refuse(RG_ERR_INVALID_ARG, "%s: x and out overlap, which this size (no workspace, one launch) cannot take", f);
  TokenGemmArgs g;
  g.a = q; g.a_scale = scale; g.w = p->w; g.w_scale = p->w_scale; g.bias = p->bias;
  g.m = p->m; g.n = p->n; g.ld = p->ld; g.ldo = p->ldo; g.act = p->act; g.act_param = p->act_param;
  g.out = p->out; g.out_dtype = p->out_dtype; g.err = error_words; g.after_quantizer = 1;
  tc_wait_hook(&g.wait_ns, &g.starve);
  if (skinny) return launched(f, launch_linear_skinny(g, p->x, p->x_dtype, p->k, p->ldx, (cudaStream_t)stream));
  launch_quantize_token(p->x, p->x_dtype, p->m, p->k, p->ldx, q, p->ld, scale, (cudaStream_t)stream);
  return launched(f, launch_gemm_token(g, (cudaStream_t)stream));
}

rg_status rg_rope_table_f32(const rg_rope_scaling* s, int64_t positions, int32_t rot_dim, float* table, void* stream) {
  const char* f = "rg_rope_table_f32";
  if (!s || !table) return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (positions < 0 || rot_dim <= 0 || (rot_dim & 1) || positions > ((int64_t)INT_MAX * 256) / rot_dim)
    return refuse(RG_ERR_INVALID_ARG, "%s: %lld positions of rot_dim %d (even)", f, (long long)positions, rot_dim);
  if (s->kind < RG_ROPE_PLAIN || s->kind > RG_ROPE_BANDS)
    return refuse(RG_ERR_INVALID_ARG, "%s: unknown scaling %d", f, s->kind);
  if (!(s->base > 1.0) || !(s->gain > 0.0) || !isfinite(s->base) || !isfinite(s->gain))
    return refuse(RG_ERR_INVALID_ARG, "%s: base must exceed 1 and gain 0", f);
  if (s->kind != RG_ROPE_PLAIN && (!(s->factor > 0.0) || !isfinite(s->factor)))
    return refuse(RG_ERR_INVALID_ARG, "%s: factor must be positive", f);
  if (s->kind == RG_ROPE_BANDS && (!(s->old_context > 0.0) || !(s->slow_turns > 0.0) ||
                                   !(s->fast_turns > s->slow_turns) || !isfinite(s->old_context) ||
                                   !isfinite(s->fast_turns)))
    return refuse(RG_ERR_INVALID_ARG, "%s: bands need old_context > 0 and fast_turns > slow_turns > 0", f);
  if (!aligned(table, 4)) return refuse(RG_ERR_INVALID_ARG, "%s: misaligned table", f);
  if (positions == 0) return RG_OK;
  launch_rope_table(*s, positions, rot_dim, table, (cudaStream_t)stream);
  return launched(f, RG_OK);
}

rg_status rg_rope(const rg_rope_args* p, int32_t* error_words, void* stream) {
  const char* f = "rg_rope";
  if (!p) return refuse(RG_ERR_INVALID_ARG, "%s: null arguments", f);
  if (!is_dtype(p->dtype)) return refuse(RG_ERR_INVALID_ARG, "%s: unknown dtype %d", f, p->dtype);
  if (p->tokens < 0 || p->heads <= 0 || p->head_dim <= 0 || (p->head_dim & 1))
    return refuse(RG_ERR_INVALID_ARG, "%s: %lld tokens of %d heads of %d (even)", f, (long long)p->tokens, p->heads,
                  p->head_dim);
  if (p->token_stride < 0 || p->head_stride < 0 || p->out_token_stride < 0 || p->out_head_stride < 0)
    return refuse(RG_ERR_INVALID_ARG, "%s: negative stride", f);
  if (p->tokens == 0) return RG_OK;
  if (!p->x || !p->out || !error_words) return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (!aligned(p->x, dtype_size(p->dtype)) || !aligned(p->out, dtype_size(p->dtype)))
    return refuse(RG_ERR_INVALID_ARG, "%s: misaligned tensor", f);
  RG_CHECK(check_rotation(f, p->positions, p->table, p->table_rows, p->rot_dim, p->head_dim));
  RopeArgs r;
  r.q = p->x; r.q_ts = p->token_stride; r.q_hs = p->head_stride;
  r.q_out = p->out; r.qo_ts = p->out_token_stride; r.qo_hs = p->out_head_stride;
  r.positions = p->positions; r.table = p->table; r.table_rows = p->table_rows; r.rot_dim = p->rot_dim;
  r.tokens = p->tokens; r.heads = p->heads; r.head_dim = p->head_dim;
  r.in_dtype = r.out_dtype = p->dtype; r.interleaved = p->interleaved; r.err = error_words;
  return launched(f, launch_rope(r, (cudaStream_t)stream));
}

rg_status rg_kv_append(const rg_kv_cache* cache, const rg_kv_append_args* a, int32_t* error_words, void* stream) {
  const char* f = "rg_kv_append";
  RG_CHECK(check_cache(f, cache));
  if (!a) return refuse(RG_ERR_INVALID_ARG, "%s: null arguments", f);
  if (a->x_dtype != RG_DTYPE_F32 && a->x_dtype != cache->dtype)
    return refuse(RG_ERR_UNSUPPORTED, "%s: x is f32 or of the cache's dtype", f);
  if (a->tokens < 0 || (cache->head_dim & 1)) return refuse(RG_ERR_INVALID_ARG, "%s: tokens >= 0 and an even head_dim", f);
  if (a->k_token_stride < 0 || a->k_head_stride < 0 || a->v_token_stride < 0 || a->v_head_stride < 0 ||
      (a->q && (a->q_token_stride < 0 || a->q_head_stride < 0 || a->q_out_token_stride < 0 ||
                a->q_out_head_stride < 0)))
    return refuse(RG_ERR_INVALID_ARG, "%s: negative stride", f);
  if (a->q && a->heads <= 0) return refuse(RG_ERR_INVALID_ARG, "%s: q of %d heads", f, a->heads);
  if (a->tokens == 0) return RG_OK;
  const size_t si = dtype_size(a->x_dtype);
  if (!a->k || !a->v || !a->slots || !error_words || (a->q && !a->q_out))
    return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (!aligned(a->k, si) || !aligned(a->v, si) || !aligned(a->q, si) || !aligned(a->q_out, 2) || !aligned(a->slots, 8))
    return refuse(RG_ERR_INVALID_ARG, "%s: misaligned tensor", f);
  if (a->table) RG_CHECK(check_rotation(f, a->positions, a->table, a->table_rows, a->rot_dim, cache->head_dim));
  RopeArgs r;
  r.q = a->q; r.q_ts = a->q_token_stride; r.q_hs = a->q_head_stride;
  r.q_out = a->q_out; r.qo_ts = a->q_out_token_stride; r.qo_hs = a->q_out_head_stride;
  r.heads = a->q ? a->heads : 0;
  r.k = a->k; r.k_ts = a->k_token_stride; r.k_hs = a->k_head_stride;
  r.v = a->v; r.v_ts = a->v_token_stride; r.v_hs = a->v_head_stride;
  r.k_out = cache->k; r.v_out = cache->v; r.kv_heads = cache->kv_heads; r.head_dim = cache->head_dim;
  r.page_stride = cache->page_stride; r.token_stride = cache->token_stride; r.head_stride = cache->head_stride;
  r.page_size = cache->page_size; r.num_slots = cache->pages * cache->page_size;
  r.slots = a->slots; r.positions = a->positions; r.table = a->table; r.table_rows = a->table_rows;
  r.rot_dim = a->table ? a->rot_dim : 0;
  r.tokens = a->tokens; r.in_dtype = a->x_dtype; r.out_dtype = cache->dtype; r.interleaved = a->interleaved;
  r.err = error_words;
  return launched(f, launch_rope(r, (cudaStream_t)stream));
}

static rg_status check_attention(const char* f, const rg_kv_cache* c, const rg_paged_attention_args* a) {
  RG_CHECK(check_cache(f, c));
  if (!a) return refuse(RG_ERR_INVALID_ARG, "%s: null arguments", f);
  if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256)
    return refuse(RG_ERR_UNSUPPORTED, "%s: head_dim %d (64, 96, 128 and 256 are built)", f, c->head_dim);
  if (a->batch < 0 || a->batch > 65535 || a->tokens < 0 || a->heads <= 0 || a->heads > 65535 ||
      a->heads % c->kv_heads || a->max_q_len < 0 || a->max_kv_len < 0 || a->max_pages < 0 || a->block_table_stride < 0)
    return refuse(RG_ERR_INVALID_ARG,
                  "%s: batch %d, tokens %lld, heads %d over %d key heads, max_q_len %d, max_kv_len %d", f, a->batch,
                  (long long)a->tokens, a->heads, c->kv_heads, a->max_q_len, a->max_kv_len);
  if ((int64_t)a->max_pages * c->page_size < a->max_kv_len)
    return refuse(RG_ERR_INVALID_ARG, "%s: %d pages of %d tokens hold fewer than max_kv_len %d keys", f, a->max_pages,
                  c->page_size, a->max_kv_len);
  if (!isfinite(a->scale)) return refuse(RG_ERR_INVALID_ARG, "%s: scale is not finite", f);
  if (a->q_token_stride < 0 || a->q_head_stride < 0 || a->out_token_stride < 0 || a->out_head_stride < 0)
    return refuse(RG_ERR_INVALID_ARG, "%s: negative stride", f);
  // rows of a head are read and written 16 bytes at a time
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || (c->page_stride & 7) || (c->token_stride & 7) ||
      (c->head_stride & 7) || !aligned(a->q, 16) || !aligned(a->out, 16) || (a->q_token_stride & 7) ||
      (a->q_head_stride & 7) || (a->out_token_stride & 7) || (a->out_head_stride & 7))
    return refuse(RG_ERR_INVALID_ARG, "%s: q, out and cache must be 16-byte aligned, strides multiples of 8", f);
  return RG_OK;
}

int64_t rg_attention_paged_workspace_size(const rg_kv_cache* cache, const rg_paged_attention_args* args) {
  if (check_attention("rg_attention_paged_workspace_size", cache, args) != RG_OK) return -1;
  if (args->batch == 0 || args->tokens == 0 || args->max_q_len == 0) return 0;
  PagedAttnArgs p;
  p.c = *cache;
  p.a = *args;
  return attention_paged_workspace(p);
}

rg_status rg_attention_paged(const rg_kv_cache* cache, const rg_paged_attention_args* args, void* workspace,
                             int32_t* error_words, void* stream) {
  const char* f = "rg_attention_paged";
  RG_CHECK(check_attention(f, cache, args));
  if (args->batch == 0 || args->tokens == 0) return RG_OK;  // (max_q_len 0: the lengths are looked at all the same)
  if (!args->q || !args->out || !args->kv_len || !args->cu_q || !error_words ||
      (!args->block_table && args->max_kv_len > 0))
    return refuse(RG_ERR_INVALID_ARG, "%s: null argument", f);
  if (!aligned(args->block_table, 4) || !aligned(args->kv_len, 4) || !aligned(args->cu_q, 4))
    return refuse(RG_ERR_INVALID_ARG, "%s: misaligned lengths or block table", f);
  PagedAttnArgs p;
  p.c = *cache;
  p.a = *args;
  p.workspace = workspace;
  p.err = error_words;
  tc_wait_hook(&p.wait_ns, &p.starve);
  const int64_t need = attention_paged_workspace(p);
  if (need > 0 && (!workspace || !aligned(workspace, 256)))
    return refuse(RG_ERR_INVALID_ARG, "%s: a workspace of %lld bytes, 256-byte aligned, is needed", f, (long long)need);
  return launched(f, launch_attention_paged(p, (cudaStream_t)stream));
}

}  // extern "C"

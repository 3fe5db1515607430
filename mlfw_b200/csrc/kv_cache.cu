// The int8 key/value cache: writing new rows (per-token quantize of every head's row), reading rows back, keeping the
// accepted rows of a drafted tree; and the C entry points of the cache (declared in include/b200q.h).
//
// The reference keeps no cache between calls of its attention (src/nn/functional/attention.ts:42-74 takes whole K and V);
// a cached row is quantized by the rule its dynamic quantization applies to a row of activations
// (quantization_types.ts:299-317, 118-130), here one row = one head of one token.
#include <cmath>
#include <new>

#include "../../include/b200q.h"
#include "kernels.cuh"
#include "kv.cuh"
#include "quant_math.cuh"

namespace b200q {

namespace {

struct KvArgs {
  KvGeom g;
  int8_t *k, *v;
  float *ks, *vs;
  const int32_t *page_table, *start, *count;
  int B, T;
  uint32_t* status;
};

KvArgs kv_args(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s) {
  return KvArgs{KvGeom{c.pages, s.max_pages, c.page_shift, c.heads}, c.k, c.v, c.ks, c.vs, s.page_table, s.start, s.count, s.B, s.T, ctx->status_dev};
}

// Scale of a row from its NaN-ignoring extremes (quantization_types.ts:308-316, 271-275).
__device__ __forceinline__ double kv_row_scale(float mn_f, float mx_f) {
  double mn = (double)mn_f, mx = (double)mx_f;
  if (!isfinite(mn)) mn = -1.0;
  if (!isfinite(mx)) mx = 1.0;
  if (mn == mx) { mn -= 0.5; mx += 0.5; }
  const double s = fmax(fabs(mn), fabs(mx)) / 127.0;
  return (s == 0.0 || s != s) ? 1e-10 : s;
}

// ---------------------------------------------------------------------------
// Write: codes and scales of the new rows.  Eight lanes per row (D / 32 float4 each: every load and every store is a
// run of whole 32-byte sectors), four heads of a token per warp, K and V of them in the same warp so that 2 * D / 32
// 16-byte loads per lane are in flight.  Codes: t = x * (127 / absmax), rounded by the 1.5 * 2^23 trick; an element
// within 127.5 * 2^-21 of a tie, or a row with a NaN, an infinity, equal elements or a range the reciprocal does not represent,
// takes the exact binary64 routine, so codes and scales are those of b200q_quantize_per_token on the same rows.
// Bound by memory latency (four bytes read and one written per element, behind the chain count, start, page): 7000 tokens of
// 8 heads of 128, 72 MB in 19 us (3.7 TB/s; with the read of the next kernel 28 to 29.5 us; where this took 27.8, three blocks per
// SM instead of four took 28.7, and K and V in warps of their own 28.0); a decoding step's 32 tokens are a launch, 4.6 us.  Four blocks
// leave 64 registers: for D = 128 one word spills.
// ---------------------------------------------------------------------------
template <int V4>   // float4 per lane: D = 32 * V4
__device__ __forceinline__ void append_row(const float4 (&x)[V4], bool live, int sub, uint32_t* codes, float* scale) {
  float mn = __int_as_float(0x7f800000), mx = __int_as_float(0xff800000);
#pragma unroll
  for (int i = 0; i < V4; i++) {
    mn = fminf(fminf(mn, x[i].x), fminf(fminf(x[i].y, x[i].z), x[i].w));
    mx = fmaxf(fmaxf(mx, x[i].x), fmaxf(fmaxf(x[i].y, x[i].z), x[i].w));
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (!live) return;
  const float absmax = fmaxf(fabsf(mn), fabsf(mx));
  const float inv = __fdiv_rn(127.0f, absmax);
  const bool exact_only = !((mn < mx) && absmax <= 3.402823466e38f && inv >= 1.17549435e-38f && inv <= 3.402823466e38f);
  const uint64_t inv2 = f2_dup(inv), magic2 = f2_dup(12582912.0f);
#pragma unroll
  for (int i = 0; i < V4; i++) {
    float far = 0.0f;
    uint32_t w = pack4_fast_lean_nan(x[i], inv2, magic2, far);
    if (exact_only || !(far < 0.49993920f)) {   // 0.5 - 127.5 * 2^-21; a NaN counts as near
      const double sd = kv_row_scale(mn, mx);
      w = pack_codes(quantize_exact_p(x[i].x, sd, -127.f, 127.f), quantize_exact_p(x[i].y, sd, -127.f, 127.f),
                     quantize_exact_p(x[i].z, sd, -127.f, 127.f), quantize_exact_p(x[i].w, sd, -127.f, 127.f));
    }
    codes[sub + 8 * i] = w;
  }
  if (sub == 0) *scale = exact_only ? (float)kv_row_scale(mn, mx) : __fdiv_rn(absmax, 127.0f);
}

template <int D>
__global__ void __launch_bounds__(256, 4) kv_append_kernel(const KvArgs a, const float* k, const float* v, int64_t ld_k,
                                                           int64_t ld_v, uint32_t units, uint32_t chunks) {
  constexpr int V4 = D / 32;
  kv_after_previous();
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const uint32_t u = kv_warp(blockIdx.x, blockDim.x, threadIdx.x);
  if (u >= units) return;
  const uint32_t token = u / chunks, head = (u - token * chunks) * 4 + (lane >> 3);
  const uint32_t b = token / (uint32_t)a.T, t = token - b * (uint32_t)a.T;
  if ((int)t >= kv_rows_in_use(a.count, b, a.T)) return;
  const bool has = head < (uint32_t)a.g.heads;
  const int64_t row = kv_row(a.g, a.page_table, b, has ? head : 0, (int64_t)a.start[b] + t);
  if (row < 0) {
    if (lane == 0) atomicOr(a.status, STATUS_BAD_INDEX);
    return;
  }
  float4 xk[V4], xv[V4];
  const float4* kr = reinterpret_cast<const float4*>(k + (int64_t)token * ld_k + (has ? head : 0) * D) + sub;
  const float4* vr = reinterpret_cast<const float4*>(v + (int64_t)token * ld_v + (has ? head : 0) * D) + sub;
#pragma unroll
  for (int i = 0; i < V4; i++) xk[i] = __ldcs(kr + 8 * i);
#pragma unroll
  for (int i = 0; i < V4; i++) xv[i] = __ldcs(vr + 8 * i);
  append_row<V4>(xk, has, sub, reinterpret_cast<uint32_t*>(a.k + row * D), a.ks + row);
  append_row<V4>(xv, has, sub, reinterpret_cast<uint32_t*>(a.v + row * D), a.vs + row);
}

// ---------------------------------------------------------------------------
// Read: y = fround(code * scale).  The same split: eight lanes per row, four heads of a token per warp, K and V.  A row
// whose position is outside the cache reads as zeros and sets the status bit.  Bound by memory: 8 x 4096 tokens of 8 heads of
// 128, 337 MB in 56.6 us (5.95 TB/s of the 6.5 measured).
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvArgs a, float* __restrict__ k_out, float* __restrict__ v_out, int64_t ld_k,
                                                      int64_t ld_v, uint32_t units, uint32_t chunks) {
  constexpr int V4 = D / 32;
  kv_after_previous();
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const uint32_t u = kv_warp(blockIdx.x, blockDim.x, threadIdx.x);
  if (u >= units) return;
  const uint32_t token = u / chunks, head = (u - token * chunks) * 4 + (lane >> 3);
  const uint32_t b = token / (uint32_t)a.T, t = token - b * (uint32_t)a.T;
  if ((int)t >= kv_rows_in_use(a.count, b, a.T) || head >= (uint32_t)a.g.heads) return;
  const int64_t row = kv_row(a.g, a.page_table, b, head, (int64_t)a.start[b] + t);
  if (row < 0 && sub == 0) atomicOr(a.status, STATUS_BAD_INDEX);
  uint32_t w[2][V4];
  float s[2];
#pragma unroll
  for (int kv = 0; kv < 2; kv++) {
    const uint32_t* codes = reinterpret_cast<const uint32_t*>((kv ? a.v : a.k) + (row < 0 ? 0 : row) * D) + sub;
    s[kv] = row < 0 ? 0.0f : __ldcg((kv ? a.vs : a.ks) + row);
#pragma unroll
    for (int i = 0; i < V4; i++) w[kv][i] = row < 0 ? 0u : __ldcg(codes + 8 * i);
  }
#pragma unroll
  for (int kv = 0; kv < 2; kv++) {
    float4* y = reinterpret_cast<float4*>((kv ? v_out : k_out) + (int64_t)token * (kv ? ld_v : ld_k) + head * D) + sub;
#pragma unroll
    for (int i = 0; i < V4; i++) {
      const uint32_t x = w[kv][i];
      __stcs(y + 8 * i, make_float4(__fmul_rn((float)(int8_t)x, s[kv]), __fmul_rn((float)(int8_t)(x >> 8), s[kv]),
                                    __fmul_rn((float)(int8_t)(x >> 16), s[kv]), __fmul_rn((float)(int8_t)(x >> 24), s[kv])));
    }
  }
}

// ---------------------------------------------------------------------------
// Keep: position start + keep[i] moves to start + i.  One block per (sequence, head): it holds all moved rows (at most 64
// of K and of V: 16 KB) in registers between the reads and the writes, so any order and any repetition of sources is right.
// A move whose source or target lies outside the cache is dropped and sets the status bit.  A few kilobytes per block behind
// three dependent loads (count and keep, the page table, the rows): latency, 4.8 us for eight sequences of 8 heads.
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(128) kv_keep_kernel(const KvArgs a, const int32_t* keep) {
  constexpr int Q = D / 16, PER = KV_MAX_TREE * Q / 128;   // 16-byte pieces of a row; pieces a thread holds of K (and of V)
  __shared__ int64_t from[KV_MAX_TREE], to[KV_MAX_TREE];
  kv_after_previous();
  const int head = blockIdx.x % a.g.heads, b = blockIdx.x / a.g.heads, tid = threadIdx.x;
  const int n = kv_rows_in_use(a.count, b, a.T);
  if (tid < n) {
    const int src = keep[(int64_t)b * a.T + tid];
    const int64_t s = a.start[b], f = (src < 0 || src >= a.T) ? -1 : kv_row(a.g, a.page_table, b, head, s + src);
    const int64_t d = kv_row(a.g, a.page_table, b, head, s + tid);
    from[tid] = (f < 0 || d < 0) ? -1 : f;
    to[tid] = d;
    if (f < 0 || d < 0) atomicOr(a.status, STATUS_BAD_INDEX);
  }
  __syncthreads();
  uint4 xk[PER], xv[PER];
  float sk = 0.0f, sv = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int r = (i * 128 + tid) / Q, c = tid % Q;
    if (r < n && from[r] >= 0) {
      xk[i] = reinterpret_cast<const uint4*>(a.k + from[r] * D)[c];
      xv[i] = reinterpret_cast<const uint4*>(a.v + from[r] * D)[c];
    }
  }
  if (tid < n && from[tid] >= 0) { sk = a.ks[from[tid]]; sv = a.vs[from[tid]]; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int r = (i * 128 + tid) / Q, c = tid % Q;
    if (r < n && from[r] >= 0) {
      reinterpret_cast<uint4*>(a.k + to[r] * D)[c] = xk[i];
      reinterpret_cast<uint4*>(a.v + to[r] * D)[c] = xv[i];
    }
  }
  if (tid < n && from[tid] >= 0) { a.ks[to[tid]] = sk; a.vs[to[tid]] = sv; }
}

// Eight warps per block and a warp per four heads of a token: no loop, so that the blocks' loads and stores overlap (a grid of
// eight blocks per SM with a loop took 62.7 us where this takes 55.4 us: 32768 tokens of 8 heads of 128 read back).
unsigned row_grid(uint32_t units) { return (units + 7) / 8; }

}  // namespace

int launch_kv_append(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const float* k, const float* v, int64_t ld_k, int64_t ld_v) {
  ProfScope prof(ctx, KK_KV_APPEND);
  const uint32_t chunks = (uint32_t)(c.heads + 3) / 4, units = (uint32_t)s.B * (uint32_t)s.T * chunks;
  const KvArgs a = kv_args(ctx, c, s);
  return kv_launch(ctx, c.head_dim == 64 ? kv_append_kernel<64> : kv_append_kernel<128>, dim3(row_grid(units)), 256, 0, a, k, v, ld_k, ld_v, units, chunks);
}

int launch_kv_read(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, float* k_out, float* v_out, int64_t ld_k, int64_t ld_v) {
  ProfScope prof(ctx, KK_KV_READ);
  const uint32_t chunks = (uint32_t)(c.heads + 3) / 4, units = (uint32_t)s.B * (uint32_t)s.T * chunks;
  const KvArgs a = kv_args(ctx, c, s);
  return kv_launch(ctx, c.head_dim == 64 ? kv_read_kernel<64> : kv_read_kernel<128>, dim3(row_grid(units)), 256, 0, a, k_out, v_out, ld_k, ld_v, units, chunks);
}

int launch_kv_keep(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const int32_t* keep) {
  ProfScope prof(ctx, KK_KV_KEEP);
  const KvArgs a = kv_args(ctx, c, s);
  const unsigned grid = (unsigned)s.B * (unsigned)c.heads;
  return kv_launch(ctx, c.head_dim == 64 ? kv_keep_kernel<64> : kv_keep_kernel<128>, dim3(grid), 128, 0, a, keep);
}

}  // namespace b200q

using namespace b200q;

extern "C" {

#define KV_ORDERLY(who, reason)                                       \
  do {                                                                \
    if (const char* _r = (reason)) {                                  \
      set_error("%s: %s", who, _r);                                   \
      return 2;                                                       \
    }                                                                 \
  } while (0)

static int kv_enter(const char* who, b200q_ctx* ctx, const b200q_kv_cache* cache) {
  B200Q_REQUIRE(ctx != nullptr, "%s: null context", who);
  B200Q_REQUIRE(cache != nullptr, "%s: null cache", who);
  B200Q_REQUIRE(cache->ctx == ctx, "%s: the cache belongs to another context", who);
  B200Q_CHECK_CUDA(cudaSetDevice(ctx->device));
  return 0;
}

int b200q_kv_create(b200q_ctx* ctx, int64_t pages, int64_t page_tokens, int64_t heads, int64_t head_dim, int8_t* k_codes, int8_t* v_codes,
                    float* k_scales, float* v_scales, b200q_kv_cache** out) {
  B200Q_REQUIRE(out != nullptr, "b200q_kv_create: null out pointer");
  *out = nullptr;
  KV_ORDERLY("b200q_kv_create", kv_refuse_geometry(pages, page_tokens, heads, head_dim));
  B200Q_REQUIRE(k_codes && v_codes && k_scales && v_scales, "b200q_kv_create: null pointer");
  B200Q_REQUIRE(kv_aligned(k_codes, 16) && kv_aligned(v_codes, 16) && kv_aligned(k_scales, 16) && kv_aligned(v_scales, 16),
                "b200q_kv_create: the cache's buffers must start on 16-byte boundaries");
  B200Q_REQUIRE(ctx != nullptr, "b200q_kv_create: null context");
  B200Q_REQUIRE(!ctx->capturing, "b200q_kv_create is not allowed between b200q_graph_begin and b200q_graph_end");
  B200Q_CHECK_CUDA(cudaSetDevice(ctx->device));
  if (int e = kv_workspace(ctx)) return e;
  b200q_kv_cache* c = new (std::nothrow) b200q_kv_cache();
  B200Q_REQUIRE(c != nullptr, "b200q_kv_create: out of host memory");
  c->ctx = ctx;
  c->pages = pages;
  while ((int64_t(1) << c->page_shift) < page_tokens) c->page_shift++;
  c->heads = (int)heads;
  c->head_dim = (int)head_dim;
  c->k = k_codes; c->v = v_codes; c->ks = k_scales; c->vs = v_scales;
  *out = c;
  return 0;
}

int b200q_kv_destroy(b200q_ctx* ctx, b200q_kv_cache* cache) {
  if (!cache) return 0;
  B200Q_REQUIRE(cache->ctx == ctx, "b200q_kv_destroy: the cache belongs to another context");
  delete cache;   // the buffers are the caller's, and queued kernels hold copies of their addresses
  return 0;
}

int b200q_kv_append(b200q_ctx* ctx, b200q_kv_cache* cache, const float* k, const float* v, int64_t ld_k, int64_t ld_v, int64_t B, int64_t T,
                    const int32_t* page_table, int64_t max_pages, const int32_t* start, const int32_t* count) {
  if (int e = kv_enter("b200q_kv_append", ctx, cache)) return e;
  KV_ORDERLY("b200q_kv_append", kv_refuse_batch(B, T, cache->heads, page_table, max_pages, start));
  if (B * T == 0) return 0;
  KV_ORDERLY("b200q_kv_append", kv_refuse_array(count, 4));
  KV_ORDERLY("b200q_kv_append", kv_refuse_rows(k, ld_k, cache->heads, cache->head_dim));
  KV_ORDERLY("b200q_kv_append", kv_refuse_rows(v, ld_v, cache->heads, cache->head_dim));
  return launch_kv_append(ctx, *cache, KvBatch{(int)B, (int)T, page_table, max_pages, start, count}, k, v, ld_k, ld_v);
}

int b200q_kv_read(b200q_ctx* ctx, b200q_kv_cache* cache, int64_t B, int64_t T, const int32_t* page_table, int64_t max_pages,
                  const int32_t* start, const int32_t* count, float* k_out, float* v_out, int64_t ld_k, int64_t ld_v) {
  if (int e = kv_enter("b200q_kv_read", ctx, cache)) return e;
  KV_ORDERLY("b200q_kv_read", kv_refuse_batch(B, T, cache->heads, page_table, max_pages, start));
  if (B * T == 0) return 0;
  KV_ORDERLY("b200q_kv_read", kv_refuse_array(count, 4));
  KV_ORDERLY("b200q_kv_read", kv_refuse_rows(k_out, ld_k, cache->heads, cache->head_dim));
  KV_ORDERLY("b200q_kv_read", kv_refuse_rows(v_out, ld_v, cache->heads, cache->head_dim));
  return launch_kv_read(ctx, *cache, KvBatch{(int)B, (int)T, page_table, max_pages, start, count}, k_out, v_out, ld_k, ld_v);
}

int b200q_kv_attention(b200q_ctx* ctx, b200q_kv_cache* cache, const float* q, int64_t ld_q, int64_t B, int64_t T, int64_t H,
                       const int32_t* page_table, int64_t max_pages, const int32_t* start, const int32_t* count, const uint64_t* tree,
                       float scale, float* out, int64_t ld_out) {
  if (int e = kv_enter("b200q_kv_attention", ctx, cache)) return e;
  B200Q_REQUIRE(H > 0 && H <= 65535 && H % cache->heads == 0, "b200q_kv_attention: %lld heads are not a multiple of the cache's %d (or above 65535)",
                (long long)H, cache->heads);
  KV_ORDERLY("b200q_kv_attention", kv_refuse_batch(B, T, H, page_table, max_pages, start));
  B200Q_REQUIRE(tree == nullptr || T <= KV_MAX_TREE, "b200q_kv_attention: a tree has at most %d drafted tokens (got %lld)", KV_MAX_TREE, (long long)T);
  B200Q_REQUIRE(std::isfinite(scale), "b200q_kv_attention: the scale must be finite");
  if (B * T == 0) return 0;
  KV_ORDERLY("b200q_kv_attention", kv_refuse_array(count, 4));
  KV_ORDERLY("b200q_kv_attention", kv_refuse_array(tree, 8));
  KV_ORDERLY("b200q_kv_attention", kv_refuse_rows(q, ld_q, H, cache->head_dim));
  KV_ORDERLY("b200q_kv_attention", kv_refuse_rows(out, ld_out, H, cache->head_dim));
  return launch_kv_attention(ctx, *cache, KvBatch{(int)B, (int)T, page_table, max_pages, start, count}, q, ld_q, (int)H, tree, scale, out, ld_out);
}

int b200q_kv_keep(b200q_ctx* ctx, b200q_kv_cache* cache, int64_t B, int64_t T, const int32_t* page_table, int64_t max_pages,
                  const int32_t* start, const int32_t* keep, const int32_t* count) {
  if (int e = kv_enter("b200q_kv_keep", ctx, cache)) return e;
  KV_ORDERLY("b200q_kv_keep", kv_refuse_batch(B, T, cache->heads, page_table, max_pages, start));
  B200Q_REQUIRE(T <= KV_MAX_TREE, "b200q_kv_keep: at most %d rows per sequence (got %lld)", KV_MAX_TREE, (long long)T);
  if (B * T == 0) return 0;
  KV_ORDERLY("b200q_kv_keep", kv_refuse_array(count, 4));
  B200Q_REQUIRE(keep != nullptr, "b200q_kv_keep: null pointer");
  KV_ORDERLY("b200q_kv_keep", kv_refuse_array(keep, 4));
  return launch_kv_keep(ctx, *cache, KvBatch{(int)B, (int)T, page_table, max_pages, start, count}, keep);
}

}  // extern "C"

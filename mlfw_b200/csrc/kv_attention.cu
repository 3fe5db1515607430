// Attention over the int8 key/value cache: softmax(scale * q k^T) v for new rows of a batch of sequences.
//
// Row t of sequence b sees the start[b] positions cached before and, of the count[b] new ones, those up to itself (no
// tree) or those whose bit is set in its row of ancestors.  Query heads h of a group H / heads share cache head h / (H / heads).
#include "kernels.cuh"
#include "kv.cuh"

namespace b200q {

namespace {

struct AttnArgs {
  KvGeom g;
  const int8_t *k, *v;
  const float *ks, *vs;
  const int32_t *page_table, *start, *count;
  const uint64_t* tree;
  const float* q;
  float* out;
  int64_t ld_q, ld_o;
  int B, T, H, group;
  float scale;
  uint32_t* status;
};

// One block per (sequence, row, query head), one warp per cached token: the plain formula in one pass over the cache.
template <int D>
__global__ void __launch_bounds__(128) kv_attention_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float part[4][D + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t bt = blockIdx.x / a.H;
  const int h = blockIdx.x % a.H, b = (int)(bt / a.T), t = (int)(bt % a.T);
  const int n = kv_rows_in_use(a.count, b, a.T);
  if (t >= n) return;
  const int64_t first = a.start[b];
  const uint64_t seen = a.tree ? a.tree[bt] : 0;
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; e++) { q[e] = a.q[bt * a.ld_q + (int64_t)h * D + lane * E + e] * a.scale; o[e] = 0.0f; }
  float m = __int_as_float(0xff800000), l = 0.0f;
  for (int64_t pos = warp; pos < first + (a.tree ? n : t + 1); pos += 4) {
    if (pos >= first && a.tree && !((seen >> (pos - first)) & 1)) continue;
    const int64_t row = kv_row(a.g, a.page_table, b, h / a.group, pos);
    if (row < 0) {
      if (lane == 0) atomicOr(a.status, STATUS_BAD_INDEX);
      continue;
    }
    float z = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) z = fmaf(q[e], (float)a.k[row * D + lane * E + e], z);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) z += __shfl_xor_sync(0xffffffffu, z, s);
    z *= a.ks[row];
    const float top = fmaxf(m, z), old = expf(m - top), p = expf(z - top);
    l = l * old + p;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = fmaf(p * a.vs[row], (float)a.v[row * D + lane * E + e], o[e] * old);
    m = top;
  }
#pragma unroll
  for (int e = 0; e < E; e++) part[warp][lane * E + e] = o[e];
  if (lane == 0) { part[warp][D] = m; part[warp][D + 1] = l; }
  __syncthreads();
  float top = part[0][D];
  for (int w = 1; w < 4; w++) top = fmaxf(top, part[w][D]);
  if (threadIdx.x < D) {
    float sum = 0.0f, val = 0.0f;
    for (int w = 0; w < 4; w++) {
      if (part[w][D + 1] == 0.0f) continue;
      const float f = expf(part[w][D] - top);
      sum += f * part[w][D + 1];
      val += f * part[w][threadIdx.x];
    }
    a.out[bt * a.ld_o + (int64_t)h * D + threadIdx.x] = sum == 0.0f ? 0.0f : val / sum;
  }
}

}  // namespace

int launch_kv_attention(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const float* q, int64_t ld_q, int H, const uint64_t* tree,
                        float scale, float* out, int64_t ld_o) {
  ProfScope prof(ctx, KK_KV_ATTENTION);
  const AttnArgs a{KvGeom{c.pages, s.max_pages, c.page_shift, c.heads}, c.k, c.v, c.ks, c.vs, s.page_table, s.start, s.count, tree, q, out,
                   ld_q, ld_o, s.B, s.T, H, H / c.heads, scale, ctx->status_dev};
  const unsigned grid = (unsigned)s.B * (unsigned)s.T * (unsigned)H;
  if (c.head_dim == 64) kv_attention_kernel<64><<<grid, 128, 0, ctx->stream>>>(a);
  else kv_attention_kernel<128><<<grid, 128, 0, ctx->stream>>>(a);
  ctx->launches++;
  B200Q_CHECK_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace b200q

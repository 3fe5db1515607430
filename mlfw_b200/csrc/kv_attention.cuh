// Attention over the int8 key/value cache: softmax(scale * q k^T) v for new rows of a batch of sequences.
//
// Row t of sequence b sees the start[b] positions cached before and, of the count[b] new ones, those up to itself (no
// tree) or those whose bit is set in its row of ancestors.  Query heads h of a group H / heads share cache head h / (H / heads).
//
// The arithmetic.  A cached value is code * scale with an integer |code| <= 128.  The codes go into the tensor cores as they
// are; queries and weights, which are binary32, are split into parts that the tensor cores take, so the cache is never dequantized
// and the result is as near as binary32 arithmetic comes: 3e-7 to 8e-7 of the largest output against binary64 on
// ordinary rows.  What each form holds in fewer bits is said with it:
//   Many rows (kv_attention_umma.cu), binary16 products, two per contraction.  A query row is scaled by a power of two to
//   x = q * 2^(14 - e) with 2^e <= max|q| < 2^(e+1), and an element is its rounding to binary16 and the rounding of what is left: 22
//   bits of its own down to 2^-17 of the row's largest, 2^-40 of the largest below that (a fixed point against the largest, tried
//   first, left an element beside one 2000 times as large 11 bits).  sum_d q_d code_d = 2^(e-14) * (sum lo code + sum hi code), in one
//   binary32 sum with the small parts first.  A weight is split the same way, the largest below 2^15.
//   Sums over tiles of 64 tokens are binary32 additions one after another, of the outputs and of p: n / 64 roundings.
//   Few rows (kv_attention.cu), integer products: queries and weights as 32-bit fixed-point numbers in four 8-bit digits, sums
//   in 32-bit integers, exact.  An element of a query row is held to 2^-31 of the row's largest (an element 2^-10 of the largest has 21
//   bits; below a largest of 1e-31 there are fewer), a weight times its scale to 2^-28 of the row's largest, with a rounding that keeps the
//   sum of many smaller ones; sums of p carry their rounding along.
// ex2.approx adds 2^-22 to a weight, and so does the rounding of z - c where c is 8 or more: c holds log2 of V's scale in the
// form for many rows, which makes it 2.5e-6 for values of V near 1e37 or 1e-35.  With z the score in units of log2 and the row's running
//     c = max over the keys of (z + log2 scale_v) - a constant,      p = 2^(z - c),      w = p * scale_v,
// the row's result is sum w code / sum p, so one running number per row replaces the softmax's maximum and the weights'
// exponent, and a key whose score is high but whose scale is small (or the other way round) costs no precision.  log2 of
// the scale only steers c, so the approximate one does; it is held from below, which keeps p inside binary32.
#pragma once
#include "kernels.cuh"
#include "kv.cuh"
namespace b200q {

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
  float scale_log2e;       // scale * log2(e): scores are kept in units of log2
  uint32_t* status;
  uint32_t* counters;      // pieces of an item that have arrived, by the run the item begins in; zero between launches
  float* slots;
  int4* items;             // the item that begins in a run and goes on behind it: (e, head, last run, 1), else w = 0
};

int launch_kv_attention_many(b200q_ctx* ctx, const AttnArgs& a, int D);   // kv_attention_umma.cu

namespace {

constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float C_NONE = -3.0e38f;       // c of a row that has seen nothing: finite, so that differences with it are numbers
constexpr float C_SEEN = -1.0e38f;       // ... and of a row that has seen something it is above this
constexpr float FAR = 0x1p20f;           // scores are taken relative to a score of the row when they are further from zero

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float log2_raw(float s) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return r;
}
__device__ __forceinline__ float log2_scale(float s) { return fmaxf(log2_raw(s), -103.0f); }
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}
// Bytes 0 and 2 (even) or 1 and 3 (odd) of a word of codes as two binary16 numbers: the byte with its sign bit flipped
// under the exponent of 1024 is 1024 + 128 + code; subtracting 1152 is exact.
__device__ __forceinline__ uint32_t codes_even(uint32_t x) {
  const uint32_t y = (x & 0x00ff00ffu) ^ 0x64806480u;
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(y), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t x) { return codes_even(x >> 8); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {   // lo in the low half
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two numbers as binary16 halves: the rounded values and what is left of them (exact before its own rounding).
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16(x0, x1);
  float y0, y1;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(y0), "=f"(y1) : "r"(hi));
  lo = pack_f16(__fsub_rn(x0, y0), __fsub_rn(x1, y1));
}
__device__ __forceinline__ float pow2(int e) {   // 2^e for -126 <= e <= 127
  return __int_as_float((e + 127) << 23);
}

// Where a query row comes from and its result goes: row R of the sequence (R = t * group + head within the group).
__device__ __forceinline__ int64_t row_offset(const AttnArgs& a, int b, int head, int R, int64_t ld, int D, int& t) {
  t = R / a.group;
  return ((int64_t)b * a.T + t) * ld + (int64_t)(head * a.group + (R - t * a.group)) * D;
}

// The run of tiles this block works on: total tiles, the item its first tile belongs to (e = sequence * row
// blocks + row block, head) and the tile inside it.  All threads take part and get the same answer.
struct Run {
  KvRuns all;
  int64_t begin, end;
  int e, head, tile;
};
// ROWS query rows per item, TILE tokens per tile, at least LEAST tiles per run: a shorter one costs more in joining than it saves.
// WHOLE: where an item has at most 32 tiles on average, that many (4 or more), so that with little work items of one length fall
// into one run each and nothing is joined between blocks.
template <int ROWS, int TILE, int LEAST, bool WHOLE>
__device__ __forceinline__ Run find_run(const AttnArgs& a, int row_blocks) {
  __shared__ int64_t warp_sum[32];
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t E = (uint32_t)(a.B * row_blocks), per = (E + blockDim.x - 1) / blockDim.x;   // E < 2^31
  const int e0 = (int)min(E, (uint32_t)tid * per), e1 = (int)min(E, (uint32_t)(tid + 1) * per);
  auto tiles = [&](int e) {
    const int b = e / row_blocks;
    return (int64_t)kv_tiles(a.g, a.start[b], kv_rows_in_use(a.count, b, a.T), a.group, ROWS, e - b * row_blocks, a.tree != nullptr, TILE) * a.g.heads;
  };
  int64_t mine = 0;
  for (int e = e0; e < e1; e++) mine += tiles(e);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;                                // of the warps before this one, and of all
#pragma unroll 4
  for (int w = 0; w < (int)blockDim.x / 32; w++) {
    const int64_t x = warp_sum[w];
    if (w < warp) before += x;
    total += x;
  }
  Run r;
  r.begin = r.end = 0;
  if (total == 0) return r;
  const int64_t mean = WHOLE ? kv_div(total, (int64_t)E * a.g.heads) : 0;
  const int least = WHOLE && mean <= 32 ? max((int)mean, 4) : LEAST;
  r.all = kv_runs(total, least, (int)gridDim.x);
  if ((int)blockIdx.x >= r.all.runs) return r;
  r.begin = kv_run_begin(r.all, (int)blockIdx.x);
  r.end = kv_run_begin(r.all, (int)blockIdx.x + 1);
  int64_t at = before + incl - mine;
  if (r.begin >= at && r.begin < at + mine) {
    int e = e0;
    int64_t n = tiles(e);
    while (r.begin >= at + n) { at += n; n = tiles(++e); }
    const int64_t per_head = kv_div(n, a.g.heads), in = r.begin - at, head = kv_div(in, per_head);
    found[0] = e; found[1] = (int)head; found[2] = (int)(in - head * per_head);
  }
  __syncthreads();
  r.e = found[0]; r.head = found[1]; r.tile = found[2];
  return r;
}

}  // namespace

}  // namespace b200q

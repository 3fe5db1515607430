// Attention over the int8 key/value cache for many query rows (chunks of a prompt, drafted trees) on the 5th-generation
// tensor cores.  What is computed and in which arithmetic stands in kv_attention.cuh.
#include "kv_attention.cuh"

namespace b200q {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// One block per SM walks a run of 64-token tiles; an item is up to 128 rows, the 128 lanes of tensor memory.  Roles:
//   three staging warps: K and V of a tile from the cache into a ring in shared memory as binary16 tiles of the tensor cores'
//     layout (V transposed), with the tokens' scales beside them, in units of sixteen tokens, which always share a page
//     (three, so that the block has 20 warps and 96 registers per thread: where the first case below took 108 us, two
//     staging warps took 127, four, which leave 80 registers, 126);
//   one thread issues the products: S = Q_lo K^T + Q_hi K^T (tcgen05.mma kind::f16, 128 x 64) of tile j + 1, then
//     O = P_lo V + P_hi V of tile j with the weights read from tensor memory;
//   sixteen softmax warps, four threads per row with sixteen tokens of a tile each: scores from tensor memory, the row's c
//     agreed on through shared memory, the weights' two halves written over the scores, and tile j - 1's O folded into a
//     quarter of the row's outputs per thread in registers: o = o * 2^(c_old - c_new) + O.  Sums over tiles are binary32
//     additions, not the tensor core's.
// Scores and O are double-buffered (384 columns of tensor memory), so products, softmax and staging of neighbouring tiles
// overlap.  Measured: two prompts' chunks of 512 rows behind up to 4000 cached tokens, 16 heads on 4, 128 wide (26 GFLOP, twice
// that in binary16 products): 110 to 123 us from run to run (median 122) with the join, whose 27 MB between L2 and the SMs take 9;
// the step with eight drafted trees of 31 over up to 5000 tokens, 32 heads on 8, 92 to 100 with its four other launches.  Bound by the softmax warps: 192 000
// cycles of an SM for 45 tiles of 64 tokens, 4200 per tile with what a piece costs, in which the tensor pipe is busy for 24 %
// (1000; the arithmetic alone is 512).  10 000 warp instructions per tile, 2.4 issued per cycle of an SM, the rest
// their latency (the scores' load from tensor memory, the row's meeting, the split and the store of the weights).  The softmax role
// has no registers left: for D = 128 the kernel spills 72 bytes of stores and 172 (176 with CS = 2) of loads.  Not kept
// (against 110 us on the same box): scores three tiles ahead 136 (far more spills), Q in tensor memory with a
// single O 117; the two parts of the scores in columns of their own, added by the softmax warps, 110 against 107.7; a
// hardware barrier for the row's meeting 107.0 against 107.7, not worth a wait without a limit; two tokens per instruction
// (f32x2) for scores, weights and outputs 120 against 114 (the pairs want aligned registers).
//
// With 64 or fewer rows (CS = 2) the lanes hold two copies of the rows, each copy takes half of a thread's tokens and has
// weights of zero elsewhere, and the copies are joined at the end: the softmax work, which would leave lanes idle,
// shrinks with the rows.
//
// Every wait is bounded: one that runs out raises the block's abort flag and STATUS_SDPA_WAIT_TIMEOUT, all roles leave,
// products in flight get 2 ms, tensor memory is freed.  Threads meet at mbarriers only, never at a hardware barrier that
// a role that has left would keep the others waiting at; the one at the end is reached by all.
// ---------------------------------------------------------------------------------------------------------------
constexpr int MT = 64, LANES = 128, SOFT_WARPS = 16, STAGE_WARPS = 3, MANY_THREADS = 32 * (SOFT_WARPS + STAGE_WARPS + 1);
template <int D>
struct Many {
  static constexpr int Q_BLOCK = LANES * 128, Q_BYTES = (D / 64) * Q_BLOCK;    // K blocks of 64 dimensions: [128 rows][128 B]
  static constexpr int K_BLOCK = MT * 128, K_BYTES = (D / 64) * K_BLOCK, V_BYTES = D * 128;
  static constexpr int STAGES = 4, STAGE = K_BYTES + V_BYTES;
  static constexpr int QHI = 0, QLO = Q_BYTES, RING = 2 * Q_BYTES, END = RING + STAGES * STAGE;
  static constexpr int SMEM = END + 1024;
};
// Weights stay below 2^15 for any scale of V: p is up to 2^118 where the scale is 2^-103 or less, 2^-106 where it is the
// largest there is.  Sums of p times this stay inside binary32 at both ends: 2^24 keys of the one, a single key of the other.
constexpr float L_UNIT = 0x1p-14f;
// columns: scores of even and odd tiles, the weights over them; O of even and odd tiles
constexpr int TM_S = 0, TM_S_STEP = 64, TM_O = 128, TM_O_STEP = 128, TM_COLS = 512;

__device__ __forceinline__ uint64_t gtimer() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Byte offset of (row, byte column) inside a [rows][128 B] tile with the 128-byte swizzle (16-byte pieces XOR row % 8).
__device__ __forceinline__ uint32_t sw128(int row, int byte_col) {
  return (uint32_t)(row * 128 + ((((byte_col >> 4) ^ (row & 7)) << 4) | (byte_col & 15)));
}
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {   // K-major, 128-byte swizzle, groups of 8 rows 1024 B apart
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16: D = F32 (1), A = B = F16 (0), both K-major.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Loads from tensor memory: consecutive columns of this warp's lanes.  The wait stands in the same statement: registers that a
// separate one ties to the wait get copied.
__device__ __forceinline__ void tm_ld(uint32_t at, uint32_t (&x)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]),
                 "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]),
                 "=r"(x[19]), "=r"(x[20]), "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]),
                 "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
               : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_ld(uint32_t at, uint32_t (&x)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]),
                 "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
               : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_ld(uint32_t at, uint32_t (&x)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7])
               : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_st(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

// Whether the phase is over; suspends the thread for up to a microsecond while it is not.
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(done) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
  return done != 0;
}

struct ManyParams {
  int row_blocks;
  uint32_t polls;          // bound of every wait
};

// The block's barriers and flags.  Counts: one arrival per warp (after __syncwarp) or per tcgen05.commit.
template <int STAGES>
struct ManyShared {
  uint64_t full[STAGES], empty[STAGES];        // ring slots: staged (4 units), consumed (commit of the tile's P V)
  uint64_t scores[2], weights[2], outputs[2];  // S ready (commit), P ready (16 warps), O ready (commit)
  uint64_t queries, soft;                      // Q staged (16 warps); meeting of the softmax warps (16 warps)
  uint64_t rows[4];                            // meeting of the four warps that share a quarter of the lanes
  uint32_t tmem;
  int abort;
  static constexpr uint32_t FULL = 0, EMPTY = 8 * STAGES, SCORES = 16 * STAGES, WEIGHTS = SCORES + 16, OUTPUTS = WEIGHTS + 16, QUERIES = OUTPUTS + 16,
                            SOFT = QUERIES + 8, ROWS = SOFT + 8;   // places of the members
};

// Pieces of a block's run, one after another: every role walks them by itself.
template <int ROWS>
struct Walk {
  int64_t left, at, first, vis;
  int e, head, tile0, tile1, tiles, b, rb, n, rows_here;
  __device__ __forceinline__ bool open(const AttnArgs& a, int row_blocks) {
    while (left > 0) {
      b = e / row_blocks; rb = e - b * row_blocks;
      first = a.start[b];
      n = kv_rows_in_use(a.count, b, a.T);
      tiles = kv_tiles(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr, MT);
      if (tiles != 0) {
        vis = kv_visible(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr);
        tile1 = (int)min((int64_t)tiles, tile0 + left);
        rows_here = min(ROWS, n * a.group - rb * ROWS);
        return true;
      }
      e++; head = 0; tile0 = 0;
    }
    return false;
  }
  __device__ __forceinline__ void close(const AttnArgs& a) {
    at += tile1 - tile0;
    left -= tile1 - tile0;
    tile0 = 0;
    if (++head == a.g.heads) { head = 0; e++; }
  }
};

// Row of the V tile that holds dimension 4 L + q, so that a thread's D / 4 columns of O are whole runs of four dimensions and
// lanes that stage neighbouring L write rows of different banks (D = 64: the halves of odd quarters change places).
template <int D>
__device__ __forceinline__ int v_row(int L, int q) {
  constexpr int W = D / 16;                                      // words of a quarter of a row
  const int r = q * W + L % W;
  return (L / W) * (D / 4) + (D == 64 ? r ^ (((L / W) & 1) * 4) : r);
}

// A row of a piece whose scores are not within FAR of zero, where binary32 has no room beside them for log2 scale_v: token by token, with
// the scores relative to their maximum m and sums in binary64.  The tensor cores' path leaves such a row with a c outside
// (-FAR, FAR] and whatever it came to; no real model has one, so this is made to be right, not fast.  A warp holds a
// row's D / 4 pieces of four dimensions in neighbouring lanes (two rows for D = 64); v and sum in units of 2^(m + c), sum times L_UNIT.
template <int D>
struct FarRow {
  float4 v;
  float sum, c, m;
};
template <int D, int ROWS>
__device__ __forceinline__ FarRow<D> far_row(const AttnArgs& a, int b, int head, int rb, int r, int tile0, int tile1, int p, bool asked) {
  auto over_row = [](auto x, auto f) {
#pragma unroll
    for (int o = 1; o < D / 4; o <<= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  };
  FarRow<D> y;
  y.v = make_float4(0.f, 0.f, 0.f, 0.f);
  y.sum = 0.0f; y.c = -FAR; y.m = 0.0f;
  // most rows that come here just see nothing of the piece: it begins behind them
  int t;
  const float* src = a.q + row_offset(a, b, head, rb * ROWS + r, a.ld_q, D, t);
  const int64_t first = a.start[b], lo = (int64_t)tile0 * MT - first;
  const int rows = kv_rows_in_use(a.count, b, a.T);
  uint64_t seen = a.tree ? a.tree[(int64_t)b * a.T + t] : 0;
  if (rows < 64) seen &= (1ull << rows) - 1;
  if (!__any_sync(0xffffffffu, asked && (lo < 0 || (a.tree ? lo < 64 && (seen >> lo) != 0 : lo <= t)))) return y;
  const float4 q = __ldcg(reinterpret_cast<const float4*>(src) + p);
  const float big = over_row(fmaxf(fmaxf(fabsf(q.x), fabsf(q.y)), fmaxf(fabsf(q.z), fabsf(q.w))), [](float x, float y) { return fmaxf(x, y); });
  const int ex = max(__float_as_int(big) >> 23, 24) - 127;
  const float up = pow2(14 - ex), rs = a.scale_log2e * pow2(ex - 14);
  const float x[4] = {q.x * up, q.y * up, q.z * up, q.w * up};
  const int32_t* table = a.page_table + (int64_t)b * a.g.max_pages;
  float m = NEG_INF;
  double l = 0.0, n[4] = {0.0, 0.0, 0.0, 0.0};
  const int64_t end = min((int64_t)tile1 * MT, kv_visible(a.g, first, rows, a.group, ROWS, rb, a.tree != nullptr));   // inside the page table
#pragma unroll 1
  for (int64_t pos = (int64_t)tile0 * MT; pos < end; pos += 4) {
    const int page = __ldcg(table + (pos >> a.g.page_shift));
    if ((uint32_t)page >= (uint32_t)a.g.pages) continue;
    const int64_t cell = (((int64_t)page * a.g.heads + head) << a.g.page_shift) + (pos & ((1 << a.g.page_shift) - 1));
    float z[4], vs[4], top = NEG_INF;
    uint32_t vc[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t k = __ldcg(reinterpret_cast<const uint32_t*>(a.k + (cell + i) * D) + p);
      vc[i] = __ldcg(reinterpret_cast<const uint32_t*>(a.v + (cell + i) * D) + p);
      const float ks = __ldcg(a.ks + cell + i);
      vs[i] = __ldcg(a.vs + cell + i);
      float dot = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; c++) dot = fmaf(x[c], (float)(int8_t)(k >> (8 * c)), dot);
      dot = over_row(dot, [](float y, float u) { return y + u; });
      const int64_t j = pos + i - first;
      const bool sees = pos + i < end && (j < 0 || (a.tree ? j < 64 && ((seen >> j) & 1) : j <= t));
      z[i] = sees ? dot * (ks * rs) : NEG_INF;
      top = fmaxf(top, z[i]);
    }
    if (top > m) {
      const double f = ex2(m - top);
      l *= f;
#pragma unroll
      for (int c = 0; c < 4; c++) n[c] *= f;
      m = top;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (z[i] > NEG_INF) {
        const float e = ex2(z[i] - m);
        l += e;
#pragma unroll
        for (int c = 0; c < 4; c++) n[c] += (double)e * ((double)vs[i] * (double)(int8_t)(vc[i] >> (8 * c)));
      }
    }
  }
  int e = -2000;                                                 // exponent of the largest
#pragma unroll
  for (int c = 0; c < 4; c++) e = max(e, ((__double2hiint(n[c]) >> 20) & 0x7ff) - 1023);
  e = over_row(e, [](int u, int v) { return max(u, v); });
  if (m > NEG_INF) {
    const int c = max(e - 24, -90);
    const double s = __hiloint2double((1023 - c) << 20, 0);
    y.v = make_float4((float)(n[0] * s), (float)(n[1] * s), (float)(n[2] * s), (float)(n[3] * s));
    y.sum = (float)(l * s * (double)L_UNIT);
    y.c = (float)c;
    y.m = m;
  }
  return y;
}

template <int D, int CS>
__global__ void __launch_bounds__(MANY_THREADS, 1) kv_attention_many_kernel(const AttnArgs a, const ManyParams mp) {
  using C = Many<D>;
  using S = ManyShared<C::STAGES>;
  constexpr int ROWS = LANES / CS, NC = 16 / CS, QD = D / 4, ST = C::STAGES;   // rows of an item; tokens of a tile and outputs of a thread
  extern __shared__ uint8_t smem_raw[];
  __shared__ ManyShared<ST> sh;
  __shared__ float top_x[2][4][LANES], sum_x[4][LANES], c_x[LANES];
  __shared__ __align__(16) float tok_ks[ST][MT], tok_vs[ST][MT], tok_lv[ST][MT];
  __shared__ uint32_t tok_there[ST][4];                          // which of a warp's sixteen tokens anybody sees
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sm_base = smem_u32(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  asm volatile("griddepcontrol.wait;" ::: "memory");             // the previous kernel of the stream wrote what is read here
  const Run run = find_run<ROWS, MT, 2, false>(a, mp.row_blocks);
  if (tid == 0) a.items[blockIdx.x] = make_int4(0, 0, 0, 0);
  if (run.begin == run.end) return;

  if (tid == 0) {
    for (int s = 0; s < ST; s++) { mbar_init(smem_u32(&sh.full[s]), 4); mbar_init(smem_u32(&sh.empty[s]), 1); }
    for (int s = 0; s < 2; s++) { mbar_init(smem_u32(&sh.scores[s]), 1); mbar_init(smem_u32(&sh.weights[s]), SOFT_WARPS); mbar_init(smem_u32(&sh.outputs[s]), 1); }
    mbar_init(smem_u32(&sh.queries), SOFT_WARPS);
    mbar_init(smem_u32(&sh.soft), SOFT_WARPS);
    for (int s = 0; s < 4; s++) mbar_init(smem_u32(&sh.rows[s]), 4);
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == SOFT_WARPS + STAGE_WARPS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"((uint32_t)TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  __syncthreads();
  fence_after();
  // Only now may the next kernel's blocks come: one that allocates tensor memory before its own wait must not take what
  // a block of this grid still needs.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = sh.tmem;
  volatile int* abort_flag = &sh.abort;
  const uint32_t sh_base = smem_u32(&sh);

  // Waits for a phase of a barrier (given by its place in `sh`), mp.polls times a microsecond at most.
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    if (mbar_try(sh_base + bar, parity)) return true;
    for (uint32_t n = mp.polls; n != 0; n--) {
      if (mbar_try(sh_base + bar, parity)) return true;
      if (*abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
  };

  Walk<ROWS> w;
  w.left = run.end - run.begin; w.at = run.begin; w.e = run.e; w.head = run.head; w.tile0 = run.tile;
  bool alive = true;
  uint32_t it = 0;                                               // tiles of the run so far

  if (warp < SOFT_WARPS) {
    // ------------------------------------------------------------------------------------------------ softmax
    const int quarter = warp & 3, cg = warp >> 2, row = quarter * 32 + lane;
    const int copy = row / ROWS, rq = row % ROWS;                // which copy of which row of the item
    const int col0 = cg * 16 + copy * NC;                        // this thread's tokens of a tile
    const uint32_t lane_tm = tmem + ((uint32_t)(quarter * 32) << 16);
    uint32_t soft_phase = 0, rows_phase = 0;
    auto meet = [&](uint32_t bar, uint32_t& phase) -> bool {     // all warps of the barrier; shared memory before it is seen after it
      __syncwarp();
      if (lane == 0) mbar_arrive(sh_base + bar);
      const bool ok = wait(bar, phase);
      phase ^= 1u;
      return __all_sync(0xffffffffu, ok);
    };
    while (alive && w.open(a, mp.row_blocks)) {
      if (tid == 0 && (w.first < 0 || w.first + w.n > (a.g.max_pages << a.g.page_shift))) atomicOr(a.status, STATUS_BAD_INDEX);
      // ---- the query row: this thread's quarter of it, below 2^15, in two binary16 parts
      float rs;
      int row_t;
      uint64_t row_seen;
      {
        const bool used = rq < w.rows_here;
        int t;
        const float* src = a.q + row_offset(a, w.b, w.head, w.rb * ROWS + (used ? rq : 0), a.ld_q, D, t) + cg * QD;
        row_t = used ? t : -1;
        row_seen = used && a.tree ? a.tree[(int64_t)w.b * a.T + t] : 0;
        if (w.n < 64) row_seen &= (1ull << w.n) - 1;
        float4 x[QD / 4];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < QD / 4; i++) {
          x[i] = used ? __ldcg(reinterpret_cast<const float4*>(src) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
          top = max(max(top, max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu)),
                    max(__float_as_uint(x[i].z) & 0x7fffffffu, __float_as_uint(x[i].w) & 0x7fffffffu));
        }
        sum_x[cg][row] = __uint_as_float(top);
        alive = meet(S::ROWS + 8 * quarter, rows_phase);
        if (!alive) break;
#pragma unroll
        for (int k = 0; k < 4; k++) top = max(top, __float_as_uint(sum_x[k][row]));
        const bool finite = top < 0x7f800000u;
        const int ex = max((int)(top >> 23), 24) - 127;
        // rs is kept positive, so that a masked x = -Inf stays -Inf: a negative scale turns the query's sign, a zero one zeroes it
        const float up = a.scale_log2e == 0.0f ? 0.0f : copysignf(pow2(14 - ex), a.scale_log2e);
        rs = finite ? fmaxf(fabsf(a.scale_log2e) * pow2(ex - 14), 1e-45f) : __int_as_float(0x7fc00000);
#pragma unroll
        for (int i = 0; i < QD / 4; i += 2) {                    // eight dimensions: 16 bytes of either half, in the order of staged K
          uint32_t h[4], l[4];
          const float y[8] = {x[i].x, x[i].y, x[i].z, x[i].w, x[i + 1].x, x[i + 1].y, x[i + 1].z, x[i + 1].w};
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int e = (c & 1) + 4 * (c >> 1);
            split_f16(finite ? y[e] * up : 0.0f, finite ? y[e + 2] * up : 0.0f, h[c], l[c]);
          }
          const int dim = cg * QD + i * 4;
          const uint32_t to = sm_base + (dim >> 6) * C::Q_BLOCK + sw128(row, (dim & 63) * 2);
          sts128(to + C::QHI, h[0], h[1], h[2], h[3]);
          sts128(to + C::QLO, l[0], l[1], l[2], l[3]);
        }
        fence_proxy();                                           // the tensor cores read what the threads wrote
        __syncwarp();
        if (lane == 0) mbar_arrive(sh_base + S::QUERIES);
      }

      float o[QD];                                               // outputs, in the order of the V tile's rows
#pragma unroll
      for (int i = 0; i < QD; i++) o[i] = 0.0f;
      float c_run = -FAR, l_run = 0.0f, fold = 0.0f;             // fold: the factor that goes with the latest tile's O
      auto take_outputs = [&](uint32_t t) -> bool {              // o = o * fold + O of tile t
        if (!__all_sync(0xffffffffu, wait(S::OUTPUTS + 8 * (t & 1), (t >> 1) & 1))) return false;
        fence_after();
        uint32_t x[QD];
        tm_ld(lane_tm + TM_O + (t & 1) * TM_O_STEP + cg * QD, x);
#pragma unroll
        for (int i = 0; i < QD; i++) o[i] = fmaf(o[i], fold, __uint_as_float(x[i]));
        return true;
      };

      const int j0 = w.tile0, j1 = w.tile1, plain = w.first <= 0 ? 0 : (int)(w.first / MT);   // tiles of cached tokens only
#pragma unroll 1
      for (int j = j0; j < j1; j++, it++) {
        const uint32_t buf = it & 1, slot = it % ST;
        const uint32_t s_tm = lane_tm + TM_S + buf * TM_S_STEP;
        // the slot's tokens (the staging warps' stores) and the scores
        bool ok = wait(S::FULL + 8 * slot, (it / ST) & 1) && wait(S::SCORES + 8 * buf, (it >> 1) & 1);
        alive = __all_sync(0xffffffffu, ok);
        if (!alive) break;
        fence_after();
        uint32_t sc[NC];
        tm_ld(s_tm + col0, sc);

        // which of this thread's tokens its row sees
        uint32_t seen = tok_there[slot][cg];
        const bool all = j < plain && seen == 0xffffu;           // the same in the whole warp
        if (!all) {
          const int64_t from = (int64_t)j * MT + cg * 16 - w.first;   // place of the first of the sixteen tokens among the new rows
          if (from + 16 > 0) {
            const uint32_t before = from >= 0 ? 0u : (1u << (int)-from) - 1;
            uint32_t fresh;
            if (a.tree) fresh = from >= 64 ? 0u : (from >= 0 ? (uint32_t)(row_seen >> (int)from) : (uint32_t)(row_seen << (int)-from));
            else {
              const int64_t k = (int64_t)row_t + 1 - from;       // tokens up to the row itself
              fresh = k <= 0 ? 0u : (k >= 16 ? 0xffffu : (1u << (int)k) - 1);
            }
            seen &= before | fresh;
          }
          seen >>= copy * NC;
        }

        // x = S * scale_k, the score z = x * rs
        float x[NC], u[NC], top = NEG_INF;
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
          const float4 k = *reinterpret_cast<const float4*>(&tok_ks[slot][col0 + i]), v = *reinterpret_cast<const float4*>(&tok_lv[slot][col0 + i]);
          const float kk[4] = {k.x, k.y, k.z, k.w}, vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int c = 0; c < 4; c++) {
            x[i + c] = __uint_as_float(sc[i + c]) * kk[c];
            u[i + c] = fmaf(x[i + c], rs, vv[c]);
          }
        }
        if (!all) {
#pragma unroll
          for (int i = 0; i < NC; i++)
            if (!((seen >> i) & 1)) x[i] = u[i] = NEG_INF;
        }
#pragma unroll
        for (int i = 0; i < NC; i += 2) top = fmaxf(fmaxf(top, u[i]), u[i + 1]);
        // the row's other tokens: warps with the same lanes (slots alternate, so one meeting per tile does)
        top_x[buf][cg][row] = top;
        alive = meet(S::ROWS + 8 * quarter, rows_phase);
        if (!alive) break;
#pragma unroll
        for (int k = 0; k < 4; k++) top = fmaxf(top, top_x[buf][k][row]);
        const float c_new = fmaxf(c_run, top - 15.0f), fold_new = ex2(c_run - c_new);
        c_run = c_new;
        float sum = 0.0f;
        uint32_t h[NC / 2], l[NC / 2];
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(&tok_vs[slot][col0 + i]);
          const float vv[4] = {v.x, v.y, v.z, v.w};
          float wt[4];
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const float p = ex2(fmaf(x[i + c], rs, -c_new));
            sum += p;
            wt[c] = p * vv[c];
          }
          split_f16(wt[0], wt[1], h[i / 2], l[i / 2]);
          split_f16(wt[2], wt[3], h[i / 2 + 1], l[i / 2 + 1]);
        }
        l_run = fmaf(l_run, fold_new, sum * L_UNIT);
        // the sixteen tokens' weights, zero where another copy has them: 8 + 8 columns over their scores
        uint32_t ph[8], pl[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const bool mine = CS == 1 || i / (NC / 2) == copy;
          ph[i] = mine ? h[i % (NC / 2)] : 0u;
          pl[i] = mine ? l[i % (NC / 2)] : 0u;
        }
        tm_st(s_tm + cg * 16, ph);
        tm_st(s_tm + cg * 16 + 8, pl);
        tm_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sh_base + S::WEIGHTS + 8 * buf);
        // the tile before: its O is ready or nearly so
        if (j > j0) {
          alive = take_outputs(it - 1);
          if (!alive) break;
        }
        fold = fold_new;
      }
      if (alive) alive = take_outputs(it - 1);
      if (!alive) break;
      fence_before();

      // ---- the rows of the piece: quarters and copies joined, then to the result or to the block's slot.  All products of the
      // piece are done, so Q's tiles are free.
      float* res = reinterpret_cast<float*>(sm + C::QHI);        // [128][D], 16-byte pieces XOR lane % 8
      sum_x[cg][row] = l_run;
      if (cg == 0) c_x[row] = c_run;
      alive = meet(S::SOFT, soft_phase);
      if (!alive) break;
      {
        float c_max = c_x[rq];
#pragma unroll
        for (int k = 1; k < CS; k++) c_max = fmaxf(c_max, c_x[k * ROWS + rq]);
        const float f = ex2(c_run - c_max);
#pragma unroll
        for (int i = 0; i < QD / 4; i++) {
          float v[4];
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int k = q * (QD / 4) + i, k2 = D == 64 ? k ^ 4 : k;   // see v_row
            v[q] = ((D == 64 && (cg & 1)) ? o[k2] : o[k]) * f;
          }
          const int piece = cg * (QD / 4) + i;
          *reinterpret_cast<float4*>(res + row * D + ((piece ^ (row & 7)) << 2)) = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
      alive = meet(S::SOFT, soft_phase);
      if (!alive) break;
      const bool whole = w.tile0 == 0 && w.tile1 == w.tiles;
      if (w.tile0 == 0 && !whole && tid == 0) a.items[blockIdx.x] = make_int4(w.e, w.head, kv_run_of(run.all, w.at + w.tiles - 1), 1);
      float* slot = a.slots + (int64_t)(2 * blockIdx.x + (w.tile0 == 0 ? 1 : 0)) * KV_SLOT_FLOATS;
      for (int x = tid; x - lane < w.rows_here * (D / 4); x += 32 * SOFT_WARPS) {   // whole warps: a row's D / 4 pieces are neighbouring lanes
        const int r = x / (D / 4), p = x % (D / 4);
        const bool used = r < w.rows_here;
        float c_max = c_x[r], sum = 0.0f, m = 0.0f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 1; k < CS; k++) c_max = fmaxf(c_max, c_x[k * ROWS + r]);
#pragma unroll
        for (int k = 0; k < CS; k++) {
          const int ln = k * ROWS + r;
          const float4 y = *reinterpret_cast<const float4*>(res + ln * D + ((p ^ (ln & 7)) << 2));
          sum = fmaf((sum_x[0][ln] + sum_x[1][ln]) + (sum_x[2][ln] + sum_x[3][ln]), ex2(c_x[ln] - c_max), sum);
          v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
        }
        const bool far = used && (c_max > FAR || (c_max <= -FAR && sum == sum));   // (sum NaN: the query has one, the row stays NaN)
        if (__any_sync(0xffffffffu, far)) {
          const FarRow<D> y = far_row<D, ROWS>(a, w.b, w.head, w.rb, used ? r : 0, w.tile0, w.tile1, p, far);
          if (far) { v = y.v; sum = y.sum; c_max = y.c; m = y.m; }
        }
        if (!used) continue;
        if (whole) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          int t;
          *reinterpret_cast<float4*>(a.out + row_offset(a, w.b, w.head, w.rb * ROWS + r, a.ld_o, D, t) + p * 4) = make_float4(v.x * L_UNIT * inv, v.y * L_UNIT * inv, v.z * L_UNIT * inv, v.w * L_UNIT * inv);
        } else {
          __stcg(reinterpret_cast<float4*>(slot + r * D) + p, v);
          if (p == 0) __stcg(reinterpret_cast<float4*>(slot + ROWS * D) + r, make_float4(c_max, sum, m, 0.0f));
        }
      }
      alive = meet(S::SOFT, soft_phase);                         // Q's tiles are about to be written again
      w.close(a);
    }
  } else if (warp < SOFT_WARPS + STAGE_WARPS) {
    // ------------------------------------------------------------------------------------------------ staging
    // Unit u of a piece is sixteen tokens of tile tile0 + u / 4: one page, so one run of codes and of scales.  Units go round the
    // warps; a unit's codes are on their way into registers while the warp waits for a free slot.
    const int sw = warp - SOFT_WARPS;
    constexpr int KN = D / 32, VN = D / 64;                      // K: 16-byte pieces of a lane; V: (eight tokens x one word) of a lane
    const int v_L = D == 128 ? lane : lane & 15, v_oct = D == 128 ? 0 : lane >> 4;
    uint32_t k_off[KN], v_off[4];                                // places in the tiles, but for the sixteen tokens' own
#pragma unroll
    for (int i = 0; i < KN; i++) {
      const int c = i * 32 + lane, tok = c / (D / 16), p = c % (D / 16);
      k_off[i] = (p >> 2) * C::K_BLOCK + sw128(tok, (p & 3) * 32);   // sixteen tokens on: 2048 bytes on, the same swizzle
    }
#pragma unroll
    for (int q = 0; q < 4; q++) v_off[q] = v_row<D>(v_L, q) * 128;
    uint32_t next = sw;                                          // the next unit of the run for this warp
    while (alive && w.open(a, mp.row_blocks)) {
      const int32_t* table = a.page_table + (int64_t)w.b * a.g.max_pages;
      const int64_t in_table = min(w.vis, a.g.max_pages << a.g.page_shift);
      const uint32_t first_unit = it * 4, end_unit = (it + (uint32_t)(w.tile1 - w.tile0)) * 4;
      const int64_t pos0 = (int64_t)w.tile0 * MT - (int64_t)first_unit * 16;
      auto page_of = [&](uint32_t u) -> int {                    // -1: nothing of the unit is visible
        const int64_t pos = pos0 + (int64_t)u * 16;
        return (u < end_unit && pos < in_table) ? __ldcg(table + (pos >> a.g.page_shift)) : -1;
      };
      uint4 rk[KN];
      uint32_t rv[VN * 8];
      float ks, vs;
      auto fetch = [&](uint32_t u, int page) {
        const int64_t pos = pos0 + (int64_t)u * 16;
        const bool ok = (uint32_t)page < (uint32_t)a.g.pages;
        const int64_t cell = ok ? (((int64_t)page * a.g.heads + w.head) << a.g.page_shift) + (pos & ((1 << a.g.page_shift) - 1)) : 0;
        const int8_t *kp = a.k + cell * D, *vp = a.v + cell * D;
#pragma unroll
        for (int i = 0; i < KN; i++) rk[i] = ok ? __ldcg(reinterpret_cast<const uint4*>(kp) + i * 32 + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int o = 0; o < VN; o++)
#pragma unroll
          for (int i = 0; i < 8; i++) rv[o * 8 + i] = ok ? __ldcg(reinterpret_cast<const uint32_t*>(vp + ((v_oct + o) * 8 + i) * D) + v_L) : 0u;
        ks = vs = 0.0f;
        if (ok && lane < 16 && pos + lane < w.vis) { ks = __ldcg(a.ks + cell + lane); vs = __ldcg(a.vs + cell + lane); }
      };
      int page = page_of(next), page_next = page_of(next + STAGE_WARPS);
      fetch(next, page);
#pragma unroll 1
      for (; next < end_unit; next += STAGE_WARPS) {
        const uint32_t t = next >> 2, slot = t % ST, part = next & 3;
        alive = __all_sync(0xffffffffu, wait(S::EMPTY + 8 * slot, ((t / ST) & 1) ^ 1u));
        if (!alive) break;
        const uint32_t kt = sm_base + C::RING + slot * C::STAGE + part * 2048, vt = sm_base + C::RING + slot * C::STAGE + C::K_BYTES;
#pragma unroll
        for (int i = 0; i < KN; i++) {                           // of four neighbouring dimensions the even ones come first
          const uint32_t to = kt + k_off[i];
          sts128(to, codes_even(rk[i].x), codes_odd(rk[i].x), codes_even(rk[i].y), codes_odd(rk[i].y));
          sts128(to ^ 16u, codes_even(rk[i].z), codes_odd(rk[i].z), codes_even(rk[i].w), codes_odd(rk[i].w));
        }
#pragma unroll
        for (int o = 0; o < VN; o++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = __byte_perm(rv[o * 8 + 2 * i], rv[o * 8 + 2 * i + 1], h ? 0x7632 : 0x5410);
            const uint32_t col = part * 2 + v_oct + o;           // which eight tokens
            const uint32_t e = vt + v_off[2 * h], d = vt + v_off[2 * h + 1];
            sts128(e + ((col ^ ((v_off[2 * h] >> 7) & 7)) << 4), codes_even(y[0]), codes_even(y[1]), codes_even(y[2]), codes_even(y[3]));
            sts128(d + ((col ^ ((v_off[2 * h + 1] >> 7) & 7)) << 4), codes_odd(y[0]), codes_odd(y[1]), codes_odd(y[2]), codes_odd(y[3]));
          }
        const bool ok = (uint32_t)page < (uint32_t)a.g.pages;
        const int64_t pos = pos0 + (int64_t)next * 16;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok && lane < 16 && pos + lane < w.vis);
        if (lane < 16) {
          tok_ks[slot][part * 16 + lane] = ks;
          tok_vs[slot][part * 16 + lane] = vs;
          tok_lv[slot][part * 16 + lane] = log2_scale(vs);
        }
        if (lane == 0) {
          tok_there[slot][part] = mask;
          if (!ok && pos < w.vis) atomicOr(a.status, STATUS_BAD_INDEX);
        }
        fence_proxy();                                           // the tensor cores read what the threads wrote
        __syncwarp();
        if (lane == 0) mbar_arrive(sh_base + S::FULL + 8 * slot);
        page = page_next;
        page_next = page_of(next + 2 * STAGE_WARPS);
        if (next + STAGE_WARPS < end_unit) fetch(next + STAGE_WARPS, page);
      }
      it += (uint32_t)(w.tile1 - w.tile0);
      if (alive) w.close(a);
    }
  } else {
    // ------------------------------------------------------------------------------------------------ products
    // The whole warp walks and waits; one lane issues.
    uint32_t q_phase = 0;
    const uint64_t qh_desc = smem_desc(sm_base + C::QHI), ql_desc = smem_desc(sm_base + C::QLO), k_desc = smem_desc(sm_base + C::RING),
                   v_desc = smem_desc(sm_base + C::RING + C::K_BYTES);
    auto score = [&](uint32_t t) -> bool {                       // S of tile t
      const uint32_t slot = t % ST;
      bool ok = wait(S::FULL + 8 * slot, (t / ST) & 1);
      if (t >= 2) ok = ok && wait(S::OUTPUTS + 8 * (t & 1), ((t - 2) >> 1) & 1);   // P V of tile t - 2 has read the weights that stand there
      if (!__all_sync(0xffffffffu, ok)) return false;
      fence_after();
      constexpr uint32_t idesc = idesc_f16(LANES, MT);
      const uint32_t s_tm = tmem + TM_S + (t & 1) * TM_S_STEP;
      const uint64_t kd = k_desc + (uint64_t)(slot * (C::STAGE >> 4));
      if (lane == 0) {
#pragma unroll
        for (int s = 0; s < D / 16; s++) {                       // 16 dimensions = 32 bytes along K per instruction
          mma_ss(s_tm, ql_desc + (s >> 2) * (C::Q_BLOCK >> 4) + 2 * (s & 3), kd + (s >> 2) * (C::K_BLOCK >> 4) + 2 * (s & 3), idesc, s != 0);
        }
#pragma unroll
        for (int s = 0; s < D / 16; s++)
          mma_ss(s_tm, qh_desc + (s >> 2) * (C::Q_BLOCK >> 4) + 2 * (s & 3), kd + (s >> 2) * (C::K_BLOCK >> 4) + 2 * (s & 3), idesc, 1);
        mma_commit(sh_base + S::SCORES + 8 * (t & 1));
      }
      __syncwarp();
      return true;
    };
    while (alive && w.open(a, mp.row_blocks)) {
      alive = __all_sync(0xffffffffu, wait(S::QUERIES, q_phase));
      q_phase ^= 1u;
      if (alive) { fence_after(); alive = score(it); }
      for (int j = w.tile0; alive && j < w.tile1; j++, it++) {
        if (j + 1 < w.tile1 && !score(it + 1)) { alive = false; break; }
        if (!__all_sync(0xffffffffu, wait(S::WEIGHTS + 8 * (it & 1), (it >> 1) & 1))) { alive = false; break; }
        fence_after();
        constexpr uint32_t idesc = idesc_f16(LANES, D);
        const uint32_t p_tm = tmem + TM_S + (it & 1) * TM_S_STEP, o_tm = tmem + TM_O + (it & 1) * TM_O_STEP;
        const uint64_t vd = v_desc + (uint64_t)((it % ST) * (C::STAGE >> 4));
        if (lane == 0) {
#pragma unroll
          for (int s = 0; s < 4; s++) mma_ts(o_tm, p_tm + s * 16 + 8, vd + 2 * s, idesc, s != 0);   // 16 tokens each; the small halves first
#pragma unroll
          for (int s = 0; s < 4; s++) mma_ts(o_tm, p_tm + s * 16, vd + 2 * s, idesc, 1);
          mma_commit(sh_base + S::OUTPUTS + 8 * (it & 1));
          mma_commit(sh_base + S::EMPTY + 8 * (it % ST));
        }
        __syncwarp();
      }
      if (alive) w.close(a);
    }
  }

  __syncwarp();
  __syncthreads();
  if (sh.abort) {
    if (tid == 0) atomicOr(a.status, STATUS_SDPA_WAIT_TIMEOUT);
    const uint64_t t0 = gtimer();
    while (gtimer() - t0 < 2000000ull) __nanosleep(1000);        // products in flight finish before tensor memory is released
    __syncthreads();
  }
  fence_before();
  if (warp == SOFT_WARPS + STAGE_WARPS) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TM_COLS) : "memory");
  }
}

// Items that several runs worked on, joined in the order of the runs: block (run an item begins in, 16 of its rows).
template <int D, int ROWS>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const AttnArgs a, int row_blocks) {
  constexpr int P = D / 4;
  kv_after_previous();
  const int run0 = blockIdx.x;
  const int4 item = __ldcg(a.items + run0);
  if (item.w == 0) return;
  const int b = item.x / row_blocks, rb = item.x - b * row_blocks;
  const int rows_here = min(ROWS, kv_rows_in_use(a.count, b, a.T) * a.group - rb * ROWS);
  const int r0 = blockIdx.y * 16, r1 = min(rows_here, r0 + 16);
  for (int x = threadIdx.x; x < (r1 - r0) * P; x += 256) {
    const int r = r0 + x / P, p = x % P;
    // pieces in units of 2^(m + c), against the largest m of one that has seen something and the largest c relative to it
    auto piece = [&](int c) { return reinterpret_cast<const float4*>(a.slots + (int64_t)(2 * c + (c == run0)) * KV_SLOT_FLOATS); };
    auto row = [&](int c) { return __ldcg(piece(c) + ROWS * P + r); };   // c, sum, m
    float far = C_NONE, top = C_NONE, sum = 0.0f;
    bool some = false;
    for (int c = run0; c <= item.z; c++) {
      const float4 x = row(c);
      top = fmaxf(top, x.x);
      far = fmaxf(far, x.x > -FAR ? x.z : C_NONE);
      some |= x.z != 0.0f;
    }
    auto beside = [&](const float4& x) { return x.x > -FAR ? x.x + (x.z - far) : C_NONE; };
    if (some) {
      top = C_NONE;
      for (int c = run0; c <= item.z; c++) top = fmaxf(top, beside(row(c)));
    }
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = run0; c <= item.z; c++) {
      const float4 x = row(c), y = __ldcg(piece(c) + r * P + p);
      const float f = ex2((some ? beside(x) : x.x) - top);
      sum = fmaf(x.y, f, sum);
      v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y); v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    int t;
    *reinterpret_cast<float4*>(a.out + row_offset(a, b, item.y, rb * ROWS + r, a.ld_o, D, t) + p * 4) = make_float4(v.x * L_UNIT * inv, v.y * L_UNIT * inv, v.z * L_UNIT * inv, v.w * L_UNIT * inv);
  }
}

template <int D, int CS>
int launch_many(b200q_ctx* ctx, const AttnArgs& a) {
  constexpr int ROWS = LANES / CS;
  constexpr uint32_t ready = 1u << ((D == 64 ? 2 : 4) + CS - 1);
  if (!(ctx->kv_ready & ready)) {
    B200Q_CHECK_CUDA(cudaFuncSetAttribute(kv_attention_many_kernel<D, CS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<D>::SMEM));
    ctx->kv_ready |= ready;
  }
  ManyParams mp;
  mp.row_blocks = (int)(((int64_t)a.T * a.group + ROWS - 1) / ROWS);
  mp.polls = (uint32_t)(ctx->wait_limit_s * 1e6) + 1000;
  const unsigned grid = (unsigned)ctx->sm_count;
  if (int e = kv_launch(ctx, kv_attention_many_kernel<D, CS>, dim3(grid), MANY_THREADS, Many<D>::SMEM, a, mp)) return e;
  return kv_launch(ctx, kv_attention_join_kernel<D, ROWS>, dim3(grid, (ROWS + 15) / 16), 256, 0, a, mp.row_blocks);
}

}  // namespace

int launch_kv_attention_many(b200q_ctx* ctx, const AttnArgs& a, int D) {
  const int64_t rows = (int64_t)a.T * a.group;
  if (D == 64) return rows <= 64 ? launch_many<64, 2>(ctx, a) : launch_many<64, 1>(ctx, a);
  return rows <= 64 ? launch_many<128, 2>(ctx, a) : launch_many<128, 1>(ctx, a);
}

}  // namespace b200q

// Attention over the int8 key/value cache for many query rows (chunks of a prompt, drafted trees) on the 5th-generation
// tensor cores.  What is computed and in which arithmetic stands in kv_attention.cuh.
#include "kv_attention.cuh"
#include "quant_math.cuh"

namespace b200q {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// One block per SM walks a run of 64-token tiles; an item is up to 128 rows, the 128 lanes of tensor memory.  Roles:
//   four staging warps: K and V of a tile from the cache into a ring in shared memory as binary16 tiles of the tensor cores'
//     layout (V transposed), with the tokens' scales beside them; a warp handles sixteen tokens, which always share a page;
//   one thread issues the products: S_hi = Q_hi K^T and S_lo = Q_lo K^T (tcgen05.mma kind::f16, 128 x 64) of tile j + 1, then
//     O = P_lo V + P_hi V of tile j with the weights read from tensor memory;
//   sixteen softmax warps, four threads per row with sixteen tokens of a tile each: scores from tensor memory, the row's c
//     agreed on through shared memory, the weights' two halves written over the scores, and tile j - 1's O folded into a
//     quarter of the row's outputs per thread in registers: o = o * 2^(c_old - c_new) + O.  Sums over tiles are binary32
//     additions, not the tensor core's.
// Scores and O are double-buffered (512 columns of tensor memory), so products, softmax and staging of neighbouring tiles
// overlap.  Bound by the instruction issue of the softmax and staging warps, with the products (1024 cycles per tile of
// 128 rows at head dimension 128) close behind.
//
// With 64 or fewer rows (CS = 2) or 32 or fewer (CS = 4) the lanes hold CS copies of the rows, each copy takes 16 / CS of a
// thread's tokens and has weights of zero elsewhere, and the copies are joined at the end: the softmax work, which
// would leave lanes idle, shrinks with the rows.
//
// Every wait is bounded: one that runs out raises the block's abort flag and STATUS_SDPA_WAIT_TIMEOUT, all roles leave,
// products in flight get 2 ms, tensor memory is freed.  Threads meet at mbarriers only, never at a hardware barrier that
// a role that has left would keep the others waiting at; the one at the end is reached by all.
// ---------------------------------------------------------------------------------------------------------------
constexpr int MT = 64, LANES = 128, SOFT_WARPS = 16, STAGE_WARPS = 4, MANY_THREADS = 32 * (SOFT_WARPS + STAGE_WARPS + 1);
template <int D>
struct Many {
  static constexpr int Q_BLOCK = LANES * 128, Q_BYTES = (D / 64) * Q_BLOCK;    // K blocks of 64 dimensions: [128 rows][128 B]
  static constexpr int K_BLOCK = MT * 128, K_BYTES = (D / 64) * K_BLOCK, V_BYTES = D * 128;
  static constexpr int STAGES = 4, STAGE = K_BYTES + V_BYTES;
  static constexpr int QHI = 0, QLO = Q_BYTES, RING = 2 * Q_BYTES, END = RING + STAGES * STAGE;
  static constexpr int SMEM = END + 1024;
};
// columns: scores (hi, lo) of even and odd tiles, the weights over them; O of even and odd tiles
constexpr int TM_S = 0, TM_SLO = 64, TM_S_STEP = 128, TM_O = 256, TM_O_STEP = 128, TM_COLS = 512;

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

// N consecutive columns of this warp's lanes; the values may be used after tm_wait_ld on the same registers.
__device__ __forceinline__ void tm_ld(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_ld(uint32_t at, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at) : "memory");
}
template <int N>
__device__ __forceinline__ void tm_wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i])::"memory");   // no use of a loaded register moves ahead of the wait
}
__device__ __forceinline__ void tm_st(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ void tm_ld(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

struct ManyParams {
  int row_blocks;
  unsigned long long limit_ns;
};

// The block's barriers and flags.  Counts: one arrival per warp (after __syncwarp) or per tcgen05.commit.
template <int STAGES>
struct ManyShared {
  uint64_t full[STAGES], empty[STAGES];        // ring slots: staged (4 warps), consumed (commit of the tile's P V)
  uint64_t scores[2], weights[2], outputs[2];  // S ready (commit), P ready (16 warps), O ready (commit)
  uint64_t queries, soft;                      // Q staged (16 warps); meeting of the softmax warps (16 warps)
  uint64_t rows[4];                            // meeting of the four warps that share a quarter of the lanes
  uint32_t tmem;
  int abort;
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

template <int D, int CS>
__global__ void __launch_bounds__(MANY_THREADS, 1) kv_attention_many_kernel(const AttnArgs a, const ManyParams mp) {
  using C = Many<D>;
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
  const Run run = find_run<ROWS, MT, 2>(a, mp.row_blocks);
  if (tid == 0) a.items[blockIdx.x] = make_int4(0, 0, 0, 0);
  if (run.begin == run.end) return;

  if (tid == 0) {
    for (int s = 0; s < ST; s++) { mbar_init(smem_u32(&sh.full[s]), STAGE_WARPS); mbar_init(smem_u32(&sh.empty[s]), 1); }
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

  auto wait = [&](const uint64_t& bar, uint32_t parity) -> bool {
    const uint32_t addr = smem_u32(&bar);
    uint32_t done = 0, it = 0;
    uint64_t t0 = 0;
    while (true) {
      asm volatile(
          "{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(done) : "r"(addr), "r"(parity), "r"(1000u) : "memory");
      if (done) return true;
      if ((++it & 7u) == 0u) {
        if (*abort_flag) return false;
        if (t0 == 0) t0 = gtimer();
        else if (gtimer() - t0 > mp.limit_ns) { *abort_flag = 1; return false; }
      }
    }
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
    auto meet = [&](const uint64_t& bar, uint32_t& phase) -> bool {   // all warps of the barrier; shared memory before it is seen after it
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar));
      const bool ok = wait(bar, phase);
      phase ^= 1u;
      return __all_sync(0xffffffffu, ok);
    };
    while (alive && w.open(a, mp.row_blocks)) {
      if (tid == 0 && (w.first < 0 || w.first + w.n > (a.g.max_pages << a.g.page_shift))) atomicOr(a.status, STATUS_BAD_INDEX);
      // ---- the query row: this thread's quarter of it, in fixed point
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
          x[i] = used ? __ldg(reinterpret_cast<const float4*>(src) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
          top = max(max(top, max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu)),
                    max(__float_as_uint(x[i].z) & 0x7fffffffu, __float_as_uint(x[i].w) & 0x7fffffffu));
        }
        sum_x[cg][row] = __uint_as_float(top);
        alive = meet(sh.rows[quarter], rows_phase);
        if (!alive) break;
#pragma unroll
        for (int k = 0; k < 4; k++) top = max(top, __float_as_uint(sum_x[k][row]));
        const bool finite = top < 0x7f800000u;
        const int ex = max((int)(top >> 23), 24) - 127;
        const float up = pow2(10 - ex);
        rs = finite ? a.scale_log2e * pow2(ex - 10) : __int_as_float(0x7fc00000);
#pragma unroll
        for (int i = 0; i < QD / 4; i += 2) {                    // eight dimensions: 16 bytes of either half, in the order of staged K
          float h[8], l[8];
          const float y[8] = {x[i].x, x[i].y, x[i].z, x[i].w, x[i + 1].x, x[i + 1].y, x[i + 1].z, x[i + 1].w};
#pragma unroll
          for (int c = 0; c < 8; c++) split_whole(finite ? y[c] * up : 0.0f, h[c], l[c]);
          const int dim = cg * QD + i * 4;
          const uint32_t to = sm_base + (dim >> 6) * C::Q_BLOCK + sw128(row, (dim & 63) * 2);
          sts128(to + C::QHI, pack_f16(h[0], h[2]), pack_f16(h[1], h[3]), pack_f16(h[4], h[6]), pack_f16(h[5], h[7]));
          sts128(to + C::QLO, pack_f16(l[0], l[2]), pack_f16(l[1], l[3]), pack_f16(l[4], l[6]), pack_f16(l[5], l[7]));
        }
        fence_proxy();                                           // the tensor cores read what the threads wrote
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.queries));
      }

      uint64_t o2[QD / 2];                                       // pairs of outputs, in the order of the V tile's rows
#pragma unroll
      for (int i = 0; i < QD / 2; i++) o2[i] = 0;
      float c_run = C_NONE, l_run = 0.0f, fold = 0.0f;           // fold: the factor that goes with the latest tile's O
      auto take_outputs = [&](uint32_t t) -> bool {              // o = o * fold + O of tile t
        if (!__all_sync(0xffffffffu, wait(sh.outputs[t & 1], (t >> 1) & 1))) return false;
        fence_after();
        const uint64_t fold2 = f2_dup(fold);
#pragma unroll
        for (int c = 0; c < QD; c += 16) {
          uint32_t x[16];
          tm_ld(lane_tm + TM_O + (t & 1) * TM_O_STEP + cg * QD + c, x);
          tm_wait_ld(x);
#pragma unroll
          for (int i = 0; i < 16; i += 2)
            o2[(c + i) / 2] = f2_fma(o2[(c + i) / 2], fold2, f2_pack(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
        }
        return true;
      };

      for (int j = w.tile0; j < w.tile1; j++, it++) {
        const uint32_t buf = it & 1, slot = it % ST;
        const uint32_t s_tm = lane_tm + TM_S + buf * TM_S_STEP;
        // the slot's tokens (the staging warps' stores) and the scores
        bool ok = wait(sh.full[slot], (it / ST) & 1) && wait(sh.scores[buf], (it >> 1) & 1);
        alive = __all_sync(0xffffffffu, ok);
        if (!alive) break;
        fence_after();
        uint32_t hi[NC], lo[NC];
        tm_ld(s_tm + col0, hi);
        tm_ld(s_tm + TM_SLO + col0, lo);

        // which of this thread's tokens its row sees
        uint32_t seen = tok_there[slot][cg];
        const int64_t from = (int64_t)j * MT + cg * 16 - w.first;   // place of the first of the sixteen tokens among the new rows
        if (from + 16 > 0) {
          const uint32_t before = from >= 0 ? 0u : (1u << (int)-from) - 1;
          uint32_t fresh;
          if (a.tree) fresh = from >= 64 ? 0u : (from >= 0 ? (uint32_t)(row_seen >> (int)from) : (uint32_t)(row_seen << (int)-from));
          else {
            const int64_t k = (int64_t)row_t + 1 - from;         // tokens up to the row itself
            fresh = k <= 0 ? 0u : (k >= 16 ? 0xffffu : (1u << (int)k) - 1);
          }
          seen &= before | fresh;
        }
        seen >>= copy * NC;
        const bool all = (seen & ((1u << NC) - 1)) == (1u << NC) - 1;

        // z = (S_hi + S_lo) * scale_k * rs
        float z[NC], top = NEG_INF;
        const uint64_t rs2 = f2_dup(rs);
        tm_wait_ld(hi);
        tm_wait_ld(lo);
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
          const float4 k = *reinterpret_cast<const float4*>(&tok_ks[slot][col0 + i]);
          const uint64_t s0 = f2_add(f2_pack(__uint_as_float(hi[i]), __uint_as_float(hi[i + 1])), f2_pack(__uint_as_float(lo[i]), __uint_as_float(lo[i + 1])));
          const uint64_t s1 = f2_add(f2_pack(__uint_as_float(hi[i + 2]), __uint_as_float(hi[i + 3])), f2_pack(__uint_as_float(lo[i + 2]), __uint_as_float(lo[i + 3])));
          f2_unpack(f2_mul(f2_mul(s0, f2_pack(k.x, k.y)), rs2), z[i], z[i + 1]);
          f2_unpack(f2_mul(f2_mul(s1, f2_pack(k.z, k.w)), rs2), z[i + 2], z[i + 3]);
        }
        if (!all) {
#pragma unroll
          for (int i = 0; i < NC; i++)
            if (!((seen >> i) & 1)) z[i] = NEG_INF;
        }
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(&tok_lv[slot][col0 + i]);
          top = fmaxf(fmaxf(top, fmaxf(z[i] + v.x, z[i + 1] + v.y)), fmaxf(z[i + 2] + v.z, z[i + 3] + v.w));
        }
        // the row's other tokens: warps with the same lanes (slots alternate, so one meeting per tile does)
        top_x[buf][cg][row] = top;
        alive = meet(sh.rows[quarter], rows_phase);
        if (!alive) break;
#pragma unroll
        for (int k = 0; k < 4; k++) top = fmaxf(top, top_x[buf][k][row]);
        const float c_new = fmaxf(c_run, top - 10.0f), fold_new = ex2(c_run - c_new);
        c_run = c_new;
        uint64_t l2 = 0;
        const uint64_t c2 = f2_dup(c_new), magic2 = f2_dup(12582912.0f);
        uint32_t h[NC / 2], l[NC / 2];
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(&tok_vs[slot][col0 + i]);
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            float d0, d1, x0, x1, y0, y1;
            f2_unpack(f2_sub(f2_pack(z[i + k], z[i + k + 1]), c2), d0, d1);
            const uint64_t p = f2_pack(ex2(d0), ex2(d1));
            l2 = f2_add(l2, p);
            const uint64_t x = f2_mul(p, k == 0 ? f2_pack(v.x, v.y) : f2_pack(v.z, v.w));
            const uint64_t xh = f2_sub(f2_add(x, magic2), magic2);
            f2_unpack(xh, x0, x1);
            f2_unpack(f2_sub(x, xh), y0, y1);
            h[(i + k) / 2] = pack_f16(x0, x1);
            l[(i + k) / 2] = pack_f16(y0, y1);
          }
        }
        {
          float p0, p1;
          f2_unpack(l2, p0, p1);
          l_run = fmaf(l_run, fold_new, (p0 + p1) * P_UNIT);
        }
        // the sixteen tokens' weights, zero where another copy has them: 8 + 8 columns over their S_hi
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
        if (lane == 0) mbar_arrive(smem_u32(&sh.weights[buf]));
        // the tile before: its O is ready or nearly so
        if (j > w.tile0) {
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
      alive = meet(sh.soft, soft_phase);
      if (!alive) break;
      {
        float c_max = c_x[rq];
#pragma unroll
        for (int k = 1; k < CS; k++) c_max = fmaxf(c_max, c_x[k * ROWS + rq]);
        const uint64_t f2 = f2_dup(ex2(c_run - c_max));
#pragma unroll
        for (int i = 0; i < QD / 4; i++) {
          float v[4];
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int k = q * (QD / 4) + i, k2 = D == 64 ? k ^ 4 : k;   // see v_row
            float x0, x1, y0, y1;
            f2_unpack(f2_mul(o2[k / 2], f2), x0, x1);
            f2_unpack(f2_mul(o2[k2 / 2], f2), y0, y1);
            v[q] = (D == 64 && (cg & 1)) ? ((k2 & 1) ? y1 : y0) : ((k & 1) ? x1 : x0);
          }
          const int piece = cg * (QD / 4) + i;
          *reinterpret_cast<float4*>(res + row * D + ((piece ^ (row & 7)) << 2)) = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
      alive = meet(sh.soft, soft_phase);
      if (!alive) break;
      const bool whole = w.tile0 == 0 && w.tile1 == w.tiles;
      if (w.tile0 == 0 && !whole && tid == 0) a.items[blockIdx.x] = make_int4(w.e, w.head, kv_run_of(run.all, w.at + w.tiles - 1), 1);
      float* slot = a.slots + (int64_t)(2 * blockIdx.x + (w.tile0 == 0 ? 1 : 0)) * KV_SLOT_FLOATS;
      for (int x = tid; x < w.rows_here * (D / 4); x += 32 * SOFT_WARPS) {
        const int r = x / (D / 4), p = x % (D / 4);
        float c_max = c_x[r], sum = 0.0f;
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
        if (whole) {
          const float inv = sum == 0.0f ? 0.0f : P_UNIT / sum;
          int t;
          *reinterpret_cast<float4*>(a.out + row_offset(a, w.b, w.head, w.rb * ROWS + r, a.ld_o, D, t) + p * 4) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        } else {
          __stcg(reinterpret_cast<float4*>(slot + r * D) + p, v);
          if (p == 0) { __stcg(slot + ROWS * D + r, c_max); __stcg(slot + ROWS * D + ROWS + r, sum); }
        }
      }
      alive = meet(sh.soft, soft_phase);                         // Q's tiles are about to be written again
      w.close(a);
    }
  } else if (warp < SOFT_WARPS + STAGE_WARPS) {
    // ------------------------------------------------------------------------------------------------ staging
    // Sixteen tokens of a tile per warp: one page, so one run of codes and of scales.  A tile's codes are on their way into
    // registers while the warp waits for a free slot, and the page of the tile after it is looked up.
    const int sw = warp - SOFT_WARPS;
    constexpr int KN = D / 32, VN = D / 64;                      // K: 16-byte pieces of a lane; V: (eight tokens x one word) of a lane
    const int v_L = D == 128 ? lane : lane & 15, v_oct = D == 128 ? 0 : lane >> 4;
    while (alive && w.open(a, mp.row_blocks)) {
      const int32_t* table = a.page_table + (int64_t)w.b * a.g.max_pages;
      const int64_t pages_tokens = a.g.max_pages << a.g.page_shift;
      auto page_of = [&](int j) -> int {
        const int64_t pos = (int64_t)j * MT + sw * 16;
        return (j < w.tile1 && pos < pages_tokens) ? __ldg(table + (pos >> a.g.page_shift)) : -1;
      };
      struct Raw { uint4 k[KN]; uint32_t v[VN * 8]; float ks, vs; };
      auto fetch = [&](int j, int page, Raw& r) {
        const int64_t pos = (int64_t)j * MT + sw * 16;
        const bool ok = (uint32_t)page < (uint32_t)a.g.pages && pos < w.vis;   // else nothing of the sixteen is visible
        const int64_t cell = ok ? (((int64_t)page * a.g.heads + w.head) << a.g.page_shift) + (pos & ((1 << a.g.page_shift) - 1)) : 0;
        const int8_t *kp = a.k + cell * D, *vp = a.v + cell * D;
#pragma unroll
        for (int i = 0; i < KN; i++) r.k[i] = ok ? __ldg(reinterpret_cast<const uint4*>(kp) + i * 32 + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < VN; u++)
#pragma unroll
          for (int i = 0; i < 8; i++) r.v[u * 8 + i] = ok ? __ldg(reinterpret_cast<const uint32_t*>(vp + ((v_oct + u) * 8 + i) * D) + v_L) : 0u;
        r.ks = r.vs = 0.0f;
        if (ok && lane < 16 && pos + lane < w.vis) { r.ks = __ldg(a.ks + cell + lane); r.vs = __ldg(a.vs + cell + lane); }
      };
      Raw cur;
      int page = page_of(w.tile0), page_next = page_of(w.tile0 + 1);
      fetch(w.tile0, page, cur);
      for (int j = w.tile0; j < w.tile1; j++, it++) {
        const uint32_t slot = it % ST;
        alive = __all_sync(0xffffffffu, wait(sh.empty[slot], ((it / ST) & 1) ^ 1u));
        if (!alive) break;
        const uint32_t kt = sm_base + C::RING + slot * C::STAGE, vt = kt + C::K_BYTES;
#pragma unroll
        for (int i = 0; i < KN; i++) {                           // of four neighbouring dimensions the even ones come first
          const int c = i * 32 + lane, tok = sw * 16 + c / (D / 16), p = c % (D / 16);
          const uint32_t to = kt + (p >> 2) * C::K_BLOCK;
          const uint4 x = cur.k[i];
          sts128(to + sw128(tok, (p & 3) * 32), codes_even(x.x), codes_odd(x.x), codes_even(x.y), codes_odd(x.y));
          sts128(to + sw128(tok, (p & 3) * 32 + 16), codes_even(x.z), codes_odd(x.z), codes_even(x.w), codes_odd(x.w));
        }
#pragma unroll
        for (int u = 0; u < VN; u++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = __byte_perm(cur.v[u * 8 + 2 * i], cur.v[u * 8 + 2 * i + 1], h ? 0x7632 : 0x5410);
            const int col = (sw * 2 + v_oct + u) * 16;           // eight tokens
            sts128(vt + sw128(v_row<D>(v_L, 2 * h), col), codes_even(y[0]), codes_even(y[1]), codes_even(y[2]), codes_even(y[3]));
            sts128(vt + sw128(v_row<D>(v_L, 2 * h + 1), col), codes_odd(y[0]), codes_odd(y[1]), codes_odd(y[2]), codes_odd(y[3]));
          }
        const int64_t pos = (int64_t)j * MT + sw * 16;
        const bool there = (uint32_t)page < (uint32_t)a.g.pages && lane < 16 && pos + lane < w.vis;
        const uint32_t mask = __ballot_sync(0xffffffffu, there);
        if (lane < 16) {
          tok_ks[slot][sw * 16 + lane] = cur.ks;
          tok_vs[slot][sw * 16 + lane] = cur.vs;
          tok_lv[slot][sw * 16 + lane] = log2_scale(cur.vs);
        }
        if (lane == 0) {
          tok_there[slot][sw] = mask;
          if ((uint32_t)page >= (uint32_t)a.g.pages && pos < w.vis) atomicOr(a.status, STATUS_BAD_INDEX);
        }
        fence_proxy();                                           // the tensor cores read what the threads wrote
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.full[slot]));
        page = page_next;
        page_next = page_of(j + 2);
        if (j + 1 < w.tile1) fetch(j + 1, page, cur);
      }
      if (alive) w.close(a);
    }
  } else if (lane == 0) {
    // ------------------------------------------------------------------------------------------------ products
    uint32_t q_phase = 0;
    auto score = [&](uint32_t t) -> bool {                       // S of tile t
      const uint32_t slot = t % ST;
      if (!wait(sh.full[slot], (t / ST) & 1)) return false;
      if (t >= 2 && !wait(sh.outputs[t & 1], ((t - 2) >> 1) & 1)) return false;   // P V of tile t - 2 has read the weights that stand there
      fence_after();
      constexpr uint32_t idesc = idesc_f16(LANES, MT);
      const uint32_t s_tm = tmem + TM_S + (t & 1) * TM_S_STEP, kt = sm_base + C::RING + slot * C::STAGE;
#pragma unroll
      for (int s = 0; s < D / 16; s++) {                         // 16 dimensions = 32 bytes along K per instruction
        const uint64_t kd = smem_desc(kt + (s >> 2) * C::K_BLOCK) + 2 * (s & 3);
        const uint32_t q = sm_base + (s >> 2) * C::Q_BLOCK;
        mma_ss(s_tm, smem_desc(q + C::QHI) + 2 * (s & 3), kd, idesc, s != 0);
        mma_ss(s_tm + TM_SLO, smem_desc(q + C::QLO) + 2 * (s & 3), kd, idesc, s != 0);
      }
      mma_commit(smem_u32(&sh.scores[t & 1]));
      return true;
    };
    while (alive && w.open(a, mp.row_blocks)) {
      alive = wait(sh.queries, q_phase);
      q_phase ^= 1u;
      if (alive) { fence_after(); alive = score(it); }
      for (int j = w.tile0; alive && j < w.tile1; j++, it++) {
        if (j + 1 < w.tile1 && !score(it + 1)) { alive = false; break; }
        if (!wait(sh.weights[it & 1], (it >> 1) & 1)) { alive = false; break; }
        fence_after();
        constexpr uint32_t idesc = idesc_f16(LANES, D);
        const uint32_t p_tm = tmem + TM_S + (it & 1) * TM_S_STEP, o_tm = tmem + TM_O + (it & 1) * TM_O_STEP;
        const uint32_t vt = sm_base + C::RING + (it % ST) * C::STAGE + C::K_BYTES;
#pragma unroll
        for (int s = 0; s < 4; s++) mma_ts(o_tm, p_tm + s * 16 + 8, smem_desc(vt) + 2 * s, idesc, s != 0);   // 16 tokens each; the small halves first
#pragma unroll
        for (int s = 0; s < 4; s++) mma_ts(o_tm, p_tm + s * 16, smem_desc(vt) + 2 * s, idesc, 1);
        mma_commit(smem_u32(&sh.outputs[it & 1]));
        mma_commit(smem_u32(&sh.empty[it % ST]));
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
    float c_max = C_NONE, sum = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = run0; c <= item.z; c++) c_max = fmaxf(c_max, __ldcg(a.slots + (int64_t)(2 * c + (c == run0)) * KV_SLOT_FLOATS + ROWS * D + r));
    for (int c = run0; c <= item.z; c++) {
      const float* s = a.slots + (int64_t)(2 * c + (c == run0)) * KV_SLOT_FLOATS;
      const float f = ex2(__ldcg(s + ROWS * D + r) - c_max);
      const float4 y = __ldcg(reinterpret_cast<const float4*>(s + r * D) + p);
      sum = fmaf(__ldcg(s + ROWS * D + ROWS + r), f, sum);
      v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y); v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
    }
    const float inv = sum == 0.0f ? 0.0f : P_UNIT / sum;
    int t;
    *reinterpret_cast<float4*>(a.out + row_offset(a, b, item.y, rb * ROWS + r, a.ld_o, D, t) + p * 4) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  }
}

template <int D, int CS>
int launch_many(b200q_ctx* ctx, const AttnArgs& a) {
  constexpr int ROWS = LANES / CS;
  constexpr uint32_t ready = 1u << ((D == 64 ? 4 : 8) + CS / 2);   // CS = 1, 2, 4: bits 0, 1, 2 of four
  if (!(ctx->kv_ready & ready)) {
    B200Q_CHECK_CUDA(cudaFuncSetAttribute(kv_attention_many_kernel<D, CS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<D>::SMEM));
    ctx->kv_ready |= ready;
  }
  ManyParams mp;
  mp.row_blocks = (int)(((int64_t)a.T * a.group + ROWS - 1) / ROWS);
  mp.limit_ns = (unsigned long long)(ctx->wait_limit_s * 1e9);
  const unsigned grid = (unsigned)ctx->sm_count;
  if (int e = kv_launch(ctx, kv_attention_many_kernel<D, CS>, dim3(grid), MANY_THREADS, Many<D>::SMEM, a, mp)) return e;
  return kv_launch(ctx, kv_attention_join_kernel<D, ROWS>, dim3(grid, (ROWS + 15) / 16), 256, 0, a, mp.row_blocks);
}

}  // namespace

int launch_kv_attention_many(b200q_ctx* ctx, const AttnArgs& a, int D) {
  const int64_t rows = (int64_t)a.T * a.group;
  if (D == 64) return rows <= 32 ? launch_many<64, 4>(ctx, a) : rows <= 64 ? launch_many<64, 2>(ctx, a) : launch_many<64, 1>(ctx, a);
  return rows <= 32 ? launch_many<128, 4>(ctx, a) : rows <= 64 ? launch_many<128, 2>(ctx, a) : launch_many<128, 1>(ctx, a);
}

}  // namespace b200q

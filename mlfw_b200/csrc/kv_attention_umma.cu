// Attention over the int8 key/value cache for many query rows (chunks of a prompt, drafted trees) on the 5th-generation
// tensor cores.  What is computed and in which arithmetic stands in kv_attention.cuh.
#include "kv_attention.cuh"
#include "quant_math.cuh"

namespace b200q {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// One block of 256 threads per run of 64-token tiles; an item is up to 128 rows, the 128 lanes of tensor memory.  Row r
// belongs to the threads r and r + 128, which take 32 tokens of a tile and half of the outputs each (warps w and w + 4 reach
// the same lanes).  Per tile:
//   S_hi = Q_hi K^T and S_lo = Q_lo K^T (tcgen05.mma kind::f16, 128 x 64, codes as binary16 in shared memory), meanwhile the
//   threads put V's codes, transposed, into shared memory;
//   every thread reads its scores twice from tensor memory -- for the row's running c, then for the weights; keeping 32
//   scores beside 64 outputs would not fit 128 registers -- and writes the weights' two halves over the scores it has read;
//   O = P_lo V + P_hi V (A operand in tensor memory), meanwhile the next tile's K goes to shared memory;
//   o = o * 2^(c_old - c_new) + O in registers: sums over tiles are binary32 additions, not the tensor core's.
// Two blocks share an SM (97 KB of shared memory and 256 columns of tensor memory each): the phases of one fill the gaps
// of the other.  Bound by the matrix products for 128 rows (1024 cycles per tile at head dimension 128 against about 900
// of the threads' work).
//
// With 64 or fewer rows (CS = 2) or 32 or fewer (CS = 4) the lanes hold CS copies of the rows, each copy takes every CS-th
// group of 32 / CS tokens of a half tile and has weights of zero elsewhere, and the copies are joined at the end: the
// softmax work, which would leave lanes idle, shrinks with the rows.
// ---------------------------------------------------------------------------------------------------------------
constexpr int MT = 64, LANES = 128, MANY_THREADS = 256;
template <int D>
struct Many {
  static constexpr int Q_BLOCK = LANES * 128, Q_BYTES = (D / 64) * Q_BLOCK;    // K blocks of 64 dimensions: [128 rows][128 B]
  static constexpr int K_BLOCK = MT * 128, K_BYTES = (D / 64) * K_BLOCK, V_BYTES = D * 128;
  static constexpr int QHI = 0, QLO = Q_BYTES, K = 2 * Q_BYTES, V = K + K_BYTES, END = V + V_BYTES;
  static constexpr int SMEM = END + 1024;
};
constexpr int TM_SHI = 0, TM_SLO = 64, TM_O = 128, TM_COLS = 256;

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
// Barrier of the two warps that share a quarter of the lanes (immediate numbers: a register operand would reserve all
// sixteen barriers of the SM for one block).
__device__ __forceinline__ void pair_barrier(int quarter) {
  switch (quarter) {
    case 0: asm volatile("bar.sync 1, 64;" ::: "memory"); break;
    case 1: asm volatile("bar.sync 2, 64;" ::: "memory"); break;
    case 2: asm volatile("bar.sync 3, 64;" ::: "memory"); break;
    default: asm volatile("bar.sync 4, 64;" ::: "memory"); break;
  }
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

struct ManyParams {
  int row_blocks;
  unsigned long long limit_ns;
};

template <int D, int CS>
__global__ void __launch_bounds__(MANY_THREADS, 2) kv_attention_many_kernel(const AttnArgs a, const ManyParams mp) {
  using C = Many<D>;
  constexpr int ROWS = LANES / CS, NC = 32 / CS, HD = D / 2;     // rows of an item; tokens of a tile and outputs of a thread
  constexpr int CW = NC < 16 ? NC : 16;                          // scores handled at a time
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar;
  __shared__ uint32_t tmem_slot;
  __shared__ float xchg[2][LANES];                               // [half][lane]
  __shared__ float copy_c[LANES];
  __shared__ int64_t row_at[2][MT];                              // rows of a tile's tokens in the cache, -1: not visible to anybody
  __shared__ __align__(16) float tok_ks[2][MT], tok_vs[2][MT], tok_lv[2][MT];
  __shared__ uint32_t tok_there[2][2];                           // which tokens have a row, by half
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sm_base = smem_u32(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int half = warp >> 2, row = tid & (LANES - 1);
  const int copy = CS == 1 ? 0 : row / ROWS, rq = row % ROWS;    // which copy of which row of the item
  const int col0 = half * 32 + copy * NC;                        // this thread's tokens of a tile: col0 .. col0 + NC - 1

  asm volatile("griddepcontrol.wait;" ::: "memory");             // the previous kernel of the stream wrote what is read here
  const Run run = find_run<ROWS, MT, 2>(a, mp.row_blocks);
  if (tid == 0 && blockIdx.x < gridDim.x) a.items[blockIdx.x] = make_int4(0, 0, 0, 0);
  if (run.begin == run.end) return;

  if (tid == 0) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&bar)), "r"(1) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((uint32_t)TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  __syncthreads();
  fence_after();
  // Only now may the next kernel's blocks come: one that allocates tensor memory before its own wait must not take what
  // a block of this grid still needs.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_slot, lane_tm = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  const uint32_t bar_addr = smem_u32(&bar);
  uint32_t phase = 0;
  bool alive = true;
  auto wait_mma = [&]() -> bool {
    bool ok = true;
    uint32_t done = 0, it = 0;
    const uint64_t t0 = gtimer();
    while (true) {
      asm volatile(
          "{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(done) : "r"(bar_addr), "r"(phase), "r"(1000u) : "memory");
      if (done) break;
      if ((++it & 7u) == 0u && gtimer() - t0 > mp.limit_ns) { ok = false; break; }
    }
    phase ^= 1u;
    return __syncthreads_and(ok ? 1 : 0) != 0;                   // all threads take the same way out
  };

  int64_t left = run.end - run.begin, at = run.begin;
  int e = run.e, head = run.head, tile0 = run.tile;
  while (left > 0 && alive) {
    const int b = e / mp.row_blocks, rb = e - b * mp.row_blocks;
    const int64_t first = a.start[b];
    const int n = kv_rows_in_use(a.count, b, a.T);
    const int tiles = kv_tiles(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr, MT);
    if (tiles == 0) { e++; head = 0; tile0 = 0; continue; }
    const int64_t vis = kv_visible(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr);
    const int tile1 = (int)min((int64_t)tiles, tile0 + left);
    const int rows_here = min(ROWS, n * a.group - rb * ROWS);
    if (tid == 0 && (first < 0 || first + n > (a.g.max_pages << a.g.page_shift))) atomicOr(a.status, STATUS_BAD_INDEX);

    // ---- tokens of a tile: threads 0 .. 63 find their rows two tiles ahead and their scales one tile ahead
    auto find_row = [&](int j) -> int64_t {
      const int64_t pos = (int64_t)j * MT + tid;
      if (j >= tile1 || pos >= vis) return -1;
      const int64_t r = kv_row(a.g, a.page_table, b, head, pos);
      if (r < 0) atomicOr(a.status, STATUS_BAD_INDEX);
      return r;
    };
    auto put_scales = [&](int j, int64_t r, float k, float v) {
      tok_ks[j & 1][tid] = k; tok_vs[j & 1][tid] = v; tok_lv[j & 1][tid] = log2_scale(v);
      const uint32_t there = __ballot_sync(0xffffffffu, r >= 0);
      if (lane == 0) tok_there[j & 1][warp] = there;
    };
    int64_t row_next = -1;                                       // this thread's token of the next tile
    if (tid < MT) {
      const int64_t r = find_row(tile0);
      row_next = find_row(tile0 + 1);
      row_at[tile0 & 1][tid] = r;
      row_at[(tile0 + 1) & 1][tid] = row_next;
      put_scales(tile0, r, r < 0 ? 0.0f : __ldg(a.ks + r), r < 0 ? 0.0f : __ldg(a.vs + r));
    }

    // ---- the query row: this thread's half of it, in fixed point
    float rs;
    int row_t;
    uint64_t row_seen;
    {
      const bool used = rq < rows_here;
      int t;
      const float* src = a.q + row_offset(a, b, head, rb * ROWS + (used ? rq : 0), a.ld_q, D, t) + half * HD;
      row_t = used ? t : -1;
      row_seen = used && a.tree ? a.tree[(int64_t)b * a.T + t] : 0;
      if (n < 64) row_seen &= (1ull << n) - 1;
      float4 x[HD / 4];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < HD / 4; i++) {
        x[i] = used ? __ldg(reinterpret_cast<const float4*>(src) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max(max(top, max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu)),
                  max(__float_as_uint(x[i].z) & 0x7fffffffu, __float_as_uint(x[i].w) & 0x7fffffffu));
      }
      xchg[half][row] = __uint_as_float(top);
      pair_barrier(warp & 3);
      top = max(top, __float_as_uint(xchg[half ^ 1][row]));
      const bool finite = top < 0x7f800000u;
      const int ex = max((int)(top >> 23), 24) - 127;
      const float up = pow2(10 - ex);
      rs = finite ? a.scale_log2e * pow2(ex - 10) : __int_as_float(0x7fc00000);
#pragma unroll
      for (int i = 0; i < HD / 4; i += 2) {                      // eight dimensions: 16 bytes of either half, in the order of staged K
        float h[8], l[8];
        const float y[8] = {x[i].x, x[i].y, x[i].z, x[i].w, x[i + 1].x, x[i + 1].y, x[i + 1].z, x[i + 1].w};
#pragma unroll
        for (int c = 0; c < 8; c++) split_whole(finite ? y[c] * up : 0.0f, h[c], l[c]);
        const int dim = half * HD + i * 4;
        const uint32_t to = sm_base + (dim >> 6) * C::Q_BLOCK + sw128(row, (dim & 63) * 2);
        sts128(to + C::QHI, pack_f16(h[0], h[2]), pack_f16(h[1], h[3]), pack_f16(h[4], h[6]), pack_f16(h[5], h[7]));
        sts128(to + C::QLO, pack_f16(l[0], l[2]), pack_f16(l[1], l[3]), pack_f16(l[4], l[6]), pack_f16(l[5], l[7]));
      }
    }
    __syncthreads();                                             // the tokens' rows are known to all

    // K of tile j: a thread's 16 codes of a token become 32 bytes; of four neighbouring dimensions the even ones come first
    auto stage_k = [&](int j) {
#pragma unroll
      for (int i = 0; i < MT * D / 16 / MANY_THREADS; i++) {
        const int c = i * MANY_THREADS + tid, tok = c / (D / 16), p = c % (D / 16);
        const int64_t r = row_at[j & 1][tok];
        const uint4 x = r < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(a.k + r * D) + p);
        const uint32_t to = sm_base + C::K + (p >> 2) * C::K_BLOCK;
        sts128(to + sw128(tok, (p & 3) * 32), codes_even(x.x), codes_odd(x.x), codes_even(x.y), codes_odd(x.y));
        sts128(to + sw128(tok, (p & 3) * 32 + 16), codes_even(x.z), codes_odd(x.z), codes_even(x.w), codes_odd(x.w));
      }
    };
    // V of tile j, transposed: a thread takes four dimensions (word L of a row) of eight tokens.  Dimension 4 L + q is row
    // HD * (L / (HD / 4)) + q * (HD / 4) + L % (HD / 4) of the tile: neighbouring lanes write neighbouring rows (no bank
    // conflict), and the columns of O that a thread reads are whole runs of four dimensions.
    auto stage_v = [&](int j) {
      constexpr int W = D / 4;                                   // words of a row
      const int L = tid % W, oct = tid / W;                      // eight tokens oct * 8 ..
      if (oct < MT / 8) {
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int64_t r = row_at[j & 1][oct * 8 + i];
          x[i] = r < 0 ? 0u : __ldg(reinterpret_cast<const uint32_t*>(a.v + r * D) + L);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t y[4];
#pragma unroll
          for (int i = 0; i < 4; i++) y[i] = __byte_perm(x[2 * i], x[2 * i + 1], h ? 0x7632 : 0x5410);
#pragma unroll
          for (int odd = 0; odd < 2; odd++) {
            const int r = (L / (HD / 4)) * HD + (2 * h + odd) * (HD / 4) + L % (HD / 4);
            const uint32_t to = sm_base + C::V + sw128(r, oct * 16);
            if (odd) sts128(to, codes_odd(y[0]), codes_odd(y[1]), codes_odd(y[2]), codes_odd(y[3]));
            else sts128(to, codes_even(y[0]), codes_even(y[1]), codes_even(y[2]), codes_even(y[3]));
          }
        }
      }
    };

    uint64_t o2[HD / 2];                                         // pairs of outputs, in the order of the tile's rows
#pragma unroll
    for (int i = 0; i < HD / 2; i++) o2[i] = 0;
    float c_run = C_NONE, l_run = 0.0f;
    stage_k(tile0);

    for (int j = tile0; j < tile1; j++) {
      fence_proxy();                                             // the tensor cores read what the threads wrote
      fence_before();
      __syncthreads();
      if (tid == 0) {
        fence_after();
        constexpr uint32_t idesc = idesc_f16(LANES, MT);
#pragma unroll
        for (int s = 0; s < D / 16; s++) {                       // 16 dimensions = 32 bytes along K per instruction
          const uint64_t kd = smem_desc(sm_base + C::K + (s >> 2) * C::K_BLOCK) + 2 * (s & 3);
          const uint32_t q = sm_base + (s >> 2) * C::Q_BLOCK;
          mma_ss(tmem + TM_SHI, smem_desc(q + C::QHI) + 2 * (s & 3), kd, idesc, s != 0);
          mma_ss(tmem + TM_SLO, smem_desc(q + C::QLO) + 2 * (s & 3), kd, idesc, s != 0);
        }
        mma_commit(bar_addr);
      }
      float k_next = 0.0f, v_next = 0.0f;
      int64_t row_after = -1;
      if (tid < MT) {
        if (row_next >= 0) { k_next = __ldg(a.ks + row_next); v_next = __ldg(a.vs + row_next); }
        row_after = find_row(j + 2);
      }
      stage_v(j);
      alive = wait_mma();
      if (!alive) break;
      fence_after();
      if (j + 1 < tile1 && tid < 2 * MT) {                       // the next tile's rows on their way into L1
        const int64_t r = row_at[(j + 1) & 1][tid & (MT - 1)];
        if (r >= 0) asm volatile("prefetch.global.L1 [%0];" ::"l"((tid < MT ? a.k : a.v) + r * D));
      }

      // ---- which of this thread's tokens its row sees
      uint32_t seen = tok_there[j & 1][half];
      const int64_t from = (int64_t)j * MT + half * 32 - first;  // place of the half tile's first token among the new rows
      if (from + 32 > 0) {
        const uint32_t before = from >= 0 ? 0u : (from <= -32 ? ~0u : (1u << (int)-from) - 1);
        uint32_t fresh;
        if (a.tree) fresh = from >= 64 ? 0u : (from >= 0 ? (uint32_t)(row_seen >> (int)from) : (uint32_t)(row_seen << (int)-from));
        else {
          const int64_t k = (int64_t)row_t + 1 - from;           // tokens of the half tile up to the row itself
          fresh = k <= 0 ? 0u : (k >= 32 ? ~0u : (1u << (int)k) - 1);
        }
        seen &= before | fresh;
      }
      seen >>= copy * NC;
      const bool all = NC == 32 ? seen == ~0u : (seen & ((1u << (NC & 31)) - 1)) == (1u << (NC & 31)) - 1;
      const uint64_t rs2 = f2_dup(rs);

      // scores c .. c + CW of this thread: z = (S_hi + S_lo) * scale_k * rs
      auto scores = [&](int c, float (&z)[CW]) {
        uint32_t hi[CW], lo[CW];
        tm_ld(lane_tm + TM_SHI + col0 + c, hi);
        tm_ld(lane_tm + TM_SLO + col0 + c, lo);
        tm_wait_ld(hi);
        tm_wait_ld(lo);
#pragma unroll
        for (int i = 0; i < CW; i += 4) {
          const float4 k = *reinterpret_cast<const float4*>(&tok_ks[j & 1][col0 + c + i]);
          const uint64_t s0 = f2_add(f2_pack(__uint_as_float(hi[i]), __uint_as_float(hi[i + 1])), f2_pack(__uint_as_float(lo[i]), __uint_as_float(lo[i + 1])));
          const uint64_t s1 = f2_add(f2_pack(__uint_as_float(hi[i + 2]), __uint_as_float(hi[i + 3])), f2_pack(__uint_as_float(lo[i + 2]), __uint_as_float(lo[i + 3])));
          f2_unpack(f2_mul(f2_mul(s0, f2_pack(k.x, k.y)), rs2), z[i], z[i + 1]);
          f2_unpack(f2_mul(f2_mul(s1, f2_pack(k.z, k.w)), rs2), z[i + 2], z[i + 3]);
        }
        if (!all) {
#pragma unroll
          for (int i = 0; i < CW; i++)
            if (!((seen >> (c + i)) & 1)) z[i] = NEG_INF;
        }
      };
      float top = NEG_INF;
#pragma unroll
      for (int c = 0; c < NC; c += CW) {
        float z[CW];
        scores(c, z);
#pragma unroll
        for (int i = 0; i < CW; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(&tok_lv[j & 1][col0 + c + i]);
          top = fmaxf(fmaxf(top, fmaxf(z[i] + v.x, z[i + 1] + v.y)), fmaxf(z[i + 2] + v.z, z[i + 3] + v.w));
        }
      }
      // the other half of the row: warps w and w + 4 meet at a barrier of their own (two barriers follow before the slot
      // is written again)
      xchg[half][row] = top;
      pair_barrier(warp & 3);
      top = fmaxf(top, xchg[half ^ 1][row]);
      const float c_new = fmaxf(c_run, top - 10.0f);
      const float fold = ex2(c_run - c_new);
      c_run = c_new;
      uint64_t l2 = 0;
      const uint64_t c2 = f2_dup(c_new), magic2 = f2_dup(12582912.0f);
#pragma unroll
      for (int s = 0; s < 2; s++) {                              // 16 tokens = one k-step of P V = 8 + 8 columns of weights
        uint32_t ph[8], pl[8];
        if (CS == 1 || (CS == 2 ? copy == s : (copy >> 1) == s)) {
          constexpr int W = CW;                                  // 16, or 8 when four copies share the tile
          float z[W];
          scores(CS == 1 ? s * 16 : 0, z);
          uint32_t h[W / 2], l[W / 2];
#pragma unroll
          for (int i = 0; i < W; i += 2) {
            const float2 v = *reinterpret_cast<const float2*>(&tok_vs[j & 1][col0 + (CS == 1 ? s * 16 : 0) + i]);
            float d0, d1, x0, x1, y0, y1;
            f2_unpack(f2_sub(f2_pack(z[i], z[i + 1]), c2), d0, d1);
            const uint64_t p = f2_pack(ex2(d0), ex2(d1));
            l2 = f2_add(l2, p);
            const uint64_t w = f2_mul(p, f2_pack(v.x, v.y));
            const uint64_t hw = f2_sub(f2_add(w, magic2), magic2);
            f2_unpack(hw, x0, x1);
            f2_unpack(f2_sub(w, hw), y0, y1);
            h[i / 2] = pack_f16(x0, x1);
            l[i / 2] = pack_f16(y0, y1);
          }
          if (CS <= 2) {
#pragma unroll
            for (int i = 0; i < 8; i++) { ph[i] = h[i % (W / 2)]; pl[i] = l[i % (W / 2)]; }
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              ph[i] = (copy & 1) ? 0u : h[i % (W / 2)]; ph[4 + i] = (copy & 1) ? h[i % (W / 2)] : 0u;
              pl[i] = (copy & 1) ? 0u : l[i % (W / 2)]; pl[4 + i] = (copy & 1) ? l[i % (W / 2)] : 0u;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) ph[i] = pl[i] = 0u;
        }
        // over the scores S_hi of the same 16 tokens (of this half of the row: nobody else's)
        tm_st(lane_tm + TM_SHI + half * 32 + s * 16, ph);
        tm_st(lane_tm + TM_SHI + half * 32 + s * 16 + 8, pl);
      }
      {
        float p0, p1;
        f2_unpack(l2, p0, p1);
        l_run = fmaf(l_run, fold, (p0 + p1) * P_UNIT);
      }
      if (tid < MT) {
        put_scales(j + 1, row_next, k_next, v_next);
        row_at[j & 1][tid] = row_after;                          // tile j + 2's: V of tile j, the last to use this slot, is staged
        row_next = row_after;
      }
      tm_wait_st();
      fence_proxy();                                             // the V tile
      fence_before();
      __syncthreads();
      if (tid == 0) {
        fence_after();
        constexpr uint32_t idesc = idesc_f16(LANES, D);
#pragma unroll
        for (int s = 0; s < 4; s++) {                            // 16 tokens per instruction; the small halves first
          const uint64_t vd = smem_desc(sm_base + C::V) + 2 * s;
          mma_ts(tmem + TM_O, tmem + TM_SHI + s * 16 + 8, vd, idesc, s != 0);
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const uint64_t vd = smem_desc(sm_base + C::V) + 2 * s;
          mma_ts(tmem + TM_O, tmem + TM_SHI + s * 16, vd, idesc, 1);
        }
        mma_commit(bar_addr);
      }
      if (j + 1 < tile1) stage_k(j + 1);
      alive = wait_mma();
      if (!alive) break;
      fence_after();
      const uint64_t fold2 = f2_dup(fold);
#pragma unroll
      for (int c = 0; c < HD; c += 16) {
        uint32_t t[16];
        tm_ld(lane_tm + TM_O + half * HD + c, t);
        tm_wait_ld(t);
#pragma unroll
        for (int i = 0; i < 16; i += 2)
          o2[(c + i) / 2] = f2_fma(o2[(c + i) / 2], fold2, f2_pack(__uint_as_float(t[i]), __uint_as_float(t[i + 1])));
      }
      fence_before();                                            // the next tile's products overwrite S and O only after these loads
    }
    if (!alive) break;

    // ---- the rows of the piece: halves and copies joined, then to the result or to the block's slot
    xchg[half][row] = l_run;
    if (half == 0) copy_c[row] = c_run;
    __syncthreads();                                             // all products are done: Q's tiles are free
    float* res = reinterpret_cast<float*>(sm + C::QHI);          // [128][D], 16-byte pieces XOR lane % 8
    {
      float c_max = copy_c[rq];
#pragma unroll
      for (int k = 1; k < CS; k++) c_max = fmaxf(c_max, copy_c[k * ROWS + rq]);
      const uint64_t f2 = f2_dup(ex2(c_run - c_max));
#pragma unroll
      for (int i = 0; i < HD / 4; i++) {                         // dimensions half * HD + 4 i .. + 3: four rows of the V tile
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int k = q * (HD / 4) + i;
          float x0, x1;
          f2_unpack(f2_mul(o2[k / 2], f2), x0, x1);
          v[q] = (k & 1) ? x1 : x0;
        }
        const int piece = half * (HD / 4) + i;
        *reinterpret_cast<float4*>(res + row * D + ((piece ^ (row & 7)) << 2)) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == tiles;
    if (tile0 == 0 && !whole && tid == 0)
      a.items[blockIdx.x] = make_int4(e, head, kv_run_of(run.all, at + tiles - 1), 1);
    float* slot = a.slots + (int64_t)(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * KV_SLOT_FLOATS;
    for (int x = tid; x < rows_here * (D / 4); x += MANY_THREADS) {
      const int r = x / (D / 4), p = x % (D / 4);
      float c_max = copy_c[r], sum = 0.0f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 1; k < CS; k++) c_max = fmaxf(c_max, copy_c[k * ROWS + r]);
#pragma unroll
      for (int k = 0; k < CS; k++) {
        const int ln = k * ROWS + r;
        const float4 y = *reinterpret_cast<const float4*>(res + ln * D + ((p ^ (ln & 7)) << 2));
        sum = fmaf(xchg[0][ln] + xchg[1][ln], ex2(copy_c[ln] - c_max), sum);
        v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
      }
      if (whole) {
        const float inv = sum == 0.0f ? 0.0f : P_UNIT / sum;
        int t;
        *reinterpret_cast<float4*>(a.out + row_offset(a, b, head, rb * ROWS + r, a.ld_o, D, t) + p * 4) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      } else {
        __stcg(reinterpret_cast<float4*>(slot + r * D) + p, v);
        if (p == 0) { __stcg(slot + ROWS * D + r, c_max); __stcg(slot + ROWS * D + ROWS + r, sum); }
      }
    }
    __syncthreads();                                             // Q's tiles are about to be written again
    at += tile1 - tile0;
    left -= tile1 - tile0;
    tile0 = 0;
    if (++head == a.g.heads) { head = 0; e++; }
  }

  if (!alive) {
    if (tid == 0) atomicOr(a.status, STATUS_SDPA_WAIT_TIMEOUT);
    const uint64_t t0 = gtimer();
    while (gtimer() - t0 < 2000000ull) __nanosleep(1000);        // products in flight finish before tensor memory is released
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
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
  const unsigned grid = (unsigned)ctx->sm_count * KV_BLOCKS_PER_SM;
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

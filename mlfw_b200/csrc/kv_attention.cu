// Attention over the int8 key/value cache for few query rows (decoding steps, small trees), and the choice of the kernel by rows.
// What is computed and in which arithmetic stands in kv_attention.cuh.
#include "kv_attention.cuh"

namespace b200q {

namespace {

// Byte offset of 16-byte piece c of token t in a tile of [16][D]: swizzled so that neither the reads of K (eight tokens'
// rows, four neighbouring pieces each) nor those of V (a piece of every second token) meet in a bank.
template <int D>
__device__ __forceinline__ uint32_t k_at(int t, int c) {
  if (D == 128) return (uint32_t)(t * 128 + ((c ^ ((t & 1) << 2)) << 4));
  return (uint32_t)((t >> 1) * 128 + (((((t & 1) << 2) | c) ^ (((t >> 1) & 3) << 1)) << 4));
}
template <int D>
__device__ __forceinline__ uint32_t v_at(int t, int c) {
  if (D == 128) return (uint32_t)(t * 128 + ((c ^ (((t >> 1) & 3) << 1)) << 4));
  return k_at<64>(t, c);
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows (a decoding step: the query heads that share a cache head; small trees), four at a time, on the integer tensor
// cores: m16n8k32 with the codes as they are, so that K needs no conversion and V a transpose of bytes.  Items of more than
// four rows are several items, whose tiles come from L2 after the first.  A query row and a row of weights are 32-bit
// fixed-point numbers in four 8-bit digits, and the sixteen rows of the A operand are four rows times four digits: of row r
// the rows 2 r and 2 r + 1 hold the digits 3 and 2, the rows 8 + 2 r and 9 + 2 r the digits 1 and 0.  A thread of an even
// row therefore finds sum d3 code and sum d1 code, its neighbour in the odd row those of d2 and d0; each takes one of their two
// columns after one exchange, so no score is computed twice.  Sums are 32-bit integers and exact: scores carry the rounding of
// adding the digits, and the outputs are added up without rounding until a row's c changes (or 2^15 tokens have passed), when
// they are converted, scaled and moved to binary32.  c = floor(top) - 28, an integer, so that moving is exact; 3.75 bits are left
// before a larger weight (below 2^32) moves it.  The unit is thus 2^-28 of the row's largest weight or less.  Many weights below it
// must neither vanish nor count double, so a weight is rounded down after adding `dither` between 0 and 1, which goes round by the golden
// ratio from tile to tile: over many tokens a unit's share of all weights is kept, and what is left of a token's rounding is noise.
// The sum of p carries the rounding of each addition into the next one for the same reason.
// Scales of V are taken relative to a power of two 2^kappa, that of the first tile's largest until one 2^60 times as large comes, so
// that neither tiny nor huge values leave binary32 anywhere on the way: 2^kappa meets the quotient of the two sums at the end.
// Scores more than 2^20 from zero, where binary32 has no room for a difference of a few units, are taken relative to m, a score of
// the row that is, so c stays small.  m, kappa and c change in a branch that is entered when a row's largest weight
// leaves its window (`limit`), on every tile once m is not zero.
//
// About 470 instructions per tile of 32 tokens of 128 dimensions, 450 of 64, all included (conversion of the codes to binary16 for
// m16n8k16, tried first, took 1300).  Bound by reading the cache: 5.3 TB/s of the 6.5 measured at 48 sequences of up to 6000
// tokens, 32 heads on 8, 128 wide (75 to 80 us from run to run, median 78; 412 MB), launch, search of the runs and joining included.  One block per SM, eight
// warps (D = 128: 64 integer sums and 32 outputs per thread, which need more than the 168 registers that twelve warps leave)
// with two tiles each in flight, or twelve (D = 64) with three.  Where 8 x 2 took 75 us, 12 x 2 took 85, 10 x 2 83, 8 x 3 77,
// 6 x 3 76, 4 x 4 86; 64 wide, 64 sequences of up to 2000 tokens, 12 heads, 12 x 3: 34.9 us, 16 x 3: 38.9, 8 x 4: 37.1,
// 12 x 2: 35.1.
// ---------------------------------------------------------------------------------------------------------------
constexpr int IT = 32;                                          // tokens of a tile: two runs of sixteen, each in one page
template <int D>
struct Four {
  static constexpr int WARPS = D == 128 ? 8 : 12, STAGES = D == 128 ? 2 : 3;
  static constexpr int GRAN = 2 * KV_TILE * D + 2 * KV_TILE * 4, TILE = 2 * GRAN;   // sixteen tokens: K and V codes, K and V scales
  static constexpr int RING = WARPS * STAGES * TILE, SLOT = 4 * (D + 4) * 4, SMEM = RING + WARPS * SLOT;
};
__device__ __forceinline__ void imma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // s8 x s8
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void imma_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void imma_u8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // u8 x s8
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float lds_f(uint32_t a) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(a));
  return r;
}

// One item after another along a run, as a warp walks it.
struct Item {
  int e, head, b, rb, n, tiles;
  int64_t first, vis;
  template <int ROWS>
  __device__ __forceinline__ void load(const AttnArgs& a, int row_blocks) {   // skips what has no tile; the caller knows that one follows
    while (true) {
      b = e / row_blocks; rb = e - b * row_blocks;
      first = a.start[b];
      n = kv_rows_in_use(a.count, b, a.T);
      tiles = kv_tiles(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr, IT);
      if (tiles != 0) break;
      e++;
    }
    vis = kv_visible(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr);
  }
};

// Pieces first .. last of an item, at(i) each, added up in that order: outputs `mine` of row r in units of 2^(m + c + kappa), l in units of
// 2^(m + c); behind the outputs of a piece stand c, l, kappa and m of its rows.  `ld` loads four floats.  A chain of latencies: four pieces
// at a time (one sequence of 2000 tokens, 12 heads of 64, joined between blocks: 11.3 us, two at a time in the second loop 11.7).
template <int D, typename At, typename Ld>
__device__ __forceinline__ void join_pieces(int first, int last, At at, Ld ld, int r, int mine, float (&val)[D / 8], float4& row) {
  float top = C_NONE, kappa = -200.0f, far = C_NONE, sum = 0.0f;   // far: the largest m of a piece that has seen something
  bool some = false;
#pragma unroll 4
  for (int i = first; i <= last; i++) {
    const float4 x = ld(at(i) + 4 * D + 4 * r);
    top = fmaxf(top, x.x);
    kappa = fmaxf(kappa, x.z);
    far = fmaxf(far, x.x > C_SEEN ? x.w : C_NONE);
    some |= x.w != 0.0f;
  }
  if (__builtin_expect(some, 0)) {
    top = C_NONE;
    for (int i = first; i <= last; i++) {
      const float4 x = ld(at(i) + 4 * D + 4 * r);
      top = fmaxf(top, x.x + (x.w - far));
    }
  }
#pragma unroll
  for (int i = 0; i < D / 8; i++) val[i] = 0.0f;
#pragma unroll 4
  for (int i = first; i <= last; i++) {
    const float4 x = ld(at(i) + 4 * D + 4 * r);
    const float e = (some ? x.x + (x.w - far) : x.x) - top, f = ex2(e + (x.z - kappa));
    sum = fmaf(x.y, ex2(e), sum);
#pragma unroll
    for (int k = 0; k < D / 8; k += 4) {
      const float4 v = ld(at(i) + mine + k);
      val[k] = fmaf(v.x, f, val[k]); val[k + 1] = fmaf(v.y, f, val[k + 1]); val[k + 2] = fmaf(v.z, f, val[k + 2]); val[k + 3] = fmaf(v.w, f, val[k + 3]);
    }
  }
  row = make_float4(top, sum, kappa, some && far > C_SEEN ? far : 0.0f);
}

// Every warp has a run of its own, a part of the block's, and a ring that it keeps full across the items of its run; the warps
// never wait for one another.  Results of an item that several warps of the block worked on are joined by the last of them
// through shared memory, and those of an item that several blocks worked on by the last warp of the last block.
template <int D>
__global__ void __launch_bounds__(32 * Four<D>::WARPS, 1) kv_attention_four_kernel(const AttnArgs a, int row_blocks) {
  using C = Four<D>;
  constexpr int ROWS = 4, WARPS = C::WARPS, ST = C::STAGES, KS = D / 32, CH = D / 8, W = D / 32;
  constexpr float P_UNIT = 0x1p-22f;                            // sums of p are held times this: 2^24 keys of weight 2^120 stay finite
  constexpr float C_BELOW = 28.0f, C_SLACK = 31.75f, GOLDEN = 0.61803399f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int arrived[WARPS];                                // pieces of an item within the block, by the first warp that has it
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3, r = g8 >> 1, odd = g8 & 1;
  const uint32_t ring = smem_u32(smem) + warp * (ST * C::TILE);
  const uint32_t k_dst = ring + k_at<D>(lane / (D / 16), lane % (D / 16)), v_dst = ring + KV_TILE * D + v_at<D>(lane / (D / 16), lane % (D / 16));
  const uint32_t k_src = ring + k_at<D>(g8, t4);
  const uint32_t v_src = ring + KV_TILE * D + (D == 128 ? v_at<D>(2 * t4, g8) : v_at<D>(2 * t4, g8 >> 1) + (g8 & 1) * 8);
  const uint32_t s_src = ring + 2 * KV_TILE * D + (2 * t4 + odd) * 4;
  // weights of this thread's two sums; selectors of its two digits among (own, partner's) weights in the order of the tokens
  const float w0 = odd ? 0x1p16f : 0x1p24f, w2 = odd ? 1.0f : 0x1p8f;
  const uint32_t sel = odd ? 0x0426u : 0x5173u;

  kv_after_previous();
  if (tid < WARPS) arrived[tid] = 0;
  // At least 8 tiles per run, or whole items: one sequence of 500 tokens, 12 heads of 64, 8.5 us (runs of 8 tiles 9.5), 2000 tokens
  // 11.3 (whole items 12.6); 4 sequences of 1000 tokens, 32 heads on 8 of 128, 11.9 (12.3).
  const Run run = find_run<ROWS, IT, 8, true>(a, row_blocks);   // (its barriers publish `arrived`)
  if (run.begin == run.end) return;
  const KvRuns parts = kv_runs(run.end - run.begin, 1, WARPS);
  if (warp >= parts.runs) return;
  const int64_t begin = kv_run_begin(parts, warp);
  int left = (int)(kv_run_begin(parts, warp + 1) - begin);      // this warp's tiles: below 2^31 / 148 blocks / warps
  int64_t at = run.begin + begin;                               // first tile of the piece among all tiles

  Item it;                                                      // the item of the piece
  it.e = run.e; it.head = run.head;
  it.load<ROWS>(a, row_blocks);
  int tile = run.tile;
  for (int64_t skip = begin; skip > 0;) {                       // from the block's first tile to the warp's
    const int64_t rest = (int64_t)(a.g.heads - it.head) * it.tiles - tile;
    if (skip >= rest) {
      skip -= rest;
      it.e++; it.head = 0; tile = 0;
      it.load<ROWS>(a, row_blocks);
    } else {
      const int64_t to = it.head * (int64_t)it.tiles + tile + skip;
      it.head = (int)kv_div(to, it.tiles);
      tile = (int)(to - (int64_t)it.head * it.tiles);
      skip = 0;
    }
  }

  // ---- the ring: tiles in the order of the run, ST - 1 ahead of their use.  `ahead` walks by itself.  A tile of 32 tokens lies in
  // one page (pages of 32 tokens or more: one address for all of it, looked up when a page begins) or in two of 16; its
  // pages are looked up a tile early.  -1: nothing there is visible.  Positions fit 32 bits: start is below 2^31, T at most 2^24.
  const int shift = a.g.page_shift;
  const bool wide = shift >= 5;
  const uint32_t in_page = (1u << shift) - 1, page_cells = (uint32_t)a.g.heads << shift;   // < 2^24
  int ahead_e = it.e, ahead_head = it.head, ahead_tiles = it.tiles, ahead_tile = tile, ahead_left = left, page0 = -1, page1 = -1;
  uint32_t ahead_vis = (uint32_t)it.vis, ahead_cell = (uint32_t)it.head << shift;   // first cell of the head in a page
  const int32_t* ahead_table = a.page_table + (int64_t)it.b * a.g.max_pages;
  const int8_t *k_lane = a.k + lane * 16, *v_lane = a.v + lane * 16;
  const float* s_lane = (lane < 8 ? a.ks : a.vs) + (lane & 7) * 4;                          // lanes 0 .. 15: scales of K, of V
  const uint32_t s_dst = ring + 2 * KV_TILE * D + ((lane >> 2) & 1) * C::GRAN + ((lane >> 3) & 1) * 64 + (lane & 3) * 16;
  uint32_t there = 0;                                           // two bits per tile in the ring, the oldest lowest
  auto look_up = [&](bool anew) {                               // the pages of the tile `ahead`
    const uint32_t pos = (uint32_t)ahead_tile * IT;
    if (wide) {
      if (anew || (pos & in_page) == 0) page0 = pos < ahead_vis ? __ldcg(ahead_table + (pos >> shift)) : -1;
    } else {
      page0 = pos < ahead_vis ? __ldcg(ahead_table + (pos >> 4)) : -1;
      page1 = pos + 16 < ahead_vis ? __ldcg(ahead_table + (pos >> 4) + 1) : -1;
    }
  };
  auto fetch = [&](int s, int place) {
    if (ahead_left > 0) {
      const uint32_t pos = (uint32_t)ahead_tile * IT, to = s * C::TILE;
      if (wide) {
        if ((uint32_t)page0 < (uint32_t)a.g.pages) {
          const uint64_t cell = (uint64_t)(uint32_t)page0 * page_cells + (ahead_cell + (pos & in_page));
          const int8_t *kp = k_lane + cell * D, *vp = v_lane + cell * D;
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int x = 0; x < D / 32; x++) {
              cp16(k_dst + to + h * C::GRAN + x * 512, kp + h * 16 * D + x * 512);
              cp16(((D == 128 && (x & 1)) ? v_dst ^ 64u : v_dst) + to + h * C::GRAN + x * 512, vp + h * 16 * D + x * 512);
            }
          if (lane < 16) cp16(s_dst + to, s_lane + cell);
          there |= 3u << (2 * place);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int page = h ? page1 : page0;
          if ((uint32_t)page < (uint32_t)a.g.pages) {
            const uint64_t cell = (uint64_t)(uint32_t)page * page_cells + ahead_cell;
            const int8_t *kp = k_lane + cell * D, *vp = v_lane + cell * D;
#pragma unroll
            for (int x = 0; x < D / 32; x++) {
              cp16(k_dst + to + h * C::GRAN + x * 512, kp + x * 512);
              cp16(((D == 128 && (x & 1)) ? v_dst ^ 64u : v_dst) + to + h * C::GRAN + x * 512, vp + x * 512);
            }
            if (lane < 16 && (lane & 4) == 0) cp16(s_dst + to + h * C::GRAN, s_lane + cell);
            there |= (1u + h) << (2 * place);
          }
        }
      }
      ahead_left--;
      bool anew = false;
      if (++ahead_tile == ahead_tiles) {
        ahead_tile = 0;
        anew = true;
        ahead_cell += 1u << shift;
        if (++ahead_head == a.g.heads) {
          ahead_head = 0; ahead_cell = 0; ahead_e++;
          if (ahead_left > 0) {
            Item next;
            next.e = ahead_e;
            next.load<ROWS>(a, row_blocks);
            ahead_e = next.e; ahead_tiles = next.tiles; ahead_vis = (uint32_t)next.vis;
            ahead_table = a.page_table + (int64_t)next.b * a.g.max_pages;
          }
        }
      }
      if (ahead_left > 0) look_up(anew);
    }
    cp_commit();
  };
  look_up(true);
#pragma unroll
  for (int s = 0; s < ST - 1; s++) fetch(s, s);

  int slot = 0;
  while (left > 0) {
    const int tile0 = tile, tile1 = min(it.tiles, tile0 + left), rows_here = min(ROWS, it.n * a.group - it.rb * ROWS);
    const int64_t first = it.first;
    const int plain = first <= 0 ? 0 : (int)(first / IT);       // tiles of cached tokens only
    if (lane == 0 && (first < 0 || first + it.n > (a.g.max_pages << a.g.page_shift))) atomicOr(a.status, STATUS_BAD_INDEX);

    // ---- the query row r: digits of dimensions 64 m + 16 t4 + 8 h + (0..7), k-step 2 m + h
    float rs;
    int row_t;
    uint64_t row_seen;
    uint32_t qa[KS][4];
    {
      const bool used = r < rows_here;
      int t = 0;
      const float* src = a.q + row_offset(a, it.b, it.head, it.rb * ROWS + (used ? r : 0), a.ld_q, D, t);
      row_t = used ? t : -1;
      row_seen = used && a.tree ? a.tree[(int64_t)it.b * a.T + t] : 0;
      float4 x[2 * KS];
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < 2 * KS; s++) {
        x[s] = used ? __ldcg(reinterpret_cast<const float4*>(src + (s >> 2) * 64 + t4 * 16 + (s & 3) * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max(max(top, max(__float_as_uint(x[s].x) & 0x7fffffffu, __float_as_uint(x[s].y) & 0x7fffffffu)),
                  max(__float_as_uint(x[s].z) & 0x7fffffffu, __float_as_uint(x[s].w) & 0x7fffffffu));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool finite = top < 0x7f800000u;
      const int ex = max((int)(top >> 23), 30) - 127;           // exponent of the row's largest element; tiny rows keep fewer digits
      const float up = finite ? pow2(29 - ex) : 0.0f;           // |x| <= 2^30
      rs = finite ? a.scale_log2e * pow2(ex - 29) : __int_as_float(0x7fc00000);   // a NaN or an infinity in the row: every score NaN
#pragma unroll
      for (int s = 0; s < 2 * KS; s++) {
        uint32_t d[4];
        const float y[4] = {x[s].x, x[s].y, x[s].z, x[s].w};
#pragma unroll
        for (int c = 0; c < 4; c++) d[c] = ((uint32_t)__float2int_rn(finite ? y[c] * up : 0.0f) + 0x00808080u) ^ 0x00808080u;   // bytes = signed digits
        const uint32_t hi01 = __byte_perm(d[0], d[1], odd ? 0x0062 : 0x0073), hi23 = __byte_perm(d[2], d[3], odd ? 0x0062 : 0x0073);
        const uint32_t lo01 = __byte_perm(d[0], d[1], odd ? 0x0040 : 0x0051), lo23 = __byte_perm(d[2], d[3], odd ? 0x0040 : 0x0051);
        qa[s >> 1][(s & 1) * 2] = __byte_perm(hi01, hi23, 0x5410);
        qa[s >> 1][(s & 1) * 2 + 1] = __byte_perm(lo01, lo23, 0x5410);
      }
    }

    int acc[CH][4];
    float o[CH][2], c_run = C_NONE, limit = NEG_INF, m = 0.0f, l = 0.0f, l_over = 0.0f, kf = 0.0f;   // kf: 2^-kappa, 0 until a tile has a scale
    float dither = (2 * t4 + odd) * 0.125f + 0.0625f;
#pragma unroll
    for (int i = 0; i < CH; i++) { acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0; o[i][0] = o[i][1] = 0.0f; }
    int since = 0;                                              // tiles in the integer sums
    auto move_sums = [&](float f) {                             // o = (o + the integer sums) * f
#pragma unroll
      for (int i = 0; i < CH; i++) {
        o[i][0] = (o[i][0] + fmaf((float)acc[i][0], w0, (float)acc[i][2] * w2)) * f;
        o[i][1] = (o[i][1] + fmaf((float)acc[i][1], w0, (float)acc[i][3] * w2)) * f;
        acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
      }
      since = 0;
    };

#pragma unroll 1
    for (int i = tile0; i < tile1; i++) {
      cp_wait<ST - 2>();
      __syncwarp();
      const bool there0 = there & 1, there1 = there & 2;
      there >>= 2;
      const uint32_t here = slot * C::TILE;
      fetch(slot == 0 ? ST - 1 : slot - 1, ST - 2);
      slot = slot + 1 == ST ? 0 : slot + 1;

      // ---- scores: four blocks of eight tokens; this thread's are 8 j + 2 t4 + odd
      float z[4], vs[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t at_k = here + (j >> 1) * C::GRAN + (j & 1) * 8 * D;
        int c[4];
#pragma unroll
        for (int mm = 0; mm < D / 64; mm++) {
          const uint4 x = lds128((mm ? k_src ^ 64u : k_src) + at_k);
          if (mm == 0) imma_first(c, qa[0][0], qa[0][1], qa[0][2], qa[0][3], x.x, x.y);
          else imma(c, qa[2 * mm][0], qa[2 * mm][1], qa[2 * mm][2], qa[2 * mm][3], x.x, x.y);
          imma(c, qa[2 * mm + 1][0], qa[2 * mm + 1][1], qa[2 * mm + 1][2], qa[2 * mm + 1][3], x.z, x.w);
        }
        const float s0 = fmaf((float)c[0], w0, (float)c[2] * w2), s1 = fmaf((float)c[1], w0, (float)c[3] * w2);
        const float got = __shfl_xor_sync(0xffffffffu, odd ? s0 : s1, 4);
        const uint32_t at_s = s_src + here + (j >> 1) * C::GRAN + (j & 1) * 32;
        z[j] = ((odd ? s1 : s0) + got) * (lds_f(at_s) * rs);
        vs[j] = lds_f(at_s + 64);
      }
      const bool all = i < plain && there0 && there1;           // the same in the whole warp
      if (!all) {
        const int64_t pos = (int64_t)i * IT, end = min(it.vis, first + it.n);
        if (lane == 0 && ((!there0 && pos < it.vis) || (!there1 && pos + 16 < it.vis))) atomicOr(a.status, STATUS_BAD_INDEX);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t p = pos + 8 * j + 2 * t4 + odd, q = p - first;
          const bool held = (j < 2 ? there0 : there1) && p < end;
          if (!held) vs[j] = 0.0f;                              // behind the last row in use anything may stand
          if (!(held && (q < 0 || (a.tree ? (row_seen >> q) & 1 : q <= row_t)))) z[j] = NEG_INF;
        }
      }
      auto kappa_of = [](float big) {                           // 2^-kappa of a tile's scales, 0 where none is above zero
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
        return big > 0.0f ? pow2(127 - min(max(__float_as_int(big) >> 23, 1), 253)) : 0.0f;
      };
      if (kf == 0.0f) kf = kappa_of(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])));
      auto top_of = [&] {                                       // the row's largest weight in units of log2
        float top = NEG_INF;
#pragma unroll
        for (int j = 0; j < 4; j++) top = fmaxf(top, z[j] + fmaxf(log2_raw(vs[j]), -88.0f));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        return fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      };
#pragma unroll
      for (int j = 0; j < 4; j++) vs[j] *= kf;
      float top = top_of();
      if (__any_sync(0xffffffffu, top > limit) || since == 1024) {
        float c_old = c_run, lower = 0.0f, g = 1.0f;
        const bool big_vs = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])) > 0x1p60f;
        if (__builtin_expect(__any_sync(0xffffffffu, big_vs || m != 0.0f || (fabsf(top) > FAR && top > NEG_INF)), 0)) {
          if (__any_sync(0xffffffffu, big_vs)) {                // another kappa; vs may be infinite
            float big = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              vs[j] = vs[j] == 0.0f ? 0.0f : lds_f(s_src + here + (j >> 1) * C::GRAN + (j & 1) * 32 + 64);
              big = fmaxf(big, vs[j]);
            }
            const float kf_old = kf;
            kf = kappa_of(big);
#pragma unroll
            for (int j = 0; j < 4; j++) vs[j] *= kf;
            top = top_of();
            // the integer sums are in units of 2^(c + kappa).  c goes down by what kappa goes up, so that a row that does not see the
            // large values keeps its digits; by 2^80 at most, which the sums of p have room for
            const int up = (__float_as_int(kf_old) - __float_as_int(kf)) >> 23;
            g = up > 126 ? 0.0f : pow2(-up);
            lower = fminf((float)up, 80.0f);
          }
          float raw[4];                                         // z - m is exact where it matters, from the scores themselves
#pragma unroll
          for (int j = 0; j < 4; j++) raw[j] = z[j];
          for (int k = 0; k < 8; k++) {                         // each round leaves a rounding of the one before: 2^-23 of it
#pragma unroll
            for (int j = 0; j < 4; j++) z[j] = raw[j] - m;
            top = top_of();
            const bool far = top > FAR || (top < -FAR && top > NEG_INF && c_old < C_SEEN);
            if (!__any_sync(0xffffffffu, far)) break;
            const float m_old = m;
            if (far) m += top;
            c_old = fmaxf(c_old - (m - m_old), C_NONE);
          }
        }
        const float c_low = fmaxf(c_old - lower, C_NONE);
        const float c_new = top > c_low + C_SLACK ? floorf(top) - C_BELOW : c_low, f = ex2(c_old - c_new);
        if (since != 0 || g != 1.0f) move_sums(f * g);
        l *= f;
        l_over *= f;
        c_run = c_new;
        limit = m != 0.0f || c_new < C_SEEN ? NEG_INF : c_new + C_SLACK;
      }
      since++;
      float sum = 0.0f;
      uint32_t t[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float p = ex2(z[j] - c_run);
        sum += p;
        const uint32_t w = __float2uint_rz(fmaf(p, vs[j], (j & 1) ? 0.9999f - dither : dither));
        t[j] = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 4), sel);   // digits (3, 3, 1, 1) or (2, 2, 0, 0) of two neighbouring tokens
      }
      dither += dither < 0.3819f ? GOLDEN : GOLDEN - 1.0f;      // within -0.0001 .. 0.9999, so that a weight of zero stays zero
      const float add = fmaf(sum, P_UNIT, -l_over), l_new = l + add;
      l_over = (l_new - l) - add;                               // what the sum is above the true one
      l = l_new;
      const uint32_t p0 = __byte_perm(t[0], t[1], 0x5410), p1 = __byte_perm(t[0], t[1], 0x7632);
      const uint32_t p2 = __byte_perm(t[2], t[3], 0x5410), p3 = __byte_perm(t[2], t[3], 0x7632);

      // ---- sums of weight * code: tokens 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4 of either run are four neighbouring k
      uint32_t y[8][W];
#pragma unroll
      for (int c = 0; c < 8; c++) {
        const uint32_t to = here + (c >> 2) * C::GRAN;
        if (D == 128) {
          const uint4 x = lds128(v_src + to + (c & 1) * 128 + ((c >> 1) & 1) * 1024);
          y[c][0] = x.x; y[c][1] = x.y; y[c][W - 2] = x.z; y[c][W - 1] = x.w;
        } else {
          const uint2 x = lds64(((c & 1) ? v_src ^ 64u : v_src) + to + ((c >> 1) & 1) * 512);
          y[c][0] = x.x; y[c][1] = x.y;
        }
      }
#pragma unroll
      for (int w = 0; w < W; w++)
#pragma unroll
        for (int h = 0; h < 2; h++) {                           // two dimensions at a time: bytes (0, 1) and (2, 3) of a word
          const uint32_t s = h ? 0x7362 : 0x5140;
          const uint32_t u0 = __byte_perm(y[0][w], y[1][w], s), u1 = __byte_perm(y[2][w], y[3][w], s);
          const uint32_t u2 = __byte_perm(y[4][w], y[5][w], s), u3 = __byte_perm(y[6][w], y[7][w], s);
          imma_u8(acc[w * 4 + h * 2], p0, p1, p2, p3, __byte_perm(u0, u1, 0x5410), __byte_perm(u2, u3, 0x5410));
          imma_u8(acc[w * 4 + h * 2 + 1], p0, p1, p2, p3, __byte_perm(u0, u1, 0x7632), __byte_perm(u2, u3, 0x7632));
        }
    }
    move_sums(1.0f);

    // ---- the piece: outputs (2 t4 + odd) * CH .. + CH - 1 of row r in units of 2^(m + c_run + kappa), the sum of p in units of 2^(m + c_run)
    l -= l_over;
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    float4 row = make_float4(c_run, l, kf == 0.0f ? -200.0f : (float)(127 - (__float_as_int(kf) >> 23)), m);   // kappa -200: no scale was seen
    float val[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const float got = __shfl_xor_sync(0xffffffffu, odd ? o[i][0] : o[i][1], 4);
      val[i] = (odd ? o[i][1] : o[i][0]) + got;
    }
    const int mine = r * D + (2 * t4 + odd) * CH;               // this thread's place in a slot: [row][D], then (c, l, kappa, m) of the rows
    bool last = true;
    if (tile0 != 0 || tile1 != it.tiles) {
      // other warps of the block that have pieces of the item
      const int64_t in0 = max(at - tile0 - run.begin, (int64_t)0), in1 = min(at - tile0 + it.tiles, run.end) - 1 - run.begin;
      const int warp0 = kv_run_of(parts, in0), warp1 = kv_run_of(parts, in1);
      // a piece that begins in the middle of its item has a slot of its own; one that goes on behind the warp's run is the run's
      // last, so the ring is free
      auto slot_of = [&](int w) -> float* {
        const bool starts = at - tile0 >= run.begin + kv_run_begin(parts, w);
        return reinterpret_cast<float*>(smem + (starts ? w * (ST * C::TILE) : C::RING + w * C::SLOT));
      };
      if (warp0 != warp1) {
        float* s = slot_of(warp);
        if (tile0 == 0) { cp_wait<0>(); __syncwarp(); }
#pragma unroll
        for (int i = 0; i < CH; i += 4) *reinterpret_cast<float4*>(s + mine + i) = make_float4(val[i], val[i + 1], val[i + 2], val[i + 3]);
        if (t4 == 0 && !odd) *reinterpret_cast<float4*>(s + ROWS * D + 4 * r) = row;
        __threadfence_block();
        __syncwarp();
        int before = 0;
        if (lane == 0) before = atomicAdd(arrived + warp0, 1);
        last = __shfl_sync(0xffffffffu, before, 0) == warp1 - warp0;
        if (last) {
          __threadfence_block();
          join_pieces<D>(warp0, warp1, slot_of, [](const float* x) { return *reinterpret_cast<const float4*>(x); }, r, mine, val, row);
        }
      }
      // the same between blocks, through memory
      const bool starts = at - tile0 >= run.begin;
      if (last && (!starts || at - tile0 + it.tiles > run.end)) {
        const int run0 = kv_run_of(run.all, at - tile0), run1 = kv_run_of(run.all, at - tile0 + it.tiles - 1);
        auto piece = [&](int c) { return a.slots + (int64_t)(2 * c + (c == run0 ? 1 : 0)) * KV_SLOT_FLOATS; };
        float* s = piece((int)blockIdx.x);
#pragma unroll
        for (int i = 0; i < CH; i += 4) __stcg(reinterpret_cast<float4*>(s + mine + i), make_float4(val[i], val[i + 1], val[i + 2], val[i + 3]));
        if (t4 == 0 && !odd) __stcg(reinterpret_cast<float4*>(s + ROWS * D + 4 * r), row);
        __threadfence();
        __syncwarp();
        uint32_t before = 0;
        if (lane == 0) before = atomicAdd(a.counters + run0, 1u);
        last = __shfl_sync(0xffffffffu, before, 0) == (uint32_t)(run1 - run0);
        if (last) {
          __threadfence();
          if (lane == 0) a.counters[run0] = 0;
          join_pieces<D>(run0, run1, piece, [](const float* x) { return __ldcg(reinterpret_cast<const float4*>(x)); }, r, mine, val, row);
        }
      }
    }
    if (last && r < rows_here) {
      const float up = pow2((int)fmaxf(row.z, -126.0f)), inv = row.y == 0.0f ? 0.0f : 1.0f / row.y;
      int t;
      float* dst = a.out + row_offset(a, it.b, it.head, it.rb * ROWS + r, a.ld_o, D, t) + (2 * t4 + odd) * CH;
#pragma unroll
      for (int i = 0; i < CH; i++) val[i] = val[i] * P_UNIT * inv * up;
#pragma unroll
      for (int i = 0; i < CH; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(val[i], val[i + 1], val[i + 2], val[i + 3]);
    }
    at += tile1 - tile0;
    left -= tile1 - tile0;
    tile = 0;
    if (left > 0 && ++it.head == a.g.heads) {
      it.head = 0; it.e++;
      it.load<ROWS>(a, row_blocks);
    }
  }
}

template <int D>
int launch_four(b200q_ctx* ctx, const AttnArgs& a) {
  constexpr uint32_t ready = 1u << (D == 64 ? 0 : 1);
  if (!(ctx->kv_ready & ready)) {
    B200Q_CHECK_CUDA(cudaFuncSetAttribute(kv_attention_four_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Four<D>::SMEM));
    ctx->kv_ready |= ready;
  }
  const int row_blocks = (int)(((int64_t)a.T * a.group + 3) / 4);
  return kv_launch(ctx, kv_attention_four_kernel<D>, dim3(ctx->sm_count), 32 * Four<D>::WARPS, Four<D>::SMEM, a, row_blocks);
}

}  // namespace

int kv_workspace(b200q_ctx* ctx) {
  if (ctx->ws_kv.ptr) return 0;
  const size_t bytes = kv_counter_bytes(ctx) + kv_item_bytes(ctx) + (size_t)ctx->sm_count * 2 * KV_SLOT_FLOATS * sizeof(float);
  if (int e = ws_reserve(ctx, ctx->ws_kv, bytes)) return e;
  B200Q_CHECK_CUDA(cudaMemsetAsync(ctx->ws_kv.ptr, 0, kv_counter_bytes(ctx), ctx->stream));
  return 0;
}

int launch_kv_attention(b200q_ctx* ctx, const b200q_kv_cache& c, const KvBatch& s, const float* q, int64_t ld_q, int H, const uint64_t* tree,
                        float scale, float* out, int64_t ld_o) {
  ProfScope prof(ctx, KK_KV_ATTENTION);
  const AttnArgs a{KvGeom{c.pages, s.max_pages, c.page_shift, c.heads}, c.k, c.v, c.ks, c.vs, s.page_table, s.start, s.count, tree, q, out,
                   ld_q, ld_o, s.B, s.T, H, H / c.heads, scale * 1.4426950408889634f, ctx->status_dev, (uint32_t*)ctx->ws_kv.ptr,
                   (float*)((uint8_t*)ctx->ws_kv.ptr + kv_counter_bytes(ctx) + kv_item_bytes(ctx)), (int4*)((uint8_t*)ctx->ws_kv.ptr + kv_counter_bytes(ctx))};
  // Query rows per cache head.  Measured on both sides of the border, 8 cache heads, 16 sequences of up to 3000 tokens, here and
  // there: 24 rows 39 and 56 us (head dimension 64), 59 and 78 us (128); 36 rows 53 and 58, 83 and 84; 40 rows 59 and 58, 89 and
  // 84; 64 rows 87 and 60, 137 and 96.  (With 4 sequences of up to 600 tokens both take 12 to 33 us, here the fewer.)
  if ((int64_t)s.T * a.group > 36) return launch_kv_attention_many(ctx, a, c.head_dim);
  return c.head_dim == 64 ? launch_four<64>(ctx, a) : launch_four<128>(ctx, a);
}

}  // namespace b200q

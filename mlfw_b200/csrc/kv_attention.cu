// Attention over the int8 key/value cache for few query rows (decoding steps), and the choice of the kernel by rows.
// What is computed and in which arithmetic stands in kv_attention.cuh.
#include "kv_attention.cuh"

namespace b200q {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// Few rows (a decoding step: 1 .. 16 query rows share a cache head).  Bound by reading the cache: 2 (D + 4) bytes per token
// and head.  Warp-level binary16 products (m16n8k16): the sixteen rows of the A operand are eight query rows' hi and the
// same rows' lo parts, so one instruction does both parts and a thread finds the two sums of its score in its own
// accumulators.  B operands come straight from rows of codes: a lane's 16 bytes of a key row are four k-steps (which head
// dimensions make up a k-step is free as long as q follows), and of V a lane takes the same 16 dimensions of four tokens.
//
// Each warp works on 16-token tiles of its own through a ring of its own in shared memory (cp.async, no block-wide
// barrier inside a piece); eight warps of a block join their results at the end of a piece.
// ---------------------------------------------------------------------------------------------------------------
constexpr int FEW_WARPS = 8;
template <int D>
struct Few {
  static constexpr int STAGES = D == 128 ? 3 : 6;              // about 100 KB of ring per block: two blocks per SM
  static constexpr int TILE = 2 * KV_TILE * D + 2 * KV_TILE * 4;   // K and V codes, K and V scales
  static constexpr int RING = FEW_WARPS * STAGES * TILE;
  static constexpr int Q_BYTES(int rg) { return rg * (D / 16) * 512; }
};
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

// The end of a piece: the block's warps are added up, to the result when the piece is the whole item, else to the block's slot,
// and the last piece of an item to arrive joins all of them in the order of the runs.  join_o holds outputs relative to the
// largest of the warps' c.
template <int D, int ROWS, int WARPS>
__device__ __forceinline__ void finish_piece(const AttnArgs& a, const Run& run, int b, int rb, int head, int rows_here, int tile0, int tile1, int tiles,
                                             int64_t at, const float (&join_c)[WARPS][ROWS], const float (&join_l)[WARPS][ROWS], const float* join_o,
                                             uint32_t* arrived) {
  const int tid = threadIdx.x;
  const bool whole = tile0 == 0 && tile1 == tiles;
  const int64_t item0 = at - tile0;                           // first tile of the item among all tiles
  const int run0 = whole ? 0 : kv_run_of(run.all, item0), run1 = whole ? 0 : kv_run_of(run.all, item0 + tiles - 1);
  float* mine = a.slots + (int64_t)(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * KV_SLOT_FLOATS;
  for (int x = tid; x < ROWS * D; x += 32 * WARPS) {
    const int row = x / D, d = x % D;
    float top = join_c[0][row], sum = 0.0f, val = 0.0f;
#pragma unroll
    for (int w = 1; w < WARPS; w++) top = fmaxf(top, join_c[w][row]);
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      sum = fmaf(join_l[w][row], ex2(join_c[w][row] - top), sum);
      val += join_o[(w * ROWS + row) * D + d];
    }
    if (!whole) {
      __stcg(mine + row * D + d, val);
      if (d == 0) { __stcg(mine + ROWS * D + row, top); __stcg(mine + ROWS * D + ROWS + row, sum); }
    } else if (row < rows_here) {
      int t;
      a.out[row_offset(a, b, head, rb * ROWS + row, a.ld_o, D, t) + d] = sum == 0.0f ? 0.0f : val / sum * P_UNIT;
    }
  }
  // ---- the last piece of an item to arrive joins all of them, in the order of the runs
  if (!whole) {
    __threadfence();
    __syncthreads();
    if (tid == 0) *arrived = atomicAdd(a.counters + run0, 1u);
    __syncthreads();
    if (*arrived == (uint32_t)(run1 - run0)) {
      __threadfence();
      if (tid == 0) a.counters[run0] = 0;
      for (int x = tid; x < rows_here * D; x += 32 * WARPS) {
        const int row = x / D, d = x % D;
        auto piece = [&](int c) { return a.slots + (int64_t)(2 * c + (c == run0 ? 1 : 0)) * KV_SLOT_FLOATS; };
        float top = C_NONE, sum = 0.0f, val = 0.0f;
        for (int c = run0; c <= run1; c++) top = fmaxf(top, __ldcg(piece(c) + ROWS * D + row));
        for (int c = run0; c <= run1; c++) {
          const float* p = piece(c);
          const float f = ex2(__ldcg(p + ROWS * D + row) - top);
          sum = fmaf(__ldcg(p + ROWS * D + ROWS + row), f, sum);
          val = fmaf(__ldcg(p + row * D + d), f, val);
        }
        int t;
        a.out[row_offset(a, b, head, rb * ROWS + row, a.ld_o, D, t) + d] = sum == 0.0f ? 0.0f : val / sum * P_UNIT;
      }
    }
  }
}

// RG groups of eight query rows.
template <int D, int RG>
__global__ void __launch_bounds__(32 * FEW_WARPS, 2) kv_attention_few_kernel(const AttnArgs a, int row_blocks) {
  using C = Few<D>;
  constexpr int ROWS = 8 * RG, NT = D / 8, KS = D / 16, CH = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float join_c[FEW_WARPS][ROWS], join_l[FEW_WARPS][ROWS];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * (C::STAGES * C::TILE), q_smem = smem_u32(smem) + C::RING;
  float* join_o = reinterpret_cast<float*>(smem);               // [warp][row][D], over the rings between pieces

  // Places of a lane's pieces in a slot.  Of the swizzle only a flip of 64 bytes depends on more than the lane: pieces 32 lanes
  // apart are 512 bytes apart (V, D = 128: every second one flipped), tokens eight apart half a tile of rows apart.
  const uint32_t k_dst = ring + k_at<D>(lane / (D / 16), lane % (D / 16)), v_dst = ring + KV_TILE * D + v_at<D>(lane / (D / 16), lane % (D / 16));
  const uint32_t k_src = ring + k_at<D>(g8, t4);
  const uint32_t v_src = ring + KV_TILE * D + (D == 128 ? v_at<D>(2 * t4, g8) : v_at<D>(2 * t4, g8 >> 1) + (g8 & 1) * 8);
  const uint32_t q_src = q_smem + lane * 16;

  kv_after_previous();
  const Run run = find_run<ROWS, KV_TILE, FEW_WARPS>(a, row_blocks);
  int64_t left = run.end - run.begin;
  int e = run.e, head = run.head, tile0 = run.tile;
  int64_t at = run.begin;                                       // first tile of the piece among all tiles

  while (left > 0) {
    const int b = e / row_blocks, rb = e - b * row_blocks;
    const int64_t first = a.start[b];
    const int n = kv_rows_in_use(a.count, b, a.T);
    const int tiles = kv_tiles(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr, KV_TILE);
    if (tiles == 0) { e++; head = 0; tile0 = 0; continue; }
    const int64_t vis = kv_visible(a.g, first, n, a.group, ROWS, rb, a.tree != nullptr);
    const int tile1 = (int)min((int64_t)tiles, tile0 + left);
    const int rows_here = min(ROWS, n * a.group - rb * ROWS);
    if (tid == 0 && (first < 0 || first + n > (a.g.max_pages << a.g.page_shift))) atomicOr(a.status, STATUS_BAD_INDEX);

    // ---- the ring: tile i of the item into slot s
    const int32_t* table = a.page_table + (int64_t)b * a.g.max_pages;
    const int per_page = a.g.page_shift - 4;                    // log2 tiles per page
    const int in_table = (int)min((int64_t)tile1, a.g.max_pages << per_page);
    auto page_of = [&](int i) -> int { return i < in_table ? __ldg(table + (i >> per_page)) : -1; };
    auto fetch = [&](int i, int page, int s) {
      if ((uint32_t)page < (uint32_t)a.g.pages) {               // -1 behind the piece's end
        const int64_t row = (((int64_t)page * a.g.heads + head) << a.g.page_shift) + ((i & ((1 << per_page) - 1)) << 4);
        const uint32_t slot_at = s * C::TILE;
        const int64_t off = row * D + lane * 16;
        const int8_t *kp = a.k + off, *vp = a.v + off;
#pragma unroll
        for (int x = 0; x < D / 32; x++) cp16(k_dst + slot_at + x * 512, kp + x * 512);
#pragma unroll
        for (int x = 0; x < D / 32; x++) cp16(((D == 128 && (x & 1)) ? v_dst ^ 64u : v_dst) + slot_at + x * 512, vp + x * 512);
        if (lane < 8) cp16(ring + 2 * KV_TILE * D + lane * 16 + slot_at, (lane < 4 ? a.ks : a.vs) + row + (lane & 3) * 4);
      }
      cp_commit();
    };
    int page_q[C::STAGES];                                      // pages of the tiles in the ring
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; s++) page_q[s] = page_of(tile0 + warp + s * FEW_WARPS);
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; s++) fetch(tile0 + warp + s * FEW_WARPS, page_q[s], s);
    int page_next = page_of(tile0 + warp + (C::STAGES - 1) * FEW_WARPS);

    // ---- the query rows: this lane's row of every group, dimensions 64 m + 16 t4 + 0..15
    float row_scale[RG];
    int row_t[RG];
    uint64_t row_seen[RG];
#pragma unroll
    for (int r = 0; r < RG; r++) {
      const int R = rb * ROWS + r * 8 + g8;
      const bool used = r * 8 + g8 < rows_here;
      int t = 0;
      const float* src = a.q + row_offset(a, b, head, used ? R : rb * ROWS, a.ld_q, D, t);
      row_t[r] = used ? t : -1;
      row_seen[r] = used && a.tree ? a.tree[(int64_t)b * a.T + t] : 0;
      float4 x[KS];
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; s++) {
        x[s] = used ? __ldg(reinterpret_cast<const float4*>(src + (s >> 2) * 64 + t4 * 16 + (s & 3) * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max(max(top, max(__float_as_uint(x[s].x) & 0x7fffffffu, __float_as_uint(x[s].y) & 0x7fffffffu)),
                  max(__float_as_uint(x[s].z) & 0x7fffffffu, __float_as_uint(x[s].w) & 0x7fffffffu));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool finite = top < 0x7f800000u;
      const int ex = max((int)(top >> 23), 24) - 127;           // exponent of the row's largest element; tiny rows keep fewer bits
      const float up = pow2(10 - ex);                           // -117 .. 113
      row_scale[r] = finite ? a.scale_log2e * pow2(ex - 10) : __int_as_float(0x7fc00000);   // a NaN or an infinity in the row: every score NaN
      if (warp == 0) {
#pragma unroll
        for (int s = 0; s < KS; s++) {
          float h0, h1, h2, h3, l0, l1, l2, l3;
          const float4 y = finite ? x[s] : make_float4(0.f, 0.f, 0.f, 0.f);
          split_whole(y.x * up, h0, l0); split_whole(y.y * up, h1, l1); split_whole(y.z * up, h2, l2); split_whole(y.w * up, h3, l3);
          // k-step s of the key row's word: its even bytes are k = 2 t4, 2 t4 + 1, the odd ones k + 8
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(q_smem + (r * KS + s) * 512 + lane * 16), "r"(pack_f16(h0, h2)),
                         "r"(pack_f16(l0, l2)), "r"(pack_f16(h1, h3)), "r"(pack_f16(l1, l3)) : "memory");
        }
      }
    }
    __syncthreads();

    float o[RG][NT][2], c_run[RG], l[RG];
#pragma unroll
    for (int r = 0; r < RG; r++) {
      c_run[r] = C_NONE; l[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < NT; i++) o[r][i][0] = o[r][i][1] = 0.0f;
    }

    int slot = 0;
#pragma unroll 1
    for (int i = tile0 + warp; i < tile1; i += FEW_WARPS) {
      cp_wait<C::STAGES - 2>();
      __syncwarp();
      const int page = page_q[0];
#pragma unroll
      for (int s = 0; s + 2 < C::STAGES; s++) page_q[s] = page_q[s + 1];
      page_q[C::STAGES - 2] = page_next;
      fetch(i + (C::STAGES - 1) * FEW_WARPS, page_next, slot == 0 ? C::STAGES - 1 : slot - 1);
      page_next = page_of(i + C::STAGES * FEW_WARPS);
      const uint32_t slot_at = slot * C::TILE, sc = ring + 2 * KV_TILE * D + slot_at;
      slot = slot + 1 == C::STAGES ? 0 : slot + 1;
      if ((uint32_t)page >= (uint32_t)a.g.pages) {              // no such page: nothing of the tile is visible
        if (lane == 0 && (int64_t)i * KV_TILE < vis) atomicOr(a.status, STATUS_BAD_INDEX);
        continue;
      }

      // ---- scores: two blocks of eight tokens
      constexpr int CHAINS = RG == 1 ? D / 64 : 1;              // independent sums, to be added (exactly) at the end
      float acc[RG][2 * CHAINS][4];
#pragma unroll
      for (int mm = 0; mm < D / 64; mm++) {
        const uint32_t at_k = (mm ? k_src ^ 64u : k_src) + slot_at;
        const uint4 x0 = lds128(at_k), x1 = lds128(at_k + 8 * D);
        const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const uint32_t b00 = codes_even(w0[w]), b01 = codes_odd(w0[w]), b10 = codes_even(w1[w]), b11 = codes_odd(w1[w]);
#pragma unroll
          for (int r = 0; r < RG; r++) {
            const uint4 qa = lds128(q_src + (r * KS + mm * 4 + w) * 512);
            const int j = CHAINS == 2 ? 2 * mm : 0;
            if (w == 0 && (mm == 0 || CHAINS == 2)) {
              mma16816_first(acc[r][j], qa, b00, b01);
              mma16816_first(acc[r][j + 1], qa, b10, b11);
            } else {
              mma16816(acc[r][j], qa, b00, b01);
              mma16816(acc[r][j + 1], qa, b10, b11);
            }
          }
        }
      }
      const float2 ks0 = lds_f2(sc + t4 * 8), ks1 = lds_f2(sc + 32 + t4 * 8);
      float2 vs0 = lds_f2(sc + 64 + t4 * 8), vs1 = lds_f2(sc + 96 + t4 * 8);
      const int64_t pos = (int64_t)i * KV_TILE;
      const bool edge = pos + KV_TILE > first;                  // some position of the tile is among the new rows or behind them
      if (edge) {                                               // behind the last row in use anything may stand
        const int64_t end = min(vis, first + n);
        vs0.x = pos + t4 * 2 < end ? vs0.x : 0.0f; vs0.y = pos + t4 * 2 + 1 < end ? vs0.y : 0.0f;
        vs1.x = pos + 8 + t4 * 2 < end ? vs1.x : 0.0f; vs1.y = pos + 8 + t4 * 2 + 1 < end ? vs1.y : 0.0f;
      }
      const float lv0 = log2_scale(vs0.x), lv1 = log2_scale(vs0.y), lv2 = log2_scale(vs1.x), lv3 = log2_scale(vs1.y);
      uint4 pa[RG];
      float fold[RG];
#pragma unroll
      for (int r = 0; r < RG; r++) {
        if (CHAINS == 2) {
#pragma unroll
          for (int c = 0; c < 8; c++) acc[r][c >> 2][c & 3] += acc[r][2 * CHAINS - 2 + (c >> 2)][c & 3];
        }
        float z[4];
        z[0] = (acc[r][0][0] + acc[r][0][2]) * (ks0.x * row_scale[r]);
        z[1] = (acc[r][0][1] + acc[r][0][3]) * (ks0.y * row_scale[r]);
        z[2] = (acc[r][1][0] + acc[r][1][2]) * (ks1.x * row_scale[r]);
        z[3] = (acc[r][1][1] + acc[r][1][3]) * (ks1.y * row_scale[r]);
        if (edge) {
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int64_t j = pos + (c >> 1) * 8 + t4 * 2 + (c & 1) - first;
            const bool seen = first + j < vis && (j < 0 || (j < n && (a.tree ? (row_seen[r] >> j) & 1 : j <= row_t[r])));
            if (!seen) z[c] = NEG_INF;
          }
        }
        float top = fmaxf(fmaxf(z[0] + lv0, z[1] + lv1), fmaxf(z[2] + lv2, z[3] + lv3));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float c_new = fmaxf(c_run[r], top - 10.0f);
        fold[r] = ex2(c_run[r] - c_new);
        c_run[r] = c_new;
        const float p0 = ex2(z[0] - c_new), p1 = ex2(z[1] - c_new), p2 = ex2(z[2] - c_new), p3 = ex2(z[3] - c_new);
        l[r] = fmaf(l[r], fold[r], ((p0 + p1) + (p2 + p3)) * P_UNIT);
        float h0, h1, h2, h3, l0, l1, l2, l3;
        split_whole(p0 * vs0.x, h0, l0); split_whole(p1 * vs0.y, h1, l1); split_whole(p2 * vs1.x, h2, l2); split_whole(p3 * vs1.y, h3, l3);
        pa[r] = make_uint4(pack_f16(h0, h1), pack_f16(l0, l1), pack_f16(h2, h3), pack_f16(l2, l3));
      }

      // ---- o = o * fold + P V: dimension CH * g8 + d of the 16 tokens
      {
        uint32_t y[4][D / 32];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          if (D == 128) {
            const uint4 w = lds128(v_src + slot_at + (c & 1) * 128 + (c >> 1) * 1024);
            y[c][0] = w.x; y[c][1] = w.y; y[c][D / 32 - 2] = w.z; y[c][D / 32 - 1] = w.w;
          } else {
            const uint2 w = lds64(((c & 1) ? v_src ^ 64u : v_src) + slot_at + (c >> 1) * 512);
            y[c][0] = w.x; y[c][1] = w.y;
          }
        }
#pragma unroll
        for (int w = 0; w < D / 32; w++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t lo = __byte_perm(y[0][w], y[1][w], h ? 0x7632 : 0x5410), hi = __byte_perm(y[2][w], y[3][w], h ? 0x7632 : 0x5410);
#pragma unroll
            for (int odd = 0; odd < 2; odd++) {
              const int d = w * 4 + h * 2 + odd;
              const uint32_t b0 = odd ? codes_odd(lo) : codes_even(lo), b1 = odd ? codes_odd(hi) : codes_even(hi);
#pragma unroll
              for (int r = 0; r < RG; r++) {
                float c[4];
                mma16816_first(c, pa[r], b0, b1);
                o[r][d][0] = fmaf(o[r][d][0], fold[r], c[0] + c[2]);
                o[r][d][1] = fmaf(o[r][d][1], fold[r], c[1] + c[3]);
              }
            }
          }
      }
    }
    cp_wait<0>();

    // ---- the eight warps' results of the piece
#pragma unroll
    for (int r = 0; r < RG; r++) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t4 == 0) { join_c[warp][r * 8 + g8] = c_run[r]; join_l[warp][r * 8 + g8] = l[r]; }
    }
    __syncthreads();                                            // every ring is drained
#pragma unroll
    for (int r = 0; r < RG; r++) {
      const int row = r * 8 + g8;
      float top = join_c[0][row];
#pragma unroll
      for (int w = 1; w < FEW_WARPS; w++) top = fmaxf(top, join_c[w][row]);
      const float f = ex2(c_run[r] - top);
      float* dst = join_o + (warp * ROWS + row) * D + t4 * 2 * CH;
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int i = 0; i < CH; i += 4)
          *reinterpret_cast<float4*>(dst + c * CH + i) = make_float4(o[r][i][c] * f, o[r][i + 1][c] * f, o[r][i + 2][c] * f, o[r][i + 3][c] * f);
    }
    __syncthreads();
    finish_piece<D, ROWS, FEW_WARPS>(a, run, b, rb, head, rows_here, tile0, tile1, tiles, at, join_c, join_l, join_o, &arrived);
    __syncthreads();                                            // the rings are about to be filled again
    at += tile1 - tile0;
    left -= tile1 - tile0;
    tile0 = 0;
    if (++head == a.g.heads) { head = 0; e++; }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Up to four rows (decoding with up to four query heads per cache head), on the integer tensor cores: m16n8k32 with the
// codes as they are, so that K needs no conversion and V a transpose of bytes.  A query row and a row of weights are 32-bit
// fixed-point numbers in four 8-bit digits, and the sixteen rows of the A operand are four rows times four digits: of row r
// the rows 2 r and 2 r + 1 hold the digits 3 and 2, the rows 8 + 2 r and 9 + 2 r the digits 1 and 0.  A thread of an even
// row therefore finds sum d3 code and sum d1 code, its neighbour in the odd row those of d2 and d0; each takes one of their two
// columns after one exchange, so no score is computed twice.  Sums are 32-bit integers and exact: scores carry the rounding of
// adding the digits, and the outputs are added up without rounding until a row's c changes (or 2^15 tokens have passed), when
// they are converted, scaled and moved to binary32.  c = top - 26 leaves 5.5 bits before a larger weight (below 2^32) moves it.
// Scales of V are taken relative to the power of two of the first tile's largest (kappa), so that tiny values keep their digits.
//
// About 310 instructions per warp and 32 tokens of 128 dimensions, where the binary16 form above takes 1300: bound by
// reading the cache.  Twelve warps (D = 128: 64 integer sums, 32 outputs per thread) or sixteen (D = 64), one block per SM.
// ---------------------------------------------------------------------------------------------------------------
constexpr int IT = 32;                                          // tokens of a tile: two runs of sixteen, each in one page
template <int D>
struct Four {
  static constexpr int WARPS = D == 128 ? 12 : 16, STAGES = D == 128 ? 2 : 3;
  static constexpr int GRAN = 2 * KV_TILE * D + 2 * KV_TILE * 4, TILE = 2 * GRAN;   // sixteen tokens: K and V codes, K and V scales
  static constexpr int RING = WARPS * STAGES * TILE, SLOT = 4 * (D + 2) * 4, SMEM = RING + WARPS * SLOT;
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

// Every warp has a run of its own, a part of the block's, and a ring that it keeps full across the items of its run; the warps
// never wait for one another.  Results of an item that several warps of the block worked on are joined by the last of them
// through shared memory, and those of an item that several blocks worked on by the last warp of the last block.
template <int D>
__global__ void __launch_bounds__(32 * Four<D>::WARPS, 1) kv_attention_four_kernel(const AttnArgs a, int row_blocks) {
  using C = Four<D>;
  constexpr int ROWS = 4, WARPS = C::WARPS, ST = C::STAGES, KS = D / 32, CH = D / 8, W = D / 32;
  constexpr float C_BELOW = 26.0f, C_SLACK = 31.5f;
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
  const Run run = find_run<ROWS, IT, WARPS>(a, row_blocks);     // (its barriers publish `arrived`)
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

  // ---- the ring: tiles in the order of the run, ST - 1 ahead of their use.  `ahead` walks by itself; page0 and page1 are the
  // pages of its next tile's two runs of sixteen tokens, -1 where nothing is visible.
  Item ahead = it;
  int ahead_tile = tile, ahead_left = left, page0, page1;
  uint32_t there = 0;                                           // two bits per tile in the ring, the oldest lowest
  auto pages = [&]() {
    const int64_t pos = (int64_t)ahead_tile * IT;
    const int32_t* table = a.page_table + (int64_t)ahead.b * a.g.max_pages;
    page0 = ahead_left > 0 && pos < ahead.vis ? __ldg(table + (pos >> a.g.page_shift)) : -1;
    page1 = ahead_left > 0 && pos + 16 < ahead.vis ? __ldg(table + ((pos + 16) >> a.g.page_shift)) : -1;
  };
  auto fetch = [&](int s, int place) {
    if (ahead_left > 0) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int page = h ? page1 : page0;
        if ((uint32_t)page < (uint32_t)a.g.pages) {
          const int64_t row = (((int64_t)page * a.g.heads + ahead.head) << a.g.page_shift) + ((ahead_tile * IT + h * 16) & ((1 << a.g.page_shift) - 1));
          const uint32_t to = s * C::TILE + h * C::GRAN;
          const int8_t *kp = a.k + row * D + lane * 16, *vp = a.v + row * D + lane * 16;
#pragma unroll
          for (int x = 0; x < D / 32; x++) cp16(k_dst + to + x * 512, kp + x * 512);
#pragma unroll
          for (int x = 0; x < D / 32; x++) cp16(((D == 128 && (x & 1)) ? v_dst ^ 64u : v_dst) + to + x * 512, vp + x * 512);
          if (lane < 8) cp16(ring + 2 * KV_TILE * D + lane * 16 + to, (lane < 4 ? a.ks : a.vs) + row + (lane & 3) * 4);
          there |= (1u + h) << (2 * place);
        }
      }
      ahead_left--;
      if (++ahead_tile == ahead.tiles) {
        ahead_tile = 0;
        if (++ahead.head == a.g.heads) {
          ahead.head = 0; ahead.e++;
          if (ahead_left > 0) ahead.load<ROWS>(a, row_blocks);
        }
      }
      pages();
    }
    cp_commit();
  };
  pages();
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
        x[s] = used ? __ldg(reinterpret_cast<const float4*>(src + (s >> 2) * 64 + t4 * 16 + (s & 3) * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
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
    float o[CH][2], c_run = C_NONE, l = 0.0f, kf = 0.0f;        // kf: 2^-kappa, 0 until a tile has a scale
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
      if (kf == 0.0f) {                                         // kappa: the power of two of the first scales
        float big = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
        if (big > 0.0f) kf = pow2(127 - min(max(__float_as_int(big) >> 23, 1), 253));
      }
      float top = NEG_INF;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        vs[j] *= kf;
        top = fmaxf(top, z[j] + fmaxf(log2_raw(vs[j]), -88.0f));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      const bool grow = top > c_run + C_SLACK;
      if (__any_sync(0xffffffffu, grow) || since == 1024) {
        const float c_new = grow ? top - C_BELOW : c_run, f = ex2(c_run - c_new);
        move_sums(f);
        l *= f;
        c_run = c_new;
      }
      since++;
      float sum = 0.0f;
      uint32_t t[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float p = ex2(z[j] - c_run);
        sum += p;
        const uint32_t w = __float2uint_rn(p * vs[j]);
        t[j] = __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 4), sel);   // digits (3, 3, 1, 1) or (2, 2, 0, 0) of two neighbouring tokens
      }
      l = fmaf(sum, P_UNIT, l);
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

    // ---- the piece: outputs (2 t4 + odd) * CH .. + CH - 1 of row r, relative to c_run; 2^-40 as the sums of p, before 2^kappa:
    // huge values of V times weights of 2^31 would leave binary32
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    l *= 0x1p-40f;
    const float kappa = kf == 0.0f ? 1.0f : pow2(127 - (__float_as_int(kf) >> 23));
    float val[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const float got = __shfl_xor_sync(0xffffffffu, odd ? o[i][0] : o[i][1], 4);
      val[i] = ((odd ? o[i][1] : o[i][0]) + got) * 0x1p-40f * kappa;
    }
    const int mine = r * D + (2 * t4 + odd) * CH;               // this thread's place in a slot: [row][D], then c and l of the rows
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
        if (t4 == 0 && !odd) { s[ROWS * D + r] = c_run; s[ROWS * D + ROWS + r] = l; }
        __threadfence_block();
        __syncwarp();
        int before = 0;
        if (lane == 0) before = atomicAdd(arrived + warp0, 1);
        last = __shfl_sync(0xffffffffu, before, 0) == warp1 - warp0;
        if (last) {
          __threadfence_block();
          float top = C_NONE, sum = 0.0f;
          for (int w = warp0; w <= warp1; w++) top = fmaxf(top, slot_of(w)[ROWS * D + r]);
#pragma unroll
          for (int i = 0; i < CH; i++) val[i] = 0.0f;
          for (int w = warp0; w <= warp1; w++) {
            const float* x = slot_of(w);
            const float f = ex2(x[ROWS * D + r] - top);
            sum = fmaf(x[ROWS * D + ROWS + r], f, sum);
#pragma unroll
            for (int i = 0; i < CH; i += 4) {
              const float4 y = *reinterpret_cast<const float4*>(x + mine + i);
              val[i] = fmaf(y.x, f, val[i]); val[i + 1] = fmaf(y.y, f, val[i + 1]); val[i + 2] = fmaf(y.z, f, val[i + 2]); val[i + 3] = fmaf(y.w, f, val[i + 3]);
            }
          }
          c_run = top; l = sum;
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
        if (t4 == 0 && !odd) { __stcg(s + ROWS * D + r, c_run); __stcg(s + ROWS * D + ROWS + r, l); }
        __threadfence();
        __syncwarp();
        uint32_t before = 0;
        if (lane == 0) before = atomicAdd(a.counters + run0, 1u);
        last = __shfl_sync(0xffffffffu, before, 0) == (uint32_t)(run1 - run0);
        if (last) {
          __threadfence();
          if (lane == 0) a.counters[run0] = 0;
          float top = C_NONE, sum = 0.0f;
          for (int c = run0; c <= run1; c++) top = fmaxf(top, __ldcg(piece(c) + ROWS * D + r));
#pragma unroll
          for (int i = 0; i < CH; i++) val[i] = 0.0f;
#pragma unroll 2
          for (int c = run0; c <= run1; c++) {
            const float* x = piece(c);
            const float f = ex2(__ldcg(x + ROWS * D + r) - top);
            sum = fmaf(__ldcg(x + ROWS * D + ROWS + r), f, sum);
#pragma unroll
            for (int i = 0; i < CH; i += 4) {
              const float4 y = __ldcg(reinterpret_cast<const float4*>(x + mine + i));
              val[i] = fmaf(y.x, f, val[i]); val[i + 1] = fmaf(y.y, f, val[i + 1]); val[i + 2] = fmaf(y.z, f, val[i + 2]); val[i + 3] = fmaf(y.w, f, val[i + 3]);
            }
          }
          l = sum;
        }
      }
    }
    if (last && r < rows_here) {
      const float inv = l == 0.0f ? 0.0f : P_UNIT;
      int t;
      float* dst = a.out + row_offset(a, it.b, it.head, it.rb * ROWS + r, a.ld_o, D, t) + (2 * t4 + odd) * CH;
#pragma unroll
      for (int i = 0; i < CH; i += 4) {
        const float d = l == 0.0f ? 1.0f : l;
        *reinterpret_cast<float4*>(dst + i) = make_float4(val[i] / d * inv, val[i + 1] / d * inv, val[i + 2] / d * inv, val[i + 3] / d * inv);
      }
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

template <int D, int RG>
int launch_few(b200q_ctx* ctx, const AttnArgs& a) {
  const int smem = Few<D>::RING + Few<D>::Q_BYTES(RG);
  constexpr uint32_t ready = 1u << ((D == 64 ? 0 : 2) + RG - 1);
  if (!(ctx->kv_ready & ready)) {
    B200Q_CHECK_CUDA(cudaFuncSetAttribute(kv_attention_few_kernel<D, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    ctx->kv_ready |= ready;
  }
  const int row_blocks = (int)(((int64_t)a.T * a.group + 8 * RG - 1) / (8 * RG));
  return kv_launch(ctx, kv_attention_few_kernel<D, RG>, dim3(ctx->sm_count * KV_BLOCKS_PER_SM), 32 * FEW_WARPS, smem, a, row_blocks);
}

template <int D>
int launch_four(b200q_ctx* ctx, const AttnArgs& a) {
  constexpr uint32_t ready = 1u << (D == 64 ? 12 : 13);
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
  const size_t bytes = kv_counter_bytes(ctx) + kv_item_bytes(ctx) + (size_t)ctx->sm_count * KV_BLOCKS_PER_SM * 2 * KV_SLOT_FLOATS * sizeof(float);
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
  const int64_t rows = (int64_t)s.T * a.group;
  int e;
  if (rows <= 4) return c.head_dim == 64 ? launch_four<64>(ctx, a) : launch_four<128>(ctx, a);
  // Measured on both sides of the border: 16 rows (12 heads of 64, 32 sequences of up to 1000 tokens) 61 us here and 88 us
  // there with everything around it; 124 rows (head dimension 128, 8 sequences of up to 5000 tokens) 209 and 129 us.
  if (rows > 16) return launch_kv_attention_many(ctx, a, c.head_dim);
  if (c.head_dim == 64) e = rows <= 8 ? launch_few<64, 1>(ctx, a) : launch_few<64, 2>(ctx, a);
  else e = rows <= 8 ? launch_few<128, 1>(ctx, a) : launch_few<128, 2>(ctx, a);
  return e;
}

}  // namespace b200q

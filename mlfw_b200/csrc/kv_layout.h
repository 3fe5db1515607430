// Where a token lives in the key/value cache, and which calls on it are refused.  Plain C++ as well as device code, so
// that both are checked on the host without a GPU (tests/test_kv_layout.py).
//
// A cache is `pages` pages of 2^page_shift tokens.  Codes: int8 [page][head][token][head_dim]; scales: f32
// [page][head][token].  K and V have arrays of their own with the same layout.  Position `pos` of sequence b is token
// pos mod 2^page_shift of page page_table[b * max_pages + pos / 2^page_shift]: a page may hold tokens of one
// sequence only as far as writing goes, and may appear in the tables of several sequences as far as reading goes (a shared
// prefix).
#pragma once
#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define B200Q_HD __host__ __device__ __forceinline__
#else
#define B200Q_HD inline
#endif

namespace b200q {

constexpr int KV_MAX_TREE = 64;   // drafted tokens a 64-bit row of ancestors can name; also the rows b200q_kv_keep moves at most

struct KvGeom {
  int64_t pages;
  int64_t max_pages;   // entries of a sequence in the page table
  int page_shift;
  int heads;
};

// Row (token of a head; code offset = row * head_dim) of a position, -1 when the position lies outside the page table or
// its page outside the cache.  Rows are 64-bit: a cache may hold more than 2^31 bytes.
B200Q_HD int64_t kv_row(const KvGeom& g, const int32_t* page_table, int64_t b, int head, int64_t pos) {
  if (pos < 0) return -1;
  const int64_t slot = pos >> g.page_shift;
  if (slot >= g.max_pages) return -1;
  const int64_t page = page_table[b * g.max_pages + slot];
  if (page < 0 || page >= g.pages) return -1;
  return (((page * g.heads + head) << g.page_shift) | (pos & ((int64_t(1) << g.page_shift) - 1)));
}

// New rows of sequence b that are in use: count[b] held to 0..T, T without a count.
B200Q_HD int kv_rows_in_use(const int32_t* count, int64_t b, int T) {
  if (count == nullptr) return T;
  const int c = count[b];
  return c < 0 ? 0 : (c > T ? T : c);
}

// The warp a thread belongs to, counted over a grid of blocks of whole warps: up to 2^31 - 1, where threads no longer fit 32 bits.
B200Q_HD uint32_t kv_warp(uint32_t block, uint32_t threads, uint32_t thread) { return block * (threads / 32) + thread / 32; }

// ---------------------------------------------------------------------------------------------- work of the attention
// An item is one block of `rows` query rows (row R = t * group + query head within the group) of one sequence and one cache head; its
// work is the 16-token tiles of the positions any of its rows sees.  All items' tiles, in the order (sequence, row block,
// head, tile), are cut into equal runs, one per block of the grid.  An item that spans several runs is joined from its pieces.
constexpr int KV_TILE = 16;

// Positions visible to row block rb of a sequence with `n` rows in use: [0, result).
B200Q_HD int64_t kv_visible(const KvGeom& g, int64_t start, int n, int group, int rows, int rb, bool tree) {
  const uint32_t last = (uint32_t)(rb + 1) * (uint32_t)rows - 1;           // last row of the block (rows of a sequence are below 2^31)
  const int64_t t = last / (uint32_t)group + 1;                           // new tokens its rows reach without a tree
  const int64_t vis = start + (tree || t > n ? n : t), most = g.max_pages << g.page_shift;
  return vis < 0 ? 0 : (vis > most ? most : vis);
}
// Tiles of that block: none when it has no row in use, else at least one (a block that sees nothing still writes zeros).
B200Q_HD int kv_tiles(const KvGeom& g, int64_t start, int n, int group, int rows, int rb, bool tree, int tile) {
  if ((int64_t)rb * rows >= (int64_t)n * group) return 0;
  const int64_t vis = kv_visible(g, start, n, group, rows, rb, tree);
  return vis <= tile ? 1 : (int)((vis + tile - 1) / tile);
}
B200Q_HD int64_t kv_div(int64_t a, int64_t b) {   // a >= 0, b > 0: in 32 bits where that does (a 64-bit division is a subroutine)
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// `total` > 0 tiles cut into at most `grid` runs of at least `least` tiles (of all there are, when that is fewer): the first
// `rem` runs hold base + 1, the others base.
struct KvRuns {
  int64_t total, base;
  int runs, rem;
};
B200Q_HD KvRuns kv_runs(int64_t total, int least, int grid) {
  const int64_t want = total / least;
  KvRuns r;
  r.total = total;
  r.runs = want < 1 ? 1 : (want < grid ? (int)want : grid);
  r.base = kv_div(total, r.runs);
  r.rem = (int)(total - r.base * r.runs);
  return r;
}
// The first tile of a run, and the run that holds a tile.
B200Q_HD int64_t kv_run_begin(const KvRuns& r, int c) { return r.base * c + (c < r.rem ? c : r.rem); }
B200Q_HD int kv_run_of(const KvRuns& r, int64_t tile) {
  const int64_t cut = (r.base + 1) * r.rem;
  return tile < cut ? (int)kv_div(tile, r.base + 1) : r.rem + (int)kv_div(tile - cut, r.base);
}

// ---------------------------------------------------------------------------------------------- refusals (host)
// Each returns null when the call is in order, else the reason.
inline const char* kv_refuse_geometry(int64_t pages, int64_t page_tokens, int64_t heads, int64_t head_dim) {
  if (pages < 1 || pages > INT32_MAX) return "the number of pages must be between 1 and 2^31 - 1";
  if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1))) return "a page holds 16, 32, 64, 128 or 256 tokens";
  if (heads < 1 || heads > 65535) return "the number of heads must be between 1 and 65535";
  if (head_dim != 64 && head_dim != 128) return "the head dimension must be 64 or 128";
  if (pages > (int64_t(1) << 46) / (page_tokens * heads * head_dim)) return "the cache is larger than 2^46 codes";
  return nullptr;
}
inline bool kv_aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr const char* kv_misaligned = "an array of integers does not start on a multiple of its element's size";

// B sequences of T rows; `what` holds back the pointer checks when there is nothing to do.
inline const char* kv_refuse_batch(int64_t B, int64_t T, int64_t heads, const void* page_table, int64_t max_pages, const void* start) {
  if (B < 0 || T < 0 || max_pages < 0) return "negative dimension";
  if (B > INT32_MAX || T > (1 << 24) || B * T > INT32_MAX / heads) return "batch * rows * heads must stay below 2^31 and rows at most 2^24";
  if (max_pages > INT32_MAX) return "the page table is too wide";
  if (B * T == 0) return nullptr;
  if (start == nullptr || (page_table == nullptr && max_pages > 0)) return "null pointer";
  if (!kv_aligned(page_table, 4) || !kv_aligned(start, 4)) return kv_misaligned;
  return nullptr;
}
// Optional arrays of `element` bytes each: count, tree, keep.
inline const char* kv_refuse_array(const void* p, size_t element) { return kv_aligned(p, element) ? nullptr : kv_misaligned; }
// An f32 operand whose row (b, t) of head h starts at base + (b * T + t) * ld + h * head_dim.
inline const char* kv_refuse_rows(const void* base, int64_t ld, int64_t heads, int64_t head_dim) {
  if (base == nullptr) return "null pointer";
  if (!kv_aligned(base, 16) || ld % 4 != 0) return "rows must start on 16-byte boundaries (base address, and row stride a multiple of 4)";
  if (ld < heads * head_dim) return "the row stride is below heads * head_dim";
  return nullptr;
}

}  // namespace b200q

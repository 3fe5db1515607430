"""Host checks of the key/value cache's index rules and refusals (mlfw_b200/csrc/kv_layout.h), the very functions the kernels
and the C entry points call, compiled with g++; and of the entry points' refusals that need no GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include <vector>
#include "kv_layout.h"
using namespace b200q;
extern "C" {
int64_t row(int64_t pages, int64_t max_pages, int shift, int heads, const int32_t* table, int64_t b, int head, int64_t pos) {
  return kv_row(KvGeom{pages, max_pages, shift, heads}, table, b, head, pos);
}
int64_t visible(int64_t mp, int shift, int64_t start, int n, int group, int rows, int rb, int tree) { return kv_visible(KvGeom{1, mp, shift, 1}, start, n, group, rows, rb, tree); }
int tiles(int64_t mp, int shift, int64_t start, int n, int group, int rows, int rb, int tree, int tile) { return kv_tiles(KvGeom{1, mp, shift, 1}, start, n, group, rows, rb, tree, tile); }
int in_use(const int32_t* count, int64_t b, int T) { return kv_rows_in_use(count, b, T); }
const char* geometry(int64_t p, int64_t t, int64_t h, int64_t d) { return kv_refuse_geometry(p, t, h, d); }
const char* batch(int64_t B, int64_t T, int64_t h, const void* table, int64_t mp, const void* start) { return kv_refuse_batch(B, T, h, table, mp, start); }
// The walk of the attention kernels over a batch, block by block as the device does it: every (item, tile) an owner, every slot of the
// join written once, every item's pieces as many as its last one expects.  Returns 0, or which of these fails.
int walk(int B, int T, int heads, int group, int rows, int warps, int grid, int64_t max_pages, int shift, const int32_t* start, const int32_t* count,
         int tree, int tile_tokens, int64_t* total_out) {
  const KvGeom g{1, max_pages, shift, heads};
  const int rbs = (int)(((int64_t)T * group + rows - 1) / rows);
  std::vector<int64_t> begin;                      // first tile of (e, head)
  std::vector<int> tiles;
  int64_t total = 0;
  for (int e = 0; e < B * rbs; e++) {
    const int n = kv_tiles(g, start[e / rbs], kv_rows_in_use(count, e / rbs, T), group, rows, e % rbs, tree, tile_tokens);
    for (int h = 0; h < heads; h++) { begin.push_back(total); tiles.push_back(n); total += n; }
  }
  *total_out = total;
  if (total == 0) return 0;
  const KvRuns all = kv_runs(total, warps, grid);
  const int runs = all.runs;
  std::vector<int> slot(2 * grid, 0), pieces(begin.size(), 0), expected(begin.size(), 0), counter(grid, -1);
  size_t item = 0;
  int64_t covered = 0;
  for (int c = 0; c < runs; c++) {
    int64_t at = kv_run_begin(all, c), end = kv_run_begin(all, c + 1);
    if (at != covered || end <= at) return 1;
    covered = end;
    while (at < end) {
      while (tiles[item] == 0 || begin[item] + tiles[item] <= at) item++;
      const int64_t t0 = at - begin[item], t1 = tiles[item] < t0 + end - at ? tiles[item] : t0 + end - at;
      if (t0 < 0 || t1 <= t0) return 2;
      if (!(t0 == 0 && t1 == tiles[item])) {
        const int64_t r0 = kv_run_of(all, begin[item]), r1 = kv_run_of(all, begin[item] + tiles[item] - 1);
        if (r0 > c || r1 < c || r0 < 0 || r1 >= runs || (t0 == 0) != (r0 == c)) return 3;
        if (slot[2 * c + (t0 == 0 ? 1 : 0)]++) return 4;
        if (counter[r0] >= 0 && counter[r0] != (int)item) return 5;
        counter[r0] = (int)item;
        pieces[item]++;
        expected[item] = (int)(r1 - r0 + 1);
      }
      at += t1 - t0;
    }
  }
  if (covered != total) return 6;
  for (size_t i = 0; i < begin.size(); i++)
    if (pieces[i] != expected[i]) return 7;
  return 0;
}
uint32_t warp(uint32_t block, uint32_t threads, uint32_t thread) { return kv_warp(block, threads, thread); }
const char* array(const void* p, int64_t element) { return kv_refuse_array(p, (size_t)element); }
const char* rows(const void* base, int64_t ld, int64_t h, int64_t d) { return kv_refuse_rows(base, ld, h, d); }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv")
    (d / "h.cpp").write_text(SOURCE)
    so = str(d / "h.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "mlfw_b200", "csrc"), str(d / "h.cpp"), "-o", so],
                   check=True)
    lib = C.CDLL(so)
    i64, vp = C.c_int64, C.c_void_p
    lib.row.restype, lib.row.argtypes = i64, [i64, i64, C.c_int, C.c_int, vp, i64, C.c_int, i64]
    lib.warp.restype, lib.warp.argtypes = C.c_uint32, [C.c_uint32] * 3
    lib.in_use.argtypes = [vp, i64, C.c_int]
    lib.walk.argtypes = [C.c_int] * 7 + [i64, C.c_int, vp, vp, C.c_int, C.c_int, C.POINTER(i64)]
    lib.visible.restype, lib.visible.argtypes = i64, [i64, C.c_int, i64] + [C.c_int] * 5
    lib.tiles.argtypes = [i64, C.c_int, i64] + [C.c_int] * 6
    for f, a in (("geometry", [i64] * 4), ("array", [vp, i64]), ("batch", [i64, i64, i64, vp, i64, vp]), ("rows", [vp, i64, i64, i64])):
        getattr(lib, f).restype, getattr(lib, f).argtypes = C.c_char_p, a
    return lib


def test_rows_of_positions(host):
    rng = np.random.default_rng(0)
    for shift, heads, pages, per in ((4, 1, 9, 3), (6, 12, 40, 5), (8, 3, 7, 2)):
        P = 1 << shift
        table = np.ascontiguousarray(rng.permutation(pages)[: 2 * per].reshape(2, per) if 2 * per <= pages else rng.integers(0, pages, (2, per)), np.int32)
        for b in range(2):
            for pos in range(per * P):
                for head in {0, heads - 1}:
                    want = (int(table[b, pos // P]) * heads + head) * P + pos % P
                    assert host.row(pages, per, shift, heads, table.ctypes.data, b, head, pos) == want


def test_positions_outside_have_no_row(host):
    table = np.array([[0, -1, 5, 4]], np.int32)     # a cache of five pages: -1 and 5 are not among them
    row = lambda pos: host.row(5, 4, 4, 2, table.ctypes.data, 0, 1, pos)  # noqa: E731
    assert [row(p) for p in (-1, -17, 16, 31, 32, 47, 64, 1 << 40)] == [-1] * 8
    assert row(15) == 16 + 15 and row(48) == (4 * 2 + 1) * 16 and row(63) == (4 * 2 + 1) * 16 + 15
    big = np.array([[2**31 - 2]], np.int32)          # rows past 2^31 and codes past 2^38
    assert host.row(2**31 - 1, 1, 8, 64, big.ctypes.data, 0, 63, 255) == ((2**31 - 2) * 64 + 63) * 256 + 255


def test_rows_in_use(host):
    c = np.array([-3, 0, 2, 9], np.int32)
    assert [host.in_use(c.ctypes.data, b, 4) for b in range(4)] == [0, 0, 2, 4] and host.in_use(None, 7, 4) == 4


def test_the_runs_cover_every_tile_once(host):
    rng = np.random.default_rng(5)
    total = C.c_int64()
    seen = 0
    for _ in range(3000):
        B, T, heads, group = (int(rng.integers(1, m)) for m in (9, 70, 5, 9))
        rows, warps, grid = int(rng.choice([8, 16, 128])), int(rng.choice([1, 8])), int(rng.choice([1, 7, 148, 296]))
        shift, tile = int(rng.integers(4, 9)), int(rng.choice([16, 64]))
        most = int(rng.choice([1, 40, 3000]))
        max_pages = -(-(most + T) // (1 << shift)) if rng.random() < 0.9 else int(rng.integers(0, 3))
        start = rng.integers(0, most + 1, B).astype(np.int32)
        if rng.random() < 0.1:
            start[rng.integers(0, B)] = rng.choice([-5, -(2**31), 2**31 - 1])
        count = rng.integers(-1, T + 2, B).astype(np.int32)
        code = host.walk(B, T, heads, group, rows, warps, grid, max_pages, shift, start.ctypes.data, count.ctypes.data if rng.random() < 0.8 else None,
                         int(T <= 64 and rng.random() < 0.5), tile, C.byref(total))
        assert code == 0, (code, B, T, heads, group, rows, warps, grid, max_pages, shift, start, count)
        seen += total.value > 8 * grid
    assert seen > 100


def test_visible_positions(host):
    """kv_visible against the rule, row by row: the largest position any row of a block sees."""
    rng = np.random.default_rng(6)
    for _ in range(500):
        T, group, rows = (int(rng.integers(1, m)) for m in (50, 9, 33))
        start, n, tree = int(rng.integers(0, 100)), 0, bool(rng.integers(0, 2))
        n = int(rng.integers(1, T + 1))
        for rb in range(-(-n * group // rows)):
            used = range(rb * rows, min((rb + 1) * rows, n * group))
            want = start + (n if tree else max(R // group for R in used) + 1)
            assert host.visible(64, 4, start, n, group, rows, rb, tree) == want
            assert host.tiles(64, 4, start, n, group, rows, rb, tree, 16) == -(-want // 16)
        past = -(-n * group // rows)
        assert host.tiles(64, 4, start, n, group, rows, past, tree, 16) == 0
    assert host.visible(2, 4, 100, 3, 1, 8, 0, False) == 32 and host.visible(2, 4, -100, 3, 1, 8, 0, False) == 0
    assert host.tiles(2, 4, -100, 3, 1, 8, 0, False, 16) == 1 and host.tiles(0, 4, 0, 3, 1, 8, 0, True, 16) == 1


def test_warps_of_a_large_grid(host):
    """A batch of nearly 2^31 rows has as many warps: more threads than 32 bits count."""
    for block, thread in ((0, 0), (3, 255), (1 << 24, 0), ((1 << 28) - 1, 255)):
        assert host.warp(block, 256, thread) == (block * 256 + thread) // 32


def test_refusals(host):
    assert host.geometry(1, 16, 1, 64) is None and host.geometry(1000, 256, 65535, 128) is None
    for bad in ((0, 64, 1, 64), (-1, 64, 1, 64), (2**31, 64, 1, 64), (4, 8, 1, 64), (4, 48, 1, 64), (4, 512, 1, 64), (4, 0, 1, 64), (4, 64, 0, 64),
                (4, 64, 65536, 64), (4, 64, 2, 32), (4, 64, 2, 96), (2**31 - 1, 256, 65535, 128)):
        assert host.geometry(*bad), bad
    p = 4096
    assert host.batch(3, 5, 8, p, 7, p) is None and host.batch(0, 5, 8, None, 0, None) is None and host.batch(3, 5, 8, None, 0, p) is None
    for bad in ((-1, 5, 8, p, 7, p), (3, -5, 8, p, 7, p), (3, 5, 8, p, -7, p), (3, 5, 8, None, 7, p), (3, 5, 8, p, 7, None), (2**16, 2**15, 1, p, 7, p),
                (2**62, 2**62, 1, p, 7, p), (1, 2**25, 1, p, 7, p), (1, 1, 1, p, 2**31, p)):
        assert host.batch(*bad), bad
    assert host.rows(p, 128, 2, 64) is None and host.rows(p, 400, 3, 128) is None
    for bad in ((None, 128, 2, 64), (p + 4, 128, 2, 64), (p, 130, 2, 64), (p, 124, 2, 64), (p, -128, 2, 64)):
        assert host.rows(*bad), bad


def test_refusals_of_integer_arrays(host):
    """An address that is no multiple of the element's size would fault on the GPU."""
    assert host.array(None, 8) is None and host.array(4096, 8) is None and host.array(4100, 4) is None
    assert b"multiple of its element" in host.array(4100, 8) and host.array(4098, 4)
    for table, start in ((4098, 4096), (4096, 4097)):
        assert b"multiple of its element" in host.batch(3, 5, 8, table, 7, start)
    assert host.batch(0, 5, 8, 4098, 7, 4097) is None


def test_entry_points_refuse_without_a_gpu():
    from mlfw_b200 import _lib
    from mlfw_b200 import build
    build.build()
    lib = _lib.lib()
    message = lambda: lib.b200q_last_error().decode()  # noqa: E731
    out = C.c_void_p(1)
    assert lib.b200q_kv_create(None, 4, 48, 2, 64, 4096, 4096, 4096, 4096, C.byref(out)) != 0 and "a page holds" in message() and out.value is None
    assert lib.b200q_kv_create(None, 4, 64, 2, 64, 4096, None, 4096, 4096, C.byref(out)) != 0 and "null pointer" in message()
    assert lib.b200q_kv_create(None, 4, 64, 2, 64, 4096, 4100, 4096, 4096, C.byref(out)) != 0 and "16-byte" in message()
    assert lib.b200q_kv_create(None, 4, 64, 2, 64, 4096, 4096, 4096, 4096, C.byref(out)) != 0 and "null context" in message()
    assert lib.b200q_kv_create(None, 4, 64, 2, 64, 4096, 4096, 4096, 4096, None) != 0 and "out pointer" in message()
    assert lib.b200q_kv_destroy(None, None) == 0
    for name, n in (("append", 12), ("read", 12), ("attention", 15), ("keep", 9)):
        args = [None if t is C.c_void_p else t(0) for t in _lib.PROTOTYPES["b200q_kv_" + name][1]]
        assert len(args) == n
        assert getattr(lib, "b200q_kv_" + name)(*args) != 0 and "null context" in message()

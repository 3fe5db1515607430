"""GPU parity of the int8 key/value cache and the attention that reads it.

What the cache holds is exact: codes and scales are those of the per-token quantization (CPU oracle) of every head's
row, reading back is one binary32 product, keeping moves bytes; whole buffers are compared, so that a write beside the
new rows shows.  Attention is compared with the formula in binary64 over the cache's contents, row by row, within the bound
derived in :func:`attention_bound`.
"""
import numpy as np
import pytest

from gpu_util import Guarded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mlfw_b200
    c = mlfw_b200.Context(0)
    yield c
    c.check_status()
    c.close()


class Setup:
    """A cache whose buffers start as garbage (codes -128, scales NaN), a shuffled page table, and their host copies."""

    def __init__(self, ctx, B, most, page, heads, dim, seed=0, spare=2):
        import mlfw_b200
        self.ctx, self.B, self.page, self.heads, self.dim = ctx, B, page, heads, dim
        self.rng = np.random.default_rng([seed, B, most, page, heads, dim])
        self.per = -(-most // page)
        self.pages = B * self.per + spare
        shape = (self.pages, heads, page)
        self.codes = [np.full(shape + (dim,), -128, np.int8) for _ in range(2)]
        self.scales = [np.full(shape, np.nan, np.float32) for _ in range(2)]
        self.bufs = [Guarded(ctx, a.shape, a.dtype, a) for a in self.codes + self.scales]
        self.cache = mlfw_b200.KVCache(ctx, self.pages, page, heads, dim, buffers=tuple(b.ptr for b in self.bufs))
        self.table = self.rng.permutation(self.pages)[: B * self.per].reshape(B, self.per).astype(np.int32)
        self.dtable = ctx.to_device(self.table)

    def dev(self, a, dtype=np.int32):
        return None if a is None else self.ctx.to_device(np.ascontiguousarray(a, dtype))

    def fill(self, tokens):
        """Random contents for positions < tokens[b], on both sides."""
        for b, n in enumerate(tokens):
            for pos in range(int(n)):
                p, r = self.table[b, pos // self.page], pos % self.page
                for i in range(2):
                    c = np.clip(np.round(self.rng.standard_normal((self.heads, self.dim)) * 42), -127, 127)
                    self.codes[i][p, :, r] = c
                    self.scales[i][p, :, r] = self.rng.uniform(0.01, 0.03, self.heads)
        self.upload()

    def upload(self):
        for b, a in zip(self.bufs, self.codes + self.scales):
            b.upload(a)

    def append(self, orc, k, v, start, count):
        """The expected buffers after an append of k, v [B, T, heads, dim]."""
        for b in range(self.B):
            for t in range(int(count[b])):
                pos = int(start[b]) + t
                p, r = self.table[b, pos // self.page], pos % self.page
                for i, x in enumerate((k, v)):
                    q, _, s = orc.quantize_per_token(np.ascontiguousarray(x[b, t]))
                    self.codes[i][p, :, r], self.scales[i][p, :, r] = q, s

    def check(self):
        for b, want in zip(self.bufs, self.codes + self.scales):
            got = b.download()
            assert (got.view(np.uint8) == want.view(np.uint8)).all(), "the cache differs from what it must hold"

    def tokens(self, b, n):
        """K, V codes and scales of positions < n: [n, heads, dim] and [n, heads]."""
        pos = np.arange(n)
        p, r = self.table[b, pos // self.page], pos % self.page
        return [a[p, :, r] for a in self.codes + self.scales]


def attention_bound(q, kc, ks, vc, vs, scale, see):
    """|result - binary64 result| for one query row and head, with u = 2^-24 (binary32 half step).

    A score: q held to 2^-23 of its largest element (a fixed-point form of 23 bits and sign; binary32 products are
    closer) gives scale * ks * sum|c| * qmax * 2^-23; combining, scaling and changing to base 2 are at most eight
    roundings of |z| or of the partial sums scale * ks * sum |q c|, of which D additions in binary32 order may each add u:
    (D + 8) u scale ks sum|q c|.  So |dz| <= E below, a weight exp(z - max) is off by a factor e^(2E) times the exponential's
    2^-21, the weights' fixed-point form by 2^-22 of the largest weight, and the sums over n tokens, taken over tiles
    in binary32, by (n/16 + 64) u; numerator and denominator both, over |v| <= vmax.
    """
    n = int(see.sum())
    if n == 0:
        return 0.0
    a = np.abs(kc[see].astype(np.float64))
    E = abs(scale) * np.max(ks[see] * (a.sum(1) * np.abs(q).max() * 2.0**-23 + (q.size + 8) * 2.0**-24 * (a @ np.abs(q))))
    vmax = np.max(vs[see, None] * np.abs(vc[see].astype(np.float64)))
    return 2 * vmax * (np.expm1(2 * E) + 2.0**-21 + 2.0**-22 * np.sqrt(n) + (n / 16 + 64) * 2.0**-24)


def attention_rows(S, q, start, count, tree, scale):
    """Formula in binary64 and its bound: [B, T, H, dim] and [B, T, H]."""
    B, T, H, D = q.shape
    want, bound = np.zeros((B, T, H, D)), np.zeros((B, T, H))
    for b in range(B):
        n = int(start[b]) + int(count[b])
        kc, vc, ks, vs = S.tokens(b, n)
        j = np.arange(n) - int(start[b])
        for t in range(int(count[b])):
            see = (j < 0) | ((j <= t) if tree is None else ((tree[b, t] >> np.clip(j, 0, 63).astype(np.uint64)) & np.uint64(1)).astype(bool))
            for h in range(H):
                g = h // (H // S.heads)
                x = q[b, t, h].astype(np.float64)
                if see.any():
                    z = scale * ks[see, g].astype(np.float64) * (kc[see, g].astype(np.float64) @ x)
                    w = np.exp(z - z.max())
                    want[b, t, h] = (w * vs[see, g]) @ vc[see, g].astype(np.float64) / w.sum()
                bound[b, t, h] = attention_bound(x, kc[:, g], ks[:, g], vc[:, g], vs[:, g], scale, see)
    return want, bound


def random_tree(rng, B, T):
    tree = np.zeros((B, T), np.uint64)
    for b in range(B):
        for t in range(T):
            parent = rng.integers(-1, t) if t else -1
            tree[b, t] = (tree[b, parent] if parent >= 0 else np.uint64(0)) | np.uint64(1 << t)
    return tree


def run_attention(S, q, start, count, tree, scale, ld_pad=0):
    B, T, H, D = q.shape
    ld = H * D + ld_pad
    rows = np.full((B * T, ld), np.nan, np.float32)
    rows[:, : H * D] = q.reshape(B * T, H * D)
    mark = np.float32(-77.25)
    out = Guarded(S.ctx, (B * T, ld), np.float32, np.full((B * T, ld), mark, np.float32))
    S.cache.attention(S.ctx.to_device(rows), ld, B, T, H, S.dtable, S.per, S.dev(start), S.dev(count), S.dev(tree, np.uint64), scale, out.ptr, ld)
    S.ctx.sync()
    got = out.download()
    assert (got[:, H * D:] == mark).all(), "written beside the rows"
    got = got[:, : H * D].reshape(B, T, H, D)
    for b in range(B):
        used = T if count is None else int(count[b])
        assert (got[b, used:] == mark).all(), "a row behind the last one in use was written"
    return got


def check_attention(S, q, start, count, tree, scale, **kw):
    B, T = q.shape[:2]
    got = run_attention(S, q, start, count, tree, scale, **kw)
    n = np.full(B, T) if count is None else count
    want, bound = attention_rows(S, q, start, n, tree, scale)
    for b in range(B):
        c = int(n[b])
        err = np.abs(got[b, :c] - want[b, :c]).max(-1)
        assert (err <= bound[b, :c]).all(), f"sequence {b}: off by {np.max(err - bound[b, :c])} over a bound of {bound[b, :c].min()}"
    return got


# ------------------------------------------------------------------------------------------------ write, read, keep
@pytest.mark.parametrize("B,T,heads,dim,page,start,count", [
    (1, 1, 1, 64, 16, [0], None), (3, 1, 12, 64, 64, [0, 63, 64], None), (2, 37, 5, 128, 16, [3, 14], [37, 20]),
    (4, 9, 8, 64, 32, [0, 31, 5, 7], [9, 0, 1, 40]), (1, 300, 2, 128, 256, [1], None)])
def test_append_and_read(ctx, orc, B, T, heads, dim, page, start, count):
    S = Setup(ctx, B, max(start) + T, page, heads, dim)
    n = np.full(B, T) if count is None else np.minimum(count, T)
    ld = (heads * 3 + 1) * dim
    rows = S.rng.standard_normal((B * T, ld)).astype(np.float32) * 3
    d = ctx.to_device(rows)
    S.cache.append(d.ptr + 4 * dim, d.ptr + 4 * 2 * heads * dim, ld, ld, B, T, S.dtable, S.per, S.dev(start), S.dev(count))
    ctx.sync()
    k = rows[:, dim:(heads + 1) * dim].reshape(B, T, heads, dim)
    v = rows[:, 2 * heads * dim:3 * heads * dim].reshape(B, T, heads, dim)
    S.append(orc, k, v, start, n)
    S.check()

    mark = np.full((B * T, heads * dim + 4), np.float32(5.5))
    outs = [Guarded(ctx, mark.shape, np.float32, mark) for _ in range(2)]
    S.cache.read(B, T, S.dtable, S.per, S.dev(start), S.dev(count), outs[0].ptr, outs[1].ptr, heads * dim + 4, heads * dim + 4)
    ctx.sync()
    for i, o in enumerate(outs):
        want = mark.copy().reshape(B, T, -1)
        for b in range(B):
            for t in range(int(n[b])):
                pos = int(start[b]) + t
                p, r = S.table[b, pos // page], pos % page
                want[b, t, : heads * dim] = (S.codes[i][p, :, r].astype(np.float32) * S.scales[i][p, :, r][:, None]).reshape(-1)
        assert (o.download().view(np.uint32) == want.reshape(mark.shape).view(np.uint32)).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_append_odd_rows(ctx, orc, dim):
    """Zeros, one value throughout, NaN, infinities, ties, the smallest and the largest magnitudes."""
    x = np.random.default_rng(dim).standard_normal((10, dim)).astype(np.float32)
    x[0] = 0
    x[1] = -2.5
    x[2, 3] = np.nan
    x[3] = np.nan
    x[4, 5], x[4, 9] = np.inf, -np.inf
    x[5] = (np.arange(dim) % 255 - 127).astype(np.float32) + np.float32(0.5)      # ties around absmax 126.5 / 127.5
    x[5, 0] = 127
    x[6] *= np.float32(1e-44)
    x[7] *= np.float32(3e38) / np.abs(x[7]).max()
    x[8] *= np.float32(1e-38)
    x[9, 0] = 1e30
    S = Setup(ctx, 1, 5, 16, 2, dim)
    v = x[::-1].copy()
    S.cache.append(ctx.to_device(x), ctx.to_device(v), 2 * dim, 2 * dim, 1, 5, S.dtable, S.per, S.dev([0]), None)
    ctx.sync()
    S.append(orc, x.reshape(1, 5, 2, dim), v.reshape(1, 5, 2, dim), [0], [5])
    S.check()


@pytest.mark.parametrize("B,T,heads,dim,page", [(1, 1, 1, 64, 16), (3, 20, 5, 64, 16), (2, 64, 3, 128, 32)])
def test_keep(ctx, B, T, heads, dim, page):
    S = Setup(ctx, B, 30 + T, page, heads, dim)
    start = S.rng.integers(0, 30, B)
    S.fill(start + T)
    for case in ("path", "any order", "nothing"):
        keep = np.zeros((B, T), np.int64)
        kept = np.zeros(B, np.int64)
        for b in range(B):
            if case == "path":
                path = np.flatnonzero(S.rng.random(T) < 0.4)
                keep[b, : path.size], kept[b] = path, path.size
            elif case == "any order":
                keep[b], kept[b] = S.rng.integers(0, T, T), T
        S.cache.keep(B, T, S.dtable, S.per, S.dev(start), S.dev(keep), S.dev(kept))
        ctx.sync()
        for a in S.codes + S.scales:
            for b in range(B):
                src, dst = start[b] + keep[b, : kept[b]], start[b] + np.arange(kept[b])
                a[S.table[b, dst // page], :, dst % page] = a[S.table[b, src // page], :, src % page]
        S.check()


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("B,T,H,heads,dim,page,start,count", [
    (1, 1, 1, 1, 64, 16, [0], None),                       # one token, nothing cached
    (1, 1, 12, 12, 64, 64, [500], None),
    (3, 1, 8, 2, 128, 32, [1, 31, 333], [1, 0, 1]),        # shared heads, a sequence without a row
    (5, 1, 16, 1, 128, 16, [0, 15, 16, 17, 1000], None),   # 16 query heads on one cache head
    (2, 1, 24, 1, 64, 64, [63, 130], None),                # more than 16
    (2, 3, 6, 2, 64, 16, [0, 77], [3, 2]),
    (1, 17, 4, 4, 128, 64, [40], None),
    (2, 65, 2, 2, 64, 16, [0, 100], [65, 33]),             # chunks of a prompt
    (1, 150, 8, 2, 128, 128, [5], None),
    (1, 130, 3, 3, 64, 256, [0], None),
])
def test_attention(ctx, B, T, H, heads, dim, page, start, count):
    S = Setup(ctx, B, max(start) + T, page, heads, dim)
    n = np.full(B, T) if count is None else np.array(count)
    S.fill(np.array(start) + n)
    q = (S.rng.standard_normal((B, T, H, dim)) * 2).astype(np.float32)
    check_attention(S, q, start, count, None, dim ** -0.5, ld_pad=4 * (B - 1))


@pytest.mark.parametrize("B,T,H,heads,dim,page,start,count", [
    (1, 1, 2, 2, 64, 16, [33], None), (2, 8, 4, 4, 64, 16, [0, 300], [8, 5]), (2, 31, 8, 2, 128, 64, [50, 0], [31, 30]),
    (1, 64, 6, 3, 64, 32, [700], None), (2, 64, 8, 1, 128, 16, [1, 129], [64, 63])])
def test_attention_tree(ctx, B, T, H, heads, dim, page, start, count):
    S = Setup(ctx, B, max(start) + T, page, heads, dim)
    n = np.full(B, T) if count is None else np.array(count)
    S.fill(np.array(start) + n)
    q = (S.rng.standard_normal((B, T, H, dim)) * 2).astype(np.float32)
    tree = random_tree(S.rng, B, T)
    if T < 64:
        tree[:, T // 2] |= ~np.uint64(0) << np.uint64(T)             # bits beyond the rows in use name nothing
    check_attention(S, q, start, count, tree, dim ** -0.5)


def test_attention_rows_that_see_nothing(ctx):
    """Nothing cached and an empty row of ancestors: zeros; its neighbours are not disturbed."""
    S = Setup(ctx, 2, 20, 16, 2, 64)
    S.fill([6, 9])
    q = S.rng.standard_normal((2, 4, 2, 64)).astype(np.float32)
    tree = np.array([[0, 1, 0, 9], [0, 0, 0, 0]], np.uint64)
    got = check_attention(S, q, [0, 5], [4, 4], tree, 0.125)
    assert (got[0, [0, 2]] == 0).all() and (got[1] != 0).any()


def test_attention_sees_nothing_of_unwritten_rows(ctx):
    """Pages hold NaN scales and codes of -128 wherever nothing was written; lengths end inside pages and at their ends."""
    for dim in (64, 128):
        for n in (1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257):
            S = Setup(ctx, 1, 320, 64, 2, dim, seed=n)
            S.fill([n])
            q = S.rng.standard_normal((1, 1, 4, dim)).astype(np.float32)
            check_attention(S, q, [n - 1], None, None, dim ** -0.5)


@pytest.mark.parametrize("T", [1, 20])
def test_attention_extreme_inputs(ctx, T):
    """Scores of hundreds, tiny and huge scales of K and V, a zero query, negative and zero scale."""
    S = Setup(ctx, 1, 200 + T, 32, 2, 64)
    S.fill([200 + T])
    q = (S.rng.standard_normal((1, T, 4, 64)) * 60).astype(np.float32)
    check_attention(S, q, [200], None, None, 0.125)
    q[0, 0, 1] = 0
    q[0, 0, 2] *= np.float32(1e-30)
    check_attention(S, q, [200], None, None, -0.125)
    check_attention(S, q, [200], None, None, 0.0)
    for i, f in ((2, 1e-30), (2, 1e30)):
        keep = [a.copy() for a in S.scales]
        S.scales[1][:, 0] *= np.float32(f)                       # V of one head far from that of the other
        S.scales[1][:, 1, ::3] *= np.float32(f) ** np.float32(0.25)
        S.upload()
        check_attention(S, q, [200], None, None, 0.125)
        S.scales[:] = keep
    S.scales[0] *= np.float32(1e-20)
    S.scales[1][:] = 0
    S.upload()
    assert (run_attention(S, q, [200], None, None, 0.125) == 0).all()


@pytest.mark.parametrize("T,heads", [(1, 2), (24, 2)])
def test_attention_nan_and_infinite_queries_stay_in_their_row(ctx, T, heads):
    S = Setup(ctx, 1, 100 + T, 16, heads, 128)
    S.fill([100 + T])
    q = S.rng.standard_normal((1, T, 4, 128)).astype(np.float32)
    clean = run_attention(S, q, [100], None, None, 0.1)
    q[0, T // 2, 0, 5], q[0, 0, 2, 7], q[0, 0, 3, 9] = np.nan, np.inf, -np.inf
    got = run_attention(S, q, [100], None, None, 0.1)
    bad = np.zeros((1, T, 4), bool)
    bad[0, T // 2, 0] = bad[0, 0, 2] = bad[0, 0, 3] = True
    assert np.isnan(got[bad]).all() and (got[~bad] == clean[~bad]).all()


def test_attention_is_the_same_every_time(ctx):
    """Split over the GPU and joined: no order of arrival changes a bit."""
    for B, T, H, heads, dim, n in ((2, 1, 8, 2, 128, 3001), (1, 16, 4, 4, 64, 900), (1, 64, 8, 2, 128, 1500)):
        S = Setup(ctx, B, n + T, 64, heads, dim)
        for i in range(2):
            S.codes[i] = S.rng.integers(-127, 128, S.codes[i].shape).astype(np.int8)
            S.scales[i] = S.rng.uniform(0.01, 0.02, S.scales[i].shape).astype(np.float32)
        S.upload()
        q = S.rng.standard_normal((B, T, H, dim)).astype(np.float32)
        first = run_attention(S, q, np.full(B, n), None, None, 0.1)
        for _ in range(5):
            assert (run_attention(S, q, np.full(B, n), None, None, 0.1).view(np.uint32) == first.view(np.uint32)).all()


@pytest.mark.parametrize("B,T,H,heads,dim,most", [(40, 1, 16, 16, 64, 420), (24, 1, 32, 8, 128, 900), (20, 3, 12, 4, 64, 700), (12, 9, 8, 8, 64, 900),
                                                  (6, 24, 16, 16, 64, 1500), (3, 40, 12, 12, 128, 1300), (3, 70, 24, 8, 128, 1100)])
def test_attention_long_runs(ctx, B, T, H, heads, dim, most):
    """Enough work that a block has many tiles of several items, of uneven lengths."""
    S = Setup(ctx, B, most + T, 64, heads, dim)
    start = S.rng.integers(0, most, B)
    start[0] = most
    for i in range(2):
        S.codes[i] = np.clip(np.round(S.rng.standard_normal(S.codes[i].shape) * 42), -127, 127).astype(np.int8)
        S.scales[i] = S.rng.uniform(0.01, 0.03, S.scales[i].shape).astype(np.float32)
    S.upload()
    q = (S.rng.standard_normal((B, T, H, dim)) * 2).astype(np.float32)
    check_attention(S, q, start, np.full(B, T), random_tree(S.rng, B, T) if T > 1 and T <= 64 else None, dim ** -0.5)


@pytest.mark.parametrize("B,T,H,heads,dim", [(3000, 1, 2, 1, 64), (700, 2, 3, 3, 128), (257, 17, 2, 1, 64)])
def test_attention_many_short_sequences(ctx, B, T, H, heads, dim):
    """More sequences than threads of a block, of no to three cached tokens, most of them padding."""
    S = Setup(ctx, B, 3 + T, 16, heads, dim)
    start = S.rng.integers(0, 4, B)
    count = np.where(S.rng.random(B) < 0.2, S.rng.integers(0, T + 1, B), 0)
    for i in range(2):
        S.codes[i] = np.clip(np.round(S.rng.standard_normal(S.codes[i].shape) * 42), -127, 127).astype(np.int8)
        S.scales[i] = S.rng.uniform(0.01, 0.03, S.scales[i].shape).astype(np.float32)
    S.upload()
    q = (S.rng.standard_normal((B, T, H, dim)) * 2).astype(np.float32)
    check_attention(S, q, start, count, None, dim ** -0.5)


@pytest.mark.parametrize("H,dim,page", [(33, 64, 16), (40, 128, 256), (64, 128, 16), (65, 64, 128), (130, 128, 32)])
def test_attention_many_heads_on_one(ctx, H, dim, page):
    """A decoding step whose query heads fill the rows of the kernels for chunks."""
    S = Setup(ctx, 2, 400, page, 1, dim)
    S.fill([40, 400])
    q = (S.rng.standard_normal((2, 1, H, dim)) * 2).astype(np.float32)
    check_attention(S, q, [39, 399], None, None, dim ** -0.5, ld_pad=8)


def test_positions_outside_the_cache(ctx):
    """A bad page or a position behind the table: the status bit, no write, zeros, not visible."""
    S = Setup(ctx, 2, 48, 16, 2, 64)
    S.fill([48, 48])
    S.table[0, 1], S.table[1, 2] = S.pages, -5
    S.dtable = S.dev(S.table)
    good = S.table.copy()
    x = S.rng.standard_normal((2 * 4, 2 * 64)).astype(np.float32)
    d = ctx.to_device(x)
    S.cache.append(d, d, 128, 128, 2, 4, S.dtable, S.per, S.dev([18, 46]), None)    # page 1 of the first; behind the table, and page 2, of the second
    ctx.sync()
    assert ctx.status_word() == 32
    ctx.clear_status()
    S.check()                                                                       # nothing was written
    outs = [Guarded(ctx, (8, 128), np.float32, np.ones((8, 128), np.float32)) for _ in range(2)]
    S.cache.read(2, 4, S.dtable, S.per, S.dev([14, -2]), None, outs[0].ptr, outs[1].ptr, 128, 128)
    ctx.sync()
    got = outs[0].download().reshape(2, 4, 128)
    assert ctx.status_word() == 32 and (got[0, 2:] == 0).all() and (got[1, :2] == 0).all() and (got[0, :2] != 0).any() and (got[1, 2:] != 0).any()
    ctx.clear_status()
    keep = np.array([[3, 1, 7, -1], [0, 1, 0, 0]])
    S.cache.keep(2, 4, S.dtable, S.per, S.dev([0, 30]), S.dev(keep), S.dev([4, 2]))   # 7 and -1 name no row; 32 is on the bad page
    ctx.sync()
    for a in S.codes + S.scales:
        a[good[0, 0], :, 0] = a[good[0, 0], :, 3]
    assert ctx.status_word() == 32
    ctx.clear_status()
    S.check()
    # attention over 48 positions of which one page is bad equals attention without that page's rows
    q = S.rng.standard_normal((2, 1, 2, 64)).astype(np.float32)
    got = run_attention(S, q, [47, 47], None, None, 0.125)
    assert ctx.status_word() == 32
    ctx.clear_status()
    for b, away in ((0, 1), (1, 2)):
        rows = np.array([p for p in range(48) if p // 16 != away])
        p, r = good[b, rows // 16], rows % 16
        kc, vc, ks, vs = (a[p, :, r] for a in S.codes + S.scales)
        for h in range(2):
            see = np.ones(32, bool)
            z = 0.125 * ks[:, h].astype(np.float64) * (kc[:, h].astype(np.float64) @ q[b, 0, h])
            w = np.exp(z - z.max())
            want = (w * vs[:, h]) @ vc[:, h].astype(np.float64) / w.sum()
            assert np.abs(got[b, 0, h] - want).max() <= attention_bound(q[b, 0, h].astype(np.float64), kc[:, h], ks[:, h], vc[:, h], vs[:, h], 0.125, see)


def test_shared_prefix_pages(ctx):
    """Two sequences read the same pages."""
    S = Setup(ctx, 2, 80, 16, 2, 64)
    S.table[1, :4] = S.table[0, :4]
    S.dtable = S.dev(S.table)
    S.fill([70, 0])
    S.fill([0, 0])
    q = S.rng.standard_normal((2, 1, 2, 64)).astype(np.float32)
    check_attention(S, q, [63, 40], None, None, 0.125)


def test_offsets_past_31_bits(ctx, orc):
    """Codes behind the first 2^31 bytes of a buffer are written, read, moved and attended to."""
    import mlfw_b200
    heads, dim, page = 8, 128, 256
    pages = (1 << 31) // (heads * dim * page) + 9
    cache = mlfw_b200.KVCache(ctx, pages, page, heads, dim)
    rng = np.random.default_rng(3)
    table = np.array([[pages - 1, pages - 3]], np.int32)
    T = 300
    x = rng.standard_normal((2, T, heads, dim)).astype(np.float32)
    dk, dv, dt, d0 = ctx.to_device(x[0]), ctx.to_device(x[1]), ctx.to_device(table), ctx.to_device(np.zeros(1, np.int32))
    cache.append(dk, dv, heads * dim, heads * dim, 1, T, dt, 2, d0, None)
    keep = np.zeros((1, 64), np.int32)
    keep[0] = np.arange(64)[::-1]
    d230 = ctx.to_device(np.array([230], np.int32))
    cache.keep(1, 64, dt, 2, d230, ctx.to_device(keep), None)
    outs = [ctx.empty((T, heads, dim), np.float32) for _ in range(2)]
    cache.read(1, T, dt, 2, d0, None, outs[0], outs[1], heads * dim, heads * dim)
    q = rng.standard_normal((1, 1, heads, dim)).astype(np.float32)
    o = ctx.empty((1, heads, dim), np.float32)
    cache.attention(ctx.to_device(q), heads * dim, 1, 1, heads, dt, 2, ctx.to_device(np.array([T - 1], np.int32)), None, None, 0.1, o, heads * dim)
    ctx.sync()
    order = np.arange(T)
    order[230:294] = order[230:294][::-1].copy()
    held = []
    for i in range(2):
        c, _, s = orc.quantize_per_token(x[i].reshape(-1, dim))
        held += [(c.reshape(T, heads, dim)[order], s.reshape(T, heads)[order])]
        want = held[i][0].astype(np.float32) * held[i][1][..., None]
        assert (outs[i].download().view(np.uint32) == want.view(np.uint32)).all()
    got = o.download()[0]
    for h in range(heads):
        (kc, ks), (vc, vs) = [(c[:, h], s[:, h]) for c, s in held]
        z = 0.1 * ks.astype(np.float64) * (kc.astype(np.float64) @ q[0, 0, h])
        w = np.exp(z - z.max())
        want = (w * vs) @ vc.astype(np.float64) / w.sum()
        assert np.abs(got[h] - want).max() <= attention_bound(q[0, 0, h].astype(np.float64), kc, ks, vc, vs, 0.1, np.ones(T, bool))
    cache.close()


def test_padded_batch_of_many_rows(ctx, orc):
    """Nine sequences of room for 2^24 rows, of which the last has three in use: more threads than 32 bits count, operands of
    36 GB of which nothing else is touched."""
    S = Setup(ctx, 9, 32, 16, 1, 64)
    T, n = 1 << 24, 3
    x = ctx.empty((9 * T, 64), np.float32)
    at = x.ptr + 8 * T * 64 * 4
    k = S.rng.standard_normal((n, 64)).astype(np.float32)
    ctx.lib.b200q_upload(ctx.handle, at, k.ctypes.data, k.nbytes)
    count = [0] * 8 + [n]
    S.cache.append(x, x, 64, 64, 9, T, S.dtable, S.per, S.dev([14] * 9), S.dev(count))
    for t in range(n):
        q, _, s = orc.quantize_per_token(k[t][None])
        p, r = S.table[8, (14 + t) // 16], (14 + t) % 16
        for i in range(2):
            S.codes[i][p, 0, r], S.scales[i][p, 0, r] = q[0], s[0]
    S.check()
    S.cache.read(9, T, S.dtable, S.per, S.dev([14] * 9), S.dev(count), x, x, 64, 64)   # K and V are alike, so one operand takes both
    got = np.empty_like(k)
    ctx.lib.b200q_download(ctx.handle, got.ctypes.data, at, got.nbytes)
    c, _, s = orc.quantize_per_token(k)
    want = c.astype(np.float32) * np.reshape(s, (-1, 1))
    assert (got.view(np.uint32) == want.view(np.uint32)).all()
    x.free()


def test_refusals(ctx):
    import mlfw_b200
    S = Setup(ctx, 1, 32, 16, 2, 64)
    c, b, s, e = S.cache, ctx.empty((4096,), np.float32), S.dev([0]), mlfw_b200.B200QError
    other = mlfw_b200.Context(0)
    with pytest.raises(e, match="another context"):
        mlfw_b200.device.check(ctx.lib.b200q_kv_append(other.handle, c.handle, b.ptr, b.ptr, 128, 128, 1, 1, S.dtable.ptr, S.per, s.ptr, None))
    other.close()
    for what, call in (
            ("16-byte", lambda: c.append(b.ptr + 4, b, 128, 128, 1, 1, S.dtable, S.per, s)),
            ("16-byte", lambda: c.append(b, b, 128, 130, 1, 1, S.dtable, S.per, s)),
            ("below heads", lambda: c.append(b, b, 64, 128, 1, 1, S.dtable, S.per, s)),
            ("null pointer", lambda: c.append(b, None, 128, 128, 1, 1, S.dtable, S.per, s)),
            ("null pointer", lambda: c.append(b, b, 128, 128, 1, 1, None, S.per, s)),
            ("null pointer", lambda: c.read(1, 1, S.dtable, S.per, None, None, b, b, 128, 128)),
            ("negative", lambda: c.read(-1, 1, S.dtable, S.per, s, None, b, b, 128, 128)),
            ("multiple of the cache's", lambda: c.attention(b, 192, 1, 1, 3, S.dtable, S.per, s, None, None, 1.0, b, 192)),
            ("multiple of the cache's", lambda: c.attention(b, 192, 1, 1, 0, S.dtable, S.per, s, None, None, 1.0, b, 192)),
            ("at most 64", lambda: c.attention(b, 128, 1, 65, 2, S.dtable, S.per, s, None, b, 1.0, b, 128)),
            ("finite", lambda: c.attention(b, 128, 1, 1, 2, S.dtable, S.per, s, None, None, float("nan"), b, 128)),
            ("below heads", lambda: c.attention(b, 128, 1, 1, 4, S.dtable, S.per, s, None, None, 1.0, b, 256)),
            ("at most 64", lambda: c.keep(1, 65, S.dtable, S.per, s, b, None)),
            ("null pointer", lambda: c.keep(1, 4, S.dtable, S.per, s, None, None)),
            ("below 2\\^31", lambda: c.read(1 << 16, 1 << 15, S.dtable, S.per, s, None, b, b, 128, 128))):
        with pytest.raises(e, match=what):
            call()
    for call in (lambda: c.append(b, b, 128, 128, 1, 1, S.dtable.ptr + 2, S.per, s), lambda: c.read(1, 1, S.dtable, S.per, s.ptr + 1, None, b, b, 128, 128),
                 lambda: c.append(b, b, 128, 128, 1, 1, S.dtable, S.per, s, s.ptr + 2), lambda: c.keep(1, 4, S.dtable, S.per, s, b.ptr + 2, None),
                 lambda: c.attention(b, 128, 1, 1, 2, S.dtable, S.per, s, None, b.ptr + 4, 1.0, b, 128)):
        with pytest.raises(e, match="multiple of its element"):
            call()
    before = ctx.launch_count()
    c.append(b, b, 128, 128, 0, 4, None, 0, None)          # nothing to do is not an error
    c.attention(b, 128, 3, 0, 2, None, 0, None, None, None, 1.0, b, 128)
    assert ctx.launch_count() == before
    with pytest.raises(e, match="a page holds"):
        mlfw_b200.KVCache(ctx, 4, 20, 2, 64)
    S.check()


# ------------------------------------------------------------------------------------------------ together
def test_serving_run(ctx, orc):
    """A prompt in two chunks, decoding steps, a drafted tree with its accepted path, another step: every attention
    against the formula over what the cache must hold by then."""
    B, H, heads, dim, page = 3, 6, 3, 64, 16
    S = Setup(ctx, B, 120, page, heads, dim)
    length = np.zeros(B, np.int64)

    def step(T, count, tree=None):
        x = S.rng.standard_normal((B * T, (H + 2 * heads) * dim)).astype(np.float32)
        ld = x.shape[1]
        d = ctx.to_device(x)
        S.cache.append(d.ptr + 4 * H * dim, d.ptr + 4 * (H + heads) * dim, ld, ld, B, T, S.dtable, S.per, S.dev(length), S.dev(count))
        x = x.reshape(B, T, H + 2 * heads, dim)
        S.append(orc, x[:, :, H:H + heads], x[:, :, H + heads:], length, count)
        check_attention(S, np.ascontiguousarray(x[:, :, :H]), length, np.array(count), tree, dim ** -0.5)
        S.check()

    for T, count in ((40, [40, 17, 33]), (21, [21, 0, 5]), (1, [1, 1, 1]), (1, [1, 0, 1])):
        step(T, count)
        length += count
    tree = random_tree(S.rng, B, 24)
    step(24, [24, 24, 11], tree)
    keep, kept = np.zeros((B, 24), np.int64), np.zeros(B, np.int64)
    for b, leaf in enumerate((23, 20, 10)):
        path = np.flatnonzero((tree[b, leaf] >> np.arange(24, dtype=np.uint64)) & np.uint64(1))
        keep[b, : path.size], kept[b] = path, path.size
    S.cache.keep(B, 24, S.dtable, S.per, S.dev(length), S.dev(keep), S.dev(kept))
    ctx.sync()
    for a in S.codes + S.scales:
        for b in range(B):
            src, dst = length[b] + keep[b, : kept[b]], length[b] + np.arange(kept[b])
            a[S.table[b, dst // page], :, dst % page] = a[S.table[b, src // page], :, src % page]
    length += kept
    step(1, [1, 1, 1])


def test_recorded_step_follows_the_lengths(ctx, orc):
    """Append + attention recorded once and replayed while start grows; two recordings of one context in turn."""
    B, heads, dim = 2, 4, 64
    S = Setup(ctx, B, 90, 16, heads, dim)
    T2 = 20
    ld = 3 * heads * dim
    start, rows = Guarded(ctx, (B,), np.int32), [Guarded(ctx, (B * T, ld), np.float32) for T in (1, T2)]
    outs = [Guarded(ctx, (B * T, heads * dim), np.float32) for T in (1, T2)]

    def call(i, T):
        p = rows[i].ptr
        S.cache.append(p + 4 * heads * dim, p + 8 * heads * dim, ld, ld, B, T, S.dtable, S.per, start.ptr)
        S.cache.attention(p, ld, B, T, heads, S.dtable, S.per, start.ptr, None, None, 0.125, outs[i].ptr, heads * dim)

    graphs = []
    for i, T in enumerate((1, T2)):
        ctx.graph_begin()
        call(i, T)
        graphs.append(ctx.graph_end())
    length = np.array([0, 3])
    S.fill(length)
    for i in (1, 0, 0, 1, 0):
        T = (1, T2)[i]
        x = S.rng.standard_normal((B * T, ld)).astype(np.float32)
        start.upload(length.astype(np.int32))
        rows[i].upload(x)
        ctx.graph_launch(graphs[i])
        ctx.sync()
        x = x.reshape(B, T, 3, heads, dim)
        S.append(orc, x[:, :, 1], x[:, :, 2], length, [T] * B)
        S.check()
        want, bound = attention_rows(S, np.ascontiguousarray(x[:, :, 0]), length, [T] * B, None, 0.125)
        assert (np.abs(outs[i].download().reshape(want.shape) - want).max(-1) <= bound).all()
        length += T
    for g in graphs:
        ctx.graph_destroy(g)


def test_recordings_and_eager_calls_in_turn(ctx):
    """Attention of one, 40 and 140 query rows recorded, replayed in turn with eager calls on the same workspace, the pieces of
    long items among them: every result is bit for bit the first one's."""
    S = Setup(ctx, 3, 2200, 64, 2, 128)
    for i in range(2):
        S.codes[i] = np.clip(np.round(S.rng.standard_normal(S.codes[i].shape) * 42), -127, 127).astype(np.int8)
        S.scales[i] = S.rng.uniform(0.01, 0.03, S.scales[i].shape).astype(np.float32)
    S.upload()
    start, calls = S.dev([2100, 33, 700]), []
    for T, H in ((1, 4), (20, 4), (70, 4)):
        q, o = ctx.to_device(S.rng.standard_normal((3 * T, H * 128)).astype(np.float32)), ctx.empty((3 * T, H * 128), np.float32)
        calls.append((lambda q=q, o=o, T=T, H=H: S.cache.attention(q, H * 128, 3, T, H, S.dtable, S.per, start, None, None, 0.1, o, H * 128), o))
    want, graphs = [], []
    for call, o in calls:
        call()
        want.append(o.download().view(np.uint32))
        ctx.graph_begin()
        call()
        graphs.append(ctx.graph_end())
    for i, replay in ((0, 1), (1, 1), (2, 1), (2, 0), (0, 1), (1, 0), (1, 1), (0, 0), (2, 1), (2, 1), (0, 1)):
        calls[i][1].fill_bytes(0xff)
        ctx.graph_launch(graphs[i]) if replay else calls[i][0]()
        for j in range(3):
            ctx.graph_launch(graphs[j])
        assert all((calls[j][1].download().view(np.uint32) == want[j]).all() for j in range(3))
    for g in graphs:
        ctx.graph_destroy(g)


def test_two_contexts_at_once(ctx):
    """Each context has its stream and its workspace: calls of both under way together give what they give alone."""
    import mlfw_b200
    with mlfw_b200.Context(0) as other:
        both = []
        for c in (ctx, other):
            S = Setup(c, 4, 1500, 32, 2, 64, seed=5)
            for i in range(2):
                S.codes[i] = np.clip(np.round(S.rng.standard_normal(S.codes[i].shape) * 42), -127, 127).astype(np.int8)
                S.scales[i] = S.rng.uniform(0.01, 0.03, S.scales[i].shape).astype(np.float32)
            S.upload()
            start = S.dev([1400, 0, 900, 77])
            for T, H in ((1, 6), (24, 4), (65, 4)):
                q, o = c.to_device(S.rng.standard_normal((4 * T, H * 64)).astype(np.float32)), c.empty((4 * T, H * 64), np.float32)
                both.append((c, lambda S=S, q=q, o=o, T=T, H=H, start=start: S.cache.attention(q, H * 64, 4, T, H, S.dtable, S.per, start, None, None, 0.1, o, H * 64), o, S))
        want = []
        for c, call, o, _ in both:
            call()
            want.append(o.download().view(np.uint32))
            o.fill_bytes(0xff)
            c.sync()
        for _ in range(20):
            for k in (0, 3, 1, 4, 2, 5):
                both[k][1]()
        for (c, _, o, _), w in zip(both, want):
            assert (o.download().view(np.uint32) == w).all()
        other.check_status()
        both.clear()
        del call, o, S, q, start


def test_block_with_a_cache(ctx):
    """GPTBlock.forward_cached: the same linears as GPTBlock.forward around an attention over the cache's rows."""
    import mlfw_b200
    from mlfw_b200.block import GPTBlock, random_block_params
    D, H, FF, B, page = 128, 2, 512, 2, 16
    blk = GPTBlock(ctx, D, H, FF, random_block_params(D, FF, seed=4, std=0.3))
    rng = np.random.default_rng(8)
    table = rng.permutation(12).reshape(B, 6).astype(np.int32)
    cache = mlfw_b200.KVCache(ctx, 12, page, H, 64)
    dt = ctx.to_device(table)
    length = np.zeros(B, np.int32)
    for T, tree in ((37, None), (1, None), (1, None), (8, random_tree(rng, B, 8)), (37, None)):
        h = rng.standard_normal((B * T, D)).astype(np.float32)
        dh, out = ctx.to_device(h), Guarded(ctx, (B * T, D), np.float32)
        t = blk.forward_cached(dh, B, T, cache, dt, 6, ctx.to_device(length), out.ptr, tree=None if tree is None else ctx.to_device(tree))
        ctx.sync()
        n = int(length.max()) + T
        outs = [ctx.empty((B, n, H, 64), np.float32) for _ in range(2)]
        cache.read(B, n, dt, 6, ctx.to_device(np.zeros(B, np.int32)), None, outs[0], outs[1], D, D)
        ctx.sync()
        k, v = (o.download().astype(np.float64) for o in outs)
        qkv = t["qkv"].download().reshape(B, T, 3, H, 64)
        # the new rows in the cache are the projections to half a code step
        for i, x in ((1, k), (2, v)):
            step = np.abs(qkv[:, :, i]).max(-1, keepdims=True) / 127
            assert (np.abs(x[:, length[0]:length[0] + T] - qkv[:, :, i]) <= 0.5 * step * (1 + 2.0**-20)).all()
        attn = t["attn"].download().reshape(B, T, H, 64)
        j = np.arange(n) - int(length[0])
        for b in range(B):
            for r in range(T):
                see = (j < 0) | ((j <= r) if tree is None else ((tree[b, r] >> np.clip(j, 0, 63).astype(np.uint64)) & np.uint64(1)).astype(bool))
                for hd in range(H):
                    z = 0.125 * (k[b, see, hd] @ qkv[b, r, 0, hd].astype(np.float64))
                    w = np.exp(z - z.max())
                    want = w @ v[b, see, hd] / w.sum()
                    # the bound of the attention test with the rows' values in place of code * scale
                    tol = attention_bound(qkv[b, r, 0, hd].astype(np.float64), k[b, :, hd], np.ones(n), v[b, :, hd], np.ones(n), 0.125, see)
                    assert np.abs(attn[b, r, hd] - want).max() <= tol
        # what follows the attention is what forward() does with the same attention output
        again = Guarded(ctx, (B * T, D), np.float32)
        blk._after_attention(dh, B * T, t, again.ptr)
        ctx.sync()
        assert (again.download().view(np.uint32) == out.download().view(np.uint32)).all()
        length += T if T != 8 else 0                 # the drafted rows are all refused
    cache.close()


def test_recorded_block_step_survives_larger_prompts(ctx):
    """A recorded decoding step of a block, replayed after prompts that made every workspace of the context grow."""
    import mlfw_b200
    from mlfw_b200.block import GPTBlock, random_block_params
    with mlfw_b200.Context(0) as c:
        D, H, FF, B = 128, 2, 512, 2
        blk = GPTBlock(c, D, H, FF, random_block_params(D, FF, seed=6, std=0.3))
        cache = mlfw_b200.KVCache(c, 2 * 8, 64, H, 64)
        table = c.to_device(np.arange(16, dtype=np.int32).reshape(B, 8))
        rng = np.random.default_rng(9)
        step, out, length = c.to_device(rng.standard_normal((B, D)).astype(np.float32)), c.empty((B, D), np.float32), c.to_device(np.array([3, 5], np.int32))
        first = c.to_device(np.zeros(B, np.int32))
        prompt = rng.standard_normal((B * 8, D)).astype(np.float32)

        def run(T, h, where, o):
            blk.forward_cached(h, B, T, cache, table, 8, where, o)

        run(8, c.to_device(prompt), first, c.empty((B * 8, D), np.float32))
        run(1, step, length, out)
        c.sync()
        want = out.download()
        c.graph_begin()
        run(1, step, length, out)
        graph = c.graph_end()
        big = c.to_device(rng.standard_normal((B * 400, D)).astype(np.float32))
        run(400, big, first, c.empty((B * 400, D), np.float32))          # the workspaces grow
        run(8, c.to_device(prompt), first, c.empty((B * 8, D), np.float32))
        for _ in range(3):
            out.fill_bytes(0)
            c.graph_launch(graph)
            run(400, big, c.to_device(np.array([100, 100], np.int32)), c.empty((B * 400, D), np.float32))
            c.sync()
            assert (out.download().view(np.uint32) == want.view(np.uint32)).all()
        c.graph_destroy(graph)
        c.check_status()
        cache.close()

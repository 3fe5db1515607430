"""GPU tests of the int8 key/value cache as a serving host calls it: steps one behind the other without a wait between
them, and accuracy where the operands are uneven.

The host model of the cache, the formula in binary64 and the guarded buffers are those of test_gpu_kv_cache.py.
"""
import numpy as np
import pytest

from gpu_util import Guarded
from test_gpu_kv_cache import Setup, attention_bound, attention_rows, check_attention, random_tree, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mlfw_b200
    c = mlfw_b200.Context(0)
    yield c
    c.check_status()
    c.close()


# ------------------------------------------------------------------------------------------------ steps without a wait
@pytest.mark.parametrize("heads,H,dim,T", [(2, 4, 128, 40), (3, 3, 64, 40), (2, 2, 64, 12)])
def test_verification_steps_back_to_back(ctx, orc, heads, H, dim, T):
    """Append, tree attention, keep, read, over and over on the same positions with other data, nothing between the launches:
    every kernel reads what the one before it has just written.  Once call by call, twice as one recording."""
    B, page, steps = 2, 16, 10
    S = Setup(ctx, B, 100 + T, page, heads, dim)
    start = np.array([100, 37])
    S.fill(start)
    ld = (H + 2 * heads) * dim
    x = S.rng.standard_normal((steps, B * T, ld)).astype(np.float32)
    trees = [random_tree(S.rng, B, T) for _ in range(steps)]
    keep, kept = np.zeros((steps, B, T), np.int64), np.zeros((steps, B), np.int64)
    for i in range(steps):
        for b in range(B):
            path = np.flatnonzero((trees[i][b, S.rng.integers(T // 2, T)] >> np.arange(T, dtype=np.uint64)) & np.uint64(1))
            keep[i, b, : path.size], kept[i, b] = path, path.size
    dx, dtree, dkeep, dkept = [ctx.to_device(a) for a in x], [S.dev(t, np.uint64) for t in trees], [S.dev(a) for a in keep], [S.dev(a) for a in kept]
    dstart = S.dev(start)
    outs = [[Guarded(ctx, (B * T, n * dim), np.float32, np.zeros((B * T, n * dim))) for n in (H, heads, heads)] for _ in range(steps)]

    def run():
        for i in range(steps):
            p, (o, k, v) = dx[i].ptr, outs[i]
            S.cache.append(p + 4 * H * dim, p + 4 * (H + heads) * dim, ld, ld, B, T, S.dtable, S.per, dstart)
            S.cache.attention(p, ld, B, T, H, S.dtable, S.per, dstart, None, dtree[i], dim ** -0.5, o.ptr, H * dim)
            S.cache.keep(B, T, S.dtable, S.per, dstart, dkeep[i], dkept[i])
            S.cache.read(B, T, S.dtable, S.per, dstart, None, k.ptr, v.ptr, heads * dim, heads * dim)

    want = []
    for i in range(steps):
        r = x[i].reshape(B, T, H + 2 * heads, dim)
        S.append(orc, r[:, :, H:H + heads], r[:, :, H + heads:], start, [T] * B)
        attn = attention_rows(S, np.ascontiguousarray(r[:, :, :H]), start, [T] * B, trees[i], dim ** -0.5)
        for a in S.codes + S.scales:
            for b in range(B):
                src, dst = start[b] + keep[i, b, : kept[i, b]], start[b] + np.arange(kept[i, b])
                a[S.table[b, dst // page], :, dst % page] = a[S.table[b, src // page], :, src % page]
        back = []
        for j in range(2):
            pos = start[:, None] + np.arange(T)
            p, at = np.take_along_axis(S.table, pos // page, 1), pos % page
            back.append(S.codes[j][p, :, at].astype(np.float32) * S.scales[j][p, :, at][..., None])
        want.append((attn, back))

    def check():
        for (o, k, v), ((value, bound), back) in zip(outs, want):
            assert (np.abs(o.download().reshape(value.shape) - value).max(-1) <= bound).all()
            for got, w in ((k, back[0]), (v, back[1])):
                assert (got.download().view(np.uint32) == w.reshape(B * T, -1).view(np.uint32)).all()
        S.check()

    run()
    check()
    first = [o.download().view(np.uint32) for o, _, _ in outs]
    ctx.graph_begin()
    run()
    graph = ctx.graph_end()
    for _ in range(2):
        for row in outs:
            for buf in row:
                buf.upload(np.zeros(buf.shape))
        ctx.graph_launch(graph)
        ctx.graph_launch(graph)
        check()
        assert all((o.download().view(np.uint32) == f).all() for (o, _, _), f in zip(outs, first))
    ctx.graph_destroy(graph)


def test_a_recording_belongs_to_its_context(ctx):
    """Launching or destroying it through another context is refused: the workspaces it uses are its own context's."""
    import mlfw_b200
    S = Setup(ctx, 1, 40, 16, 2, 64)
    S.fill([40])
    start, q = S.dev([39]), ctx.to_device(S.rng.standard_normal((1, 128)).astype(np.float32))
    out = Guarded(ctx, (1, 128), np.float32, np.zeros((1, 128)))
    ctx.graph_begin()
    S.cache.attention(q, 128, 1, 1, 2, S.dtable, S.per, start, None, None, 0.125, out.ptr, 128)
    graph = ctx.graph_end()
    with mlfw_b200.Context(0) as other:
        with pytest.raises(mlfw_b200.B200QError, match="another context"):
            other.graph_launch(graph)
        with pytest.raises(mlfw_b200.B200QError, match="another context"):
            other.graph_destroy(graph)
    assert (out.download() == 0).all()
    ctx.graph_launch(graph)
    value, bound = attention_rows(S, q.download().reshape(1, 1, 2, 64), [39], [1], None, 0.125)
    assert (np.abs(out.download().reshape(value.shape) - value).max(-1) <= bound).all()
    ctx.graph_destroy(graph)


# ------------------------------------------------------------------------------------------------ the block over a cache
def block_attention(k, v, qkv, start, count, tree):
    """The formula in binary64 over rows read back (k, v [B, n, H, 64]) and its bound, for the rows in use."""
    for b in range(len(start)):
        n = int(start[b]) + int(count[b])
        j = np.arange(n) - int(start[b])
        for r in range(int(count[b])):
            see = (j < 0) | ((j <= r) if tree is None else ((tree[b, r] >> np.clip(j, 0, 63).astype(np.uint64)) & np.uint64(1)).astype(bool))
            for h in range(k.shape[2]):
                x = qkv[b, r, 0, h].astype(np.float64)
                z = 0.125 * (k[b, :n][see, h] @ x)
                w = np.exp(z - z.max())
                one = np.ones(n)
                yield b, r, h, w @ v[b, :n][see, h] / w.sum(), attention_bound(x, k[b, :n, h], one, v[b, :n, h], one, 0.125, see)


@pytest.mark.parametrize("tree", [False, True])
def test_block_with_a_padded_batch(ctx, tree):
    """forward_cached with uneven counts, none among them, call by call and recorded: rows in use follow the formula, rows behind
    them have no attention and change nothing."""
    import mlfw_b200
    from mlfw_b200.block import GPTBlock, random_block_params
    D, H, FF, B, T, page = 128, 2, 512, 4, 9, 16
    blk = GPTBlock(ctx, D, H, FF, random_block_params(D, FF, seed=12, std=0.3))
    rng = np.random.default_rng(13)
    table, cache = rng.permutation(16).reshape(B, 4).astype(np.int32), mlfw_b200.KVCache(ctx, 16, page, H, 64)
    for b in (cache.k_codes, cache.v_codes):
        b.fill_bytes(0x80)
    for b in (cache.k_scales, cache.v_scales):
        b.fill_bytes(0xff)                                        # NaN: what no call has written must not show
    dt, length, zero = ctx.to_device(table), np.array([0, 20, 7, 30], np.int32), ctx.to_device(np.zeros(B, np.int32))
    fill = rng.standard_normal((B * 30, D)).astype(np.float32)
    blk.forward_cached(ctx.to_device(fill), B, 30, cache, dt, 4, zero, ctx.empty((B * 30, D), np.float32), count=ctx.to_device(length))
    start, counts = ctx.to_device(length), [np.array(c, np.int32) for c in ([9, 0, 4, 1], [0, 0, 0, 0], [3, 9, 0, 8])]
    trees = random_tree(rng, B, T) if tree else None
    h, out = Guarded(ctx, (B * T, D), np.float32), Guarded(ctx, (B * T, D), np.float32)
    dcount, dtree = Guarded(ctx, (B,), np.int32), ctx.to_device(trees) if tree else None

    def step():
        return blk.forward_cached(h.ptr, B, T, cache, dt, 4, start, out.ptr, count=dcount.ptr, tree=dtree)

    def rows(count):
        h.upload(x)
        dcount.upload(count)

    graph = None
    for count in counts + counts:
        x = rng.standard_normal((B * T, D)).astype(np.float32)
        rows(count)
        if graph is None:
            t = step()
        else:
            ctx.graph_launch(graph)
        ctx.sync()
        attn, got = t["attn"].download().reshape(B, T, H, 64), out.download().reshape(B, T, D)
        back = [ctx.empty((B, 40, H, 64), np.float32).fill_bytes(0) for _ in range(2)]
        cache.read(B, 40, dt, 4, zero, ctx.to_device(length + count), back[0], back[1], D, D)
        k, v = (o.download().astype(np.float64) for o in back)
        qkv = t["qkv"].download().reshape(B, T, 3, H, 64)
        for b, r, hd, want, bound in block_attention(k, v, qkv, length, count, trees):
            assert np.abs(attn[b, r, hd] - want).max() <= bound
        used = np.arange(T)[None, :] < count[:, None]
        assert (attn[~used] == 0).all() and np.isfinite(got).all()
        x[~used.reshape(-1)] = rng.standard_normal((int((~used).sum()), D)) * 50      # other padding, the same rows in use
        rows(count)
        step()
        ctx.sync()
        again = out.download().reshape(B, T, D)
        assert (again[used].view(np.uint32) == got[used].view(np.uint32)).all()
        if graph is None and count is counts[-1]:
            ctx.graph_begin()
            t = step()
            graph = ctx.graph_end()
    ctx.graph_destroy(graph)
    cache.close()


# ------------------------------------------------------------------------------------------------ operands of any magnitude
MAGNITUDES = [(1e37, 1e37), (1e-35, 1e-35), (1e-36, 1e3), (1e-30, 1e12), (1e-20, 1e20), (1, 1e37), (1e37, 1), (1e3, 1e-36)]


@pytest.mark.parametrize("T,dim", [(1, 64), (1, 128), (9, 64), (9, 128)])
def test_attention_over_values_of_any_magnitude(ctx, T, dim):
    """V near both ends of binary32, changing from the first tokens to the later ones and from token to token."""
    n = 300
    S = Setup(ctx, 1, n + T, 32, 2, dim)
    S.fill([n + T])
    q = S.rng.standard_normal((1, T, 4, dim)).astype(np.float32)
    plain = [a.copy() for a in S.scales]
    pos = np.arange(n + T)
    page, row = S.table[0, pos // S.page], pos % S.page
    for a, b in MAGNITUDES:
        for which in (pos < 32, pos % 2 == 0, pos < 200):
            S.scales[1][:] = plain[1]
            S.scales[1][page, :, row] *= np.where(which, a, b).astype(np.float32)[:, None]
            S.upload()
            check_attention(S, q, [n], None, None, dim ** -0.5)
    # the largest values there are, in one sequence that the whole GPU shares
    S = Setup(ctx, 1, 6000 + T, 64, 2, dim)
    S.codes[1][:], S.scales[1][:] = 127, np.float32(2.6e36)
    S.codes[0][:] = np.clip(np.round(S.rng.standard_normal(S.codes[0].shape) * 42), -127, 127)
    S.scales[0][:] = 0.02
    S.upload()
    check_attention(S, q, [6000], None, None, dim ** -0.5)


@pytest.mark.parametrize("T,dim,n", [(1, 64, 200), (1, 128, 5000), (9, 64, 3000), (9, 128, 150), (25, 64, 200), (25, 128, 4000), (70, 64, 3000),
                                     (70, 128, 300)])
def test_attention_scores_of_any_magnitude(ctx, T, dim, n):
    """Two equal keys lead all others by more than any weight survives, at opposite ends of the sequence: their values' mean, however
    large the scores are and whichever sign they have.  One exact addition and one division: off by a few roundings."""
    S = Setup(ctx, 1, n + T, 32, 1, dim)
    S.fill([n + T])
    plain = [a.copy() for a in S.codes + S.scales]
    sign = S.rng.choice([-1, 1], dim)
    q = np.broadcast_to(sign * S.rng.uniform(0.5, 2, dim), (1, T, 2, dim)).astype(np.float32)
    lead = [5, n - 9]
    page, row = S.table[0, lead[0] // 32], lead[0] % 32
    page2, row2 = S.table[0, lead[1] // 32], lead[1] % 32
    want = np.mean([S.codes[1][p, 0, r].astype(np.float64) * S.scales[1][p, 0, r] for p, r in ((page, row), (page2, row2))], axis=0)
    vmax = np.max(np.abs(want)) * 2
    for negative in (False, True):
        for f_q, f_k in ((1e5, 1), (1e7, 1), (1e9, 1), (1e13, 1), (1e20, 1e10), (1e36, 1), (1, 1e7), (1, 1e25), (1, 1e34)):
            S.codes[0][:], S.scales[0][:] = plain[0], np.float32(0.02 * f_k)
            if negative:                                          # every score far below zero
                S.codes[0][:] = -sign * (100 + S.rng.integers(0, 28, S.codes[0].shape[:-1])[..., None])
            for p, r in ((page, row), (page2, row2)):
                S.codes[0][p, 0, r] = sign * (-60 if negative else 127)
            S.upload()
            got = run_attention(S, (q * np.float32(f_q)).astype(np.float32), [n], None, None, dim ** -0.5)
            assert np.abs(got - want).max() <= 8 * 2.0**-24 * vmax, (negative, f_q, f_k, np.abs(got - want).max() / vmax)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spread", [0.0, 0.3])
def test_attention_one_key_above_many(ctx, dim, spread):
    """One key 2^9 to 2^35 times as heavy as each of 20000 others, which one warp walks: none of the others' weight may get lost.

    Many sequences over the same pages, so that a piece is nearly a whole context.  With w the weights, v the values, r the result
    and u = 2^-24: a weight is off by its score's rounding, ten u of |z| (two terms and what combines them), ex2 (2^-21) and the
    rounding of z - c (u times its 40 or fewer bits), which moves r by w |v - r| / sum w; its rounding to units, 2^-28 of the largest weight,
    is noise of at most half a unit each, six deviations of which are 3 sqrt(sum v^2) units; 24 u of sum w |v| for the sums and joins.
    """
    B, n, page = 1300, 20000, 256
    S = Setup(ctx, 1, n, page, 1, dim)
    S.codes[0][:], S.scales[0][:] = 0, np.float32(0.01)
    S.codes[0][..., 1] = S.rng.integers(-127, 128, S.codes[0].shape[:-1])
    S.codes[1][:] = np.clip(np.round(S.rng.standard_normal(S.codes[1].shape) * 42), -127, 127)
    S.codes[1][..., 0] = 100
    S.scales[1][:] = np.float32(0.02)
    at = 777
    S.codes[0][S.table[0, at // page], 0, at % page, :2] = 127, 0
    S.codes[1][S.table[0, at // page], 0, at % page] = S.rng.integers(-127, 128, dim)
    S.upload()
    bits = np.linspace(9, 35, B)
    q = np.zeros((B, 1, 1, dim), np.float32)
    q[:, 0, 0, 0], q[:, 0, 0, 1] = bits * np.log(2) / 1.27, spread * np.log(2) / 1.27
    out = Guarded(ctx, (B, dim), np.float32, np.zeros((B, dim)))
    table = ctx.to_device(np.ascontiguousarray(np.broadcast_to(S.table, (B, S.per))))
    S.cache.attention(ctx.to_device(q), dim, B, 1, 1, table, S.per, S.dev([n - 1] * B), None, None, 1.0, out.ptr, dim)
    got = out.download()
    kc, vc, ks, vs = S.tokens(0, n)
    v = vc[:, 0].astype(np.float64) * vs[:, 0, None]
    u = 2.0**-24
    for b in range(0, B, 13):
        z = ks[:, 0].astype(np.float64) * (kc[:, 0].astype(np.float64) @ q[b, 0, 0].astype(np.float64))
        w = np.exp(z - z.max())
        total = w.sum()
        want = w @ v / total
        delta = 10 * u * np.abs(z) + 2.0**-21 + 40 * u
        bound = (w * delta) @ np.abs(v - want) / total + 3 * np.sqrt((v * v).sum(0)) * 2.0**-28 / total + 24 * u * (w @ np.abs(v)) / total
        assert (np.abs(got[b] - want) <= bound).all(), (bits[b], np.max(np.abs(got[b] - want) / bound))


@pytest.mark.parametrize("T,dim", [(1, 64), (1, 128), (40, 64), (40, 128), (130, 128)])
def test_attention_beside_a_strong_channel(ctx, T, dim):
    """One channel of the queries far above the others, on which K is zero: the others keep their digits.

    K has four channels that are not zero.  With u = 2^-24, a score is off by 16 u of sum |q k|: four products and their sum, eight
    roundings that combine and scale it, four u for a query element in two binary16 parts; in the kernel for few rows an element is
    held to 2^-31 of the row's largest as well.  That moves the result by sum w |v - r| delta / sum w, with 2^-21 for ex2 and u times the
    bits between a score and the largest; 22 bits of a weight and (n / 64 + 24) u of sum w |v| for the sums.
    """
    n = 260
    S = Setup(ctx, 1, n + T, 32, 2, dim)
    S.fill([n + T])
    S.codes[0][..., 4:] = 0
    S.upload()
    kc, vc, ks, vs = S.tokens(0, n + T)
    u = 2.0**-24
    few = T * 2 <= 36
    for strong in (1.0, 200.0, 2000.0, 1e4) + (() if few else (1e5, 1e7)):
        q = (S.rng.standard_normal((1, T, 4, dim)) * 6).astype(np.float32)
        q[..., dim - 1] = strong
        got = run_attention(S, q, [n], None, None, 0.125)
        for t in range(T):
            for h in range(4):
                g, m = h // 2, n + t + 1
                x, k = q[0, t, h].astype(np.float64), kc[:m, g].astype(np.float64) * ks[:m, g, None]
                v = vc[:m, g].astype(np.float64) * vs[:m, g, None]
                z = 0.125 * (k @ x)
                w = np.exp(z - z.max())
                r = w @ v / w.sum()
                held = np.abs(k).sum(1) * strong * 2.0**-31 if few else 0
                delta = 0.125 * (16 * u * (np.abs(k) @ np.abs(x)) + held) + 2.0**-21 + u * (z.max() - z + 16)
                bound = (w * delta) @ np.abs(v - r) / w.sum() + (4 * u + (m / 64 + 24) * u) * (w @ np.abs(v)) / w.sum()
                assert (np.abs(got[0, t, h] - r) <= bound).all(), (strong, t, h, np.max(np.abs(got[0, t, h] - r) / bound))


@pytest.mark.parametrize("dim", [64, 128])
def test_a_single_visible_value_of_any_magnitude(ctx, dim):
    """The first row of a chunk sees one token and returns its value: 22 bits of the weight, four roundings."""
    S = Setup(ctx, 1, 40, 16, 2, dim)
    S.fill([40])
    plain = S.scales[1].copy()
    q = S.rng.standard_normal((1, 40, 4, dim)).astype(np.float32)
    for f in (1e-30, 1e-10, 1, 1e10, 1e30, 1e37, 1e38):
        S.scales[1][:] = plain * np.float32(f)
        S.upload()
        got = run_attention(S, q, [0], None, None, dim ** -0.5)
        _, vc, _, vs = S.tokens(0, 1)
        want = np.repeat(vc[0].astype(np.float64) * vs[0, :, None], 2, axis=0)
        assert np.abs(got[0, 0] - want).max() <= 8 * 2.0**-24 * np.abs(want).max(), (f, np.abs(got[0, 0] - want).max() / np.abs(want).max())


@pytest.mark.parametrize("T,dim", [(1, 64), (1, 128), (9, 64), (24, 64), (20, 128), (67, 64)])
def test_equal_scores_weigh_the_same_wherever_they_are(ctx, T, dim):
    """Three equal keys among many far below, in different tiles of long runs: the mean of their values at every size of the scores.
    Many sequences over the same pages, so that a warp walks many tiles and meets the keys in the middle of its run."""
    B, n, page = 300 if T * 2 <= 36 else 40, 3000, 64
    S = Setup(ctx, 1, n + T, page, 1, dim)
    S.fill([n + T])
    sign = S.rng.choice([-1, 1], dim)
    q = np.broadcast_to(sign * S.rng.uniform(0.5, 2, dim), (B, T, 2, dim)).astype(np.float32)
    table = ctx.to_device(np.ascontiguousarray(np.broadcast_to(S.table, (B, S.per))))
    out = Guarded(ctx, (B * T, 2 * dim), np.float32, np.zeros((B * T, 2 * dim)))
    plain = S.codes[0].copy()
    for negative in (False, True):
        for f in np.geomspace(1e4, 1e8, 17):
            S.codes[0][:], S.scales[0][:] = plain, np.float32(0.02)
            if negative:
                S.codes[0][:] = -sign * (100 + S.rng.integers(0, 28, S.codes[0].shape[:-1])[..., None])
            lead = S.rng.choice(n, 3, replace=False)
            at = S.table[0, lead // page], 0, lead % page
            S.codes[0][at] = sign * (-60 if negative else 127)
            S.upload()
            values = S.codes[1][at].astype(np.float64) * S.scales[1][at][:, None]
            S.cache.attention(ctx.to_device((q * np.float32(f)).reshape(B * T, 2 * dim)), 2 * dim, B, T, 2, table, S.per, S.dev([n] * B), None, None,
                              dim ** -0.5, out.ptr, 2 * dim)
            err = np.abs(out.download().reshape(B, T, 2, dim) - values.mean(0)).max()
            assert err <= 8 * 2.0**-24 * np.abs(values).max(), (negative, f, err / np.abs(values).max())


@pytest.mark.parametrize("T,H,dim,n", [(41, 1, 64, 700), (63, 3, 64, 150), (39, 1, 128, 2000), (64, 4, 128, 90), (11, 1, 64, 700), (33, 1, 128, 90)])
def test_rows_with_large_scores_beside_ordinary_ones(ctx, T, H, dim, n):
    """A drafted tree of which every third row has scores in the millions, of either sign, and some rows see only new tokens: the large ones
    return the value of their largest score (the next is out of reach), the ordinary ones follow the formula, page ends and all."""
    S = Setup(ctx, 2, n + T, 16, 1, dim)
    start, count = [n, 0], [T, T - 2]
    S.fill(np.array(start) + count)
    q = S.rng.standard_normal((2, T, H, dim)).astype(np.float32)
    q[:, ::3] *= np.float32(1e6)
    q[:, 1::6] = 0
    tree = random_tree(S.rng, 2, T)
    tree[1, 4] = 0                                                # nothing at all
    got = run_attention(S, q, start, count, tree, 0.3)
    with np.errstate(over="ignore"):                              # the bound of the large rows says nothing
        want, bound = attention_rows(S, q, start, count, tree, 0.3)
    for b in range(2):
        m = start[b] + count[b]
        kc, vc, ks, vs = (a[:, 0] for a in S.tokens(b, m))
        j = np.arange(m) - start[b]
        for t in range(count[b]):
            see = (j < 0) | ((tree[b, t] >> np.clip(j, 0, 63).astype(np.uint64)) & np.uint64(1)).astype(bool)
            if not see.any():
                assert (got[b, t] == 0).all()
                continue
            for h in range(H):
                if t % 3:
                    assert np.abs(got[b, t, h] - want[b, t, h]).max() <= bound[b, t, h]
                    continue
                z = np.where(see, 0.3 * ks.astype(np.float64) * (kc.astype(np.float64) @ q[b, t, h].astype(np.float64)), -np.inf)
                first = int(np.argmax(z))
                if see.sum() > 1 and z[first] - np.partition(z, -2)[-2] < 1e-4 * np.abs(z[see]).max():
                    continue                                      # too near to tell in binary32
                v = vc[first].astype(np.float64) * vs[first]
                assert np.abs(got[b, t, h] - v).max() <= 8 * 2.0**-24 * np.abs(v).max(), (b, t, h)

"""The key/value cache operators as cases to time: writing K and V rows into the int8 cache and reading them back, attention of
single tokens, prompt chunks and drafted trees over the cache, and a whole verification step of drafted tokens.

``run`` computes a case in its plain form (elementary torch operations in binary32) where ``own`` is false and through
:class:`mlfw_b200.KVCache` where it is true.  Both see the same buffers: pages of ``page`` tokens, codes int8
[pages, heads, page, dim], scales f32 [pages, heads, page], a page table int32 [batch, table pages], ``start`` (tokens a
sequence holds before the call) and ``count`` (new rows of a sequence, at most ``rows``).
"""
import numpy as np
import torch

own = False

# what a pass calls:  write   append, then read the new rows back as the values the cache stands for
#                     read    read a range of the cache
#                     attend  attention of `rows` new tokens per sequence (already in the cache) over everything before them
#                     verify  append a drafted tree, tree attention, keep the accepted path, read the kept rows back


def listed():
    return [
        # one decoding step of a batch through the GPT block's heads: what every generated token pays, latency only
        dict(name="write_step_b32_h12x64", op="write", batch=32, rows=1, heads=12, kv_heads=12, dim=64, page=64, cached=700, ragged=True),
        # a padded batch of prompts of uneven length entering the cache (odd page ends)
        dict(name="write_prompt_b9x1031_h8x128", op="write", batch=9, rows=1031, heads=8, kv_heads=8, dim=128, page=32, cached=0, ragged=True),
        # a short shared prefix handed to another program
        dict(name="read_b3x77_h12x64", op="read", batch=3, rows=77, heads=12, kv_heads=12, dim=64, page=16, cached=40, ragged=True),
        # whole contexts read back for a re-run at full precision
        dict(name="read_b8x4096_h8x128", op="read", batch=8, rows=4096, heads=8, kv_heads=8, dim=128, page=64, cached=0, ragged=False),
        # one user, one token, a short chat: the smallest call
        dict(name="decode_b1_len500_h12x64", op="attend", batch=1, rows=1, heads=12, kv_heads=12, dim=64, page=64, cached=500, ragged=False),
        # a full serving batch of the GPT block's heads
        dict(name="decode_b64_len2k_h12x64", op="attend", batch=64, rows=1, heads=12, kv_heads=12, dim=64, page=64, cached=2048, ragged=True),
        # a serving batch with shared key heads and uneven contexts
        dict(name="decode_b48_len6k_h32of8x128", op="attend", batch=48, rows=1, heads=32, kv_heads=8, dim=128, page=64, cached=6000, ragged=True),
        # one very long document
        dict(name="decode_b1_len200k_h32of8x128", op="attend", batch=1, rows=1, heads=32, kv_heads=8, dim=128, page=128, cached=200001, ragged=False),
        # a chunk of two long prompts: many rows, bound by arithmetic
        dict(name="chunk_b2x512_len4k_h16of4x128", op="attend", batch=2, rows=512, heads=16, kv_heads=4, dim=128, page=64, cached=4000, ragged=True),
        # drafted tokens for one user, the smallest verification
        dict(name="verify_b1x8_len300_h12x64", op="verify", batch=1, rows=8, heads=12, kv_heads=12, dim=64, page=16, cached=300, ragged=False),
        # drafted trees for a batch of the GPT block's heads
        dict(name="verify_b32x16_len1k_h12x64", op="verify", batch=32, rows=16, heads=12, kv_heads=12, dim=64, page=64, cached=1000, ragged=True),
        # larger trees, shared key heads, contexts that end inside a page
        dict(name="verify_b8x31_len5k_h32of8x128", op="verify", batch=8, rows=31, heads=32, kv_heads=8, dim=128, page=64, cached=5003, ragged=True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    op = rng.choice(["write", "read", "attend", "attend", "attend", "verify", "verify"])
    ragged = rng.random() < 0.7
    row = 2 * kv_heads * (dim + 4)              # bytes of one cached token
    if op in ("write", "read"):
        tokens = _spread(rng, 1, 40_000_000 // row)
        batch = _spread(rng, 1, min(64, tokens))
        rows, cached = max(1, tokens // batch), rng.randrange(0, 300)
        group = 1
    elif op == "verify":
        rows, batch = rng.randint(2, 64), _spread(rng, 1, 32)
        cached = _spread(rng, 1, max(1, min(6000, 80_000_000 // (row * batch))))
    else:
        rows = rng.choice([1, 1, 2, 5, _spread(rng, 1, 500)])
        batch = _spread(rng, 1, 64 if rows < 8 else 4)
        # at most the bytes of the largest batch and the arithmetic of the largest chunk
        most = min(150_000, 400_000_000 // (row * batch), 1_500_000_000 // (batch * rows * kv_heads * group * dim))
        cached = _spread(rng, 1, max(1, most))
    return dict(op=op, batch=batch, rows=rows, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, cached=cached, ragged=ragged)


def _lengths(case, seed):
    """start and count of every sequence, drafted trees and accepted paths: host integers from the seed alone."""
    r = np.random.default_rng([seed, 77])
    B, T, L = case["batch"], case["rows"], case["cached"]
    if case["ragged"]:
        start = r.integers(L // 3, L + 1, B)
        count = r.integers((T + 1) // 2, T + 1, B)
        start[0], count[0] = L, T
    else:
        start, count = np.full(B, L), np.full(B, T)
    tree = keep = kept = None
    if case["op"] == "verify":
        parent = np.minimum(r.integers(-1, T, (B, T)), np.arange(T)[None, :] - 1)          # -1: a root; else an earlier token
        parent = np.where(r.random((B, T)) < 0.6, np.arange(T)[None, :] - 1, parent)       # mostly chains
        tree = np.zeros((B, T), np.uint64)
        for t in range(T):
            up = np.where(parent[:, t] >= 0, tree[np.arange(B), np.maximum(parent[:, t], 0)], 0).astype(np.uint64)
            tree[:, t] = up | np.uint64(1 << t)
        leaf = r.integers(0, count)                                                          # the accepted path ends here
        path = (tree[np.arange(B), leaf][:, None] >> np.arange(T, dtype=np.uint64)[None, :]) & np.uint64(1)
        kept = path.sum(1).astype(np.int64)
        keep = np.argsort(1 - path.astype(np.int64), axis=1, kind="stable")                  # the path's tokens first, ascending
        keep = np.where(np.arange(T)[None, :] < kept[:, None], keep, 0)
    return start, count, tree, keep, kept


def prepare(case, seed):
    B, T, H, G, D, P = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "dim", "page"))
    start, count, tree, keep, kept = _lengths(case, seed)
    per = -(-(case["cached"] + T) // P)                   # pages of a sequence
    pages = B * per + 3
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dev = lambda a, t=torch.int32: None if a is None else torch.from_numpy(np.ascontiguousarray(a).astype(np.int64)).to("cuda", t)  # noqa: E731
    codes = [(rand(pages, G, P, D) * 42.0).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [(torch.rand(pages, G, P, device="cuda", generator=g) + 0.5) * 0.02 for _ in range(2)]
    s = dict(case=case, k_codes=codes[0], v_codes=codes[1], k_scales=scales[0], v_scales=scales[1],
             table=torch.randperm(pages, device="cuda", generator=g)[: B * per].view(B, per).to(torch.int32).contiguous(),
             start=dev(start), count=dev(count), keep=dev(keep), kept=dev(kept), per=per,
             tree=None if tree is None else torch.from_numpy(tree.view(np.int64).copy()).cuda())
    if case["op"] in ("write", "verify"):
        # K and V as the stacked projection leaves them: q | k | v side by side in one row, with a few strong channels
        qkv = rand(B * T, (H + 2 * G) * D)
        qkv[:, ::37] *= 4.0
        s["qkv"] = qkv
    elif case["op"] == "attend":
        s["qkv"] = rand(B * T, (H + 2 * G) * D) * 1.5
    if case["op"] in ("attend", "verify"):
        s["out"] = torch.zeros(B, T, H, D, device="cuda")
    if case["op"] != "attend":
        s["k_out"], s["v_out"] = torch.zeros(B, T, G, D, device="cuda"), torch.zeros(B, T, G, D, device="cuda")
    if own:
        import mlfw_b200
        s["cache"] = mlfw_b200.KVCache(_context(), pages, P, G, D, buffers=tuple(s[k].data_ptr() for k in ("k_codes", "v_codes", "k_scales", "v_scales")))
        s["address"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
        torch.cuda.synchronize()
    return s


_CONTEXT = None


def _context():
    """The one context of the program: all its calls go to that context's stream."""
    global _CONTEXT
    if _CONTEXT is None:
        import mlfw_b200
        _CONTEXT = mlfw_b200.Context(0)
    return _CONTEXT


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case, a, cache = s["case"], s["address"], s["cache"]
    B, T, H, G, D = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "dim"))
    ld, where = (H + 2 * G) * D, (a["table"], s["per"], a["start"])
    if case["op"] in ("write", "verify"):
        cache.append(a["qkv"] + 4 * H * D, a["qkv"] + 4 * (H + G) * D, ld, ld, B, T, *where, a["count"])
    if case["op"] in ("attend", "verify"):
        cache.attention(a["qkv"], ld, B, T, H, *where, a["count"], a.get("tree"), D ** -0.5, a["out"], H * D)
    if case["op"] == "attend":
        return s["out"]
    if case["op"] == "verify":
        cache.keep(B, T, *where, a["keep"], a["kept"])
    cache.read(B, T, *where, a["kept"] if case["op"] == "verify" else a["count"], a["k_out"], a["v_out"], G * D, G * D)
    return (s["out"], s["k_out"], s["v_out"]) if case["op"] == "verify" else (s["k_out"], s["v_out"])


# ---------------------------------------------------------------- the plain form
def _places(s, count):
    """(page, row) of position start + t, and which t < rows are in use: [B, T] each."""
    P, T = s["case"]["page"], s["case"]["rows"]
    t = torch.arange(T, device="cuda")
    pos = s["start"].long()[:, None] + t
    used = t[None, :] < count.long()[:, None]
    return torch.gather(s["table"].long(), 1, pos // P), pos % P, used


def _append(s, count):
    """Codes and scales of the new rows: scale = max|x| / 127, code = floor(x / scale + 1/2), in binary64 (codes next to a tie)."""
    case = s["case"]
    B, T, H, G, D = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "dim"))
    page, row, used = _places(s, count)
    page, row = page[used], row[used]
    kv = s["qkv"].view(B, T, H + 2 * G, D)[:, :, H:].reshape(B, T, 2, G, D)[used].double()
    scale = kv.abs().amax(-1, keepdim=True) / 127.0
    codes = torch.floor(kv / scale + 0.5).clamp(-127, 127).to(torch.int8)
    scale = scale[..., 0].float()
    s["k_codes"][page, :, row], s["v_codes"][page, :, row] = codes[:, 0], codes[:, 1]
    s["k_scales"][page, :, row], s["v_scales"][page, :, row] = scale[:, 0], scale[:, 1]


def _read(s, count):
    page, row, used = _places(s, count)
    zero = torch.zeros((), device="cuda")
    return tuple(torch.where(used[..., None, None], s[c][page, :, row].float() * s[w][page, :, row][..., None], zero)
                 for c, w in (("k_codes", "k_scales"), ("v_codes", "v_scales")))


def _visible(s):
    """[B, T, L]: which positions query t of sequence b sees."""
    T, start, count = s["case"]["rows"], s["start"].long(), s["count"].long()
    L = s["per"] * s["case"]["page"]
    j = torch.arange(L, device="cuda")[None, :] - start[:, None]                 # place among the new tokens; negative: cached before
    t = torch.arange(T, device="cuda")
    if s["tree"] is None:
        seen = j[:, None, :] <= t[None, :, None]
    else:
        seen = ((s["tree"][:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1) != 0
        seen = seen | (j < 0)[:, None, :]
    return seen & (j < count[:, None])[:, None, :]


def _attend(s):
    case = s["case"]
    B, T, H, G, D = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "dim"))
    L = s["per"] * case["page"]
    whole = lambda c, w: (s[c][s["table"].long()].float() * s[w][s["table"].long()][..., None]).transpose(1, 2).reshape(B, G, L, D)  # noqa: E731
    q = s["qkv"].view(B, T, H + 2 * G, D)[:, :, :H].reshape(B, T, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    z = ((q @ whole("k_codes", "k_scales").transpose(2, 3)) * D ** -0.5).view(B, G, H // G, T, L)
    z = z.masked_fill(~_visible(s)[:, None, None], float("-inf"))
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == float("-inf"), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (p.view(B, G, -1, L) @ whole("v_codes", "v_scales")).view(B, G, H // G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D)
    t = torch.arange(T, device="cuda")
    return torch.where((t[None, :] < s["count"][:, None])[..., None, None], o, torch.zeros((), device="cuda"))


def _keep(s):
    page, row, used = _places(s, s["kept"])
    P = s["case"]["page"]
    pos = s["start"].long()[:, None] + s["keep"].long()
    from_page, from_row = torch.gather(s["table"].long(), 1, pos // P)[used], (pos % P)[used]
    page, row = page[used], row[used]
    k, v, ks, vs = (s[n][from_page, :, from_row] for n in ("k_codes", "v_codes", "k_scales", "v_scales"))
    s["k_codes"][page, :, row], s["v_codes"][page, :, row], s["k_scales"][page, :, row], s["v_scales"][page, :, row] = k, v, ks, vs


def _run_plain(s):
    op = s["case"]["op"]
    if op in ("write", "verify"):
        _append(s, s["count"])
    out = _attend(s) if op in ("attend", "verify") else None
    if op == "attend":
        return out
    if op == "verify":
        _keep(s)
        return (out,) + _read(s, s["kept"])
    return _read(s, s["count"])


# ---------------------------------------------------------------- the definition in binary64, sequence by sequence
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    B, T, H, G, D, P = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "dim", "page"))
    start, count, tree, keep, kept = _lengths(case, seed)
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    back = [torch.zeros(B, T, G, D, dtype=torch.float64, device="cuda") for _ in range(2)]
    for b in range(B):
        n, c = int(start[b]), int(count[b])
        pages = s["table"][b].long()
        first = 0 if case["op"] in ("attend", "verify") else n
        where = torch.arange(first, n + c, device="cuda")
        # [tokens, heads, dim] of this sequence, in binary64
        k, v = (s[x][pages[where // P], :, where % P].double() * s[w][pages[where // P], :, where % P].double()[..., None]
                for x, w in (("k_codes", "k_scales"), ("v_codes", "v_scales")))
        if case["op"] in ("write", "verify"):
            new = s["qkv"].view(B, T, H + 2 * G, D)[b, :c].double()
            for x, lo in ((k, H), (v, H + G)):
                rows = new[:, lo:lo + G]
                step = rows.abs().max(dim=-1, keepdim=True).values / 127
                x[n - first:] = torch.floor(rows / step + 0.5) * step
        if case["op"] in ("attend", "verify"):
            q = s["qkv"].view(B, T, H + 2 * G, D)[b, :c, :H].double()
            see = torch.ones(c, n + c, dtype=torch.bool, device="cuda")
            see[:, n:] = torch.tril(see[:, n:]) if tree is None else torch.from_numpy(
                (tree[b, :c, None] >> np.arange(c, dtype=np.uint64)[None, :]) & np.uint64(1) != 0).cuda()
            for h in range(H):
                z = (q[:, h] @ k[:, h // (H // G)].T) / D ** 0.5
                w = torch.softmax(z.masked_fill(~see, float("-inf")), dim=-1)
                out[b, :c, h] = w @ v[:, h // (H // G)]
        if case["op"] == "verify":
            m = int(kept[b])
            take = torch.from_numpy(keep[b, :m]).cuda() + n
            back[0][b, :m], back[1][b, :m] = k[take], v[take]
        elif case["op"] != "attend":
            back[0][b, :c], back[1][b, :c] = k, v
    return out if case["op"] == "attend" else (out, *back) if case["op"] == "verify" else tuple(back)


def work(case):
    """Bytes and operations of one pass.  Lengths are those of the seed-independent mean where they are uneven."""
    B, T, H, G, D, L, op = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "dim", "cached", "op"))
    if case["ragged"]:
        start, count = L + (B - 1) * (L // 3 + L) / 2, T + (B - 1) * ((T + 1) // 2 + T) / 2
    else:
        start, count = B * L, B * T
    cached, plain = 2 * G * (D + 4), 2 * G * D * 4         # bytes of a token's K and V in the cache, in binary32
    bytes_, flops = 0.0, 0.0
    if op == "write":
        bytes_ = count * (plain + cached + plain)            # the rows in, codes and scales, the values back out
    elif op == "read":
        bytes_ = count * (cached + plain)
    else:
        bytes_ = start * cached + count * H * D * 8          # the context once, queries in, results out
        bytes_ += count * (cached if op == "attend" else plain + cached)
        flops = 4.0 * H * D * (start / B + (count / B) / (2 if op == "attend" else 1)) * count
        if op == "verify":
            bytes_ += B * plain                               # at least one kept row of each sequence
    return {"bytes": float(bytes_), "flops": float(flops)}

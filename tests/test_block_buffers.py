"""Host checks of the memory GPTBlock.forward_cached holds: the Context object over a stand-in for the library that hands out
addresses and counts bytes; no GPU."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

from mlfw_b200 import B200QError, Context
from mlfw_b200.block import GPTBlock, random_block_params

D, H, FF = 128, 2, 256


class Library:
    """Every call succeeds; allocations get addresses that are never used twice."""

    def __init__(self):
        self.next, self.live = 1 << 20, {}

    def b200q_alloc(self, handle, nbytes, out):
        out._obj.value = self.next
        self.live[self.next] = nbytes
        self.next += nbytes + 256
        return 0

    def b200q_free(self, handle, ptr):
        del self.live[ptr]
        return 0

    def b200q_graph_end(self, handle, out):
        out._obj.value = 77
        return 0

    def __getattr__(self, name):
        return lambda *a: 0


@pytest.fixture
def block():
    ctx = object.__new__(Context)
    ctx.lib, ctx.device, ctx.handle, ctx._owned = Library(), 0, C.c_void_p(1), False
    blk = GPTBlock(ctx, D, H, FF, random_block_params(D, FF))
    calls = []
    cache = SimpleNamespace(heads=H, head_dim=64, append=lambda k, *a: calls.append(k), attention=lambda *a: None)
    blk.run = lambda rows, **kw: blk.forward_cached(0, 1, rows, cache, 0, 4, 0, 0, **kw)
    blk.addresses = calls                     # of K in the projections: one per call
    return blk


def per_row():
    """Bytes of one row of all intermediate buffers."""
    return D + 4 + 3 * D * 4 + 4 * D * 4 + D + 4 + FF * 4 + FF + 4


def held(blk):
    weights = sum(b.nbytes for q in (blk.qkv, blk.wo, blk.fc1, blk.fc2) for b in (q.w, q.scales, q.bias)) + 4 * D * 4
    return sum(blk.ctx.lib.live.values()) - weights


def test_prompts_of_many_lengths_share_one_set(block):
    for rows in list(range(1, 200)) + list(range(200, 0, -7)):
        t = block.run(rows)
        assert t["qkv"].shape == (rows, 3 * D) and t["n1_s"].shape == (rows,) and t["f1_q"].nbytes == rows * FF
        del t
    assert held(block) <= 200 * 1.2 * per_row()
    assert len(set(block.addresses)) < 40     # and it does not grow by a row at a time


def test_a_recorded_set_outlives_growth_and_goes_with_the_last_recording(block):
    ctx = block.ctx
    block.run(8)
    ctx.graph_begin()
    block.run(1, count=0)
    g = ctx.graph_end()
    recorded = block.addresses[-1]
    small = held(block)
    for rows in (400, 900, 3, 1200):
        block.run(rows)
    assert any(p <= recorded < p + n for p, n in ctx.lib.live.items())
    assert held(block) <= small + 1200 * 1.2 * per_row()          # the recorded set and the largest, not those between
    ctx.graph_destroy(g)
    block.run(1)
    assert not any(p <= recorded < p + n for p, n in ctx.lib.live.items())
    assert held(block) <= 1200 * 1.2 * per_row()


def test_a_recording_without_buffers_is_refused(block):
    block.run(4)
    block.ctx.graph_begin()
    with pytest.raises(B200QError, match="once before"):
        block.run(4000)
    block.run(2)
    block.ctx.graph_destroy(block.ctx.graph_end())


def test_results_keep_their_memory(block):
    t = block.run(5)
    at = t["attn"].ptr
    block.run(500)
    assert any(p <= at < p + n for p, n in block.ctx.lib.live.items())   # the caller still holds the smaller set
    del t
    assert not any(p <= at < p + n for p, n in block.ctx.lib.live.items())
    assert np.isfinite(held(block))

"""Attention over the paged 4-bit cache where a sequence's keys are shared among many workgroups and joined afterwards, with every
mask and option, against 64 bits (quant4_oracle)."""
import math

import pytest
import torch

import quant4_oracle as oracle
from test_kv4_gpu import TYPES, check, filled, ints, run

pytestmark = pytest.mark.gpu

OPTIONS = [dict(window=3000), dict(window=100), dict(one=True), dict(one=True, window=1500), dict(causal=False),
           dict(causal=False, one=True), dict(scale=-0.2), dict(scale=0.4, window=2049)]


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("kw", OPTIONS, ids=str)
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [5, 1, 3, 2], [1, 260, 40, 1], [300, 200, 40, 190]])
def test_options_over_shared_keys(dev, news, kw, t):
    lens = [6000, 4999, 40, 3001]
    cache, table = filled(lens, 2, 32, 64, 31, dev)
    run(cache, table, lens, news, 6, TYPES[t], dev, **kw)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [32, 96, 128, 192, 256])
@pytest.mark.parametrize("lens,news", [([5000], [1]), ([5000], [200]), ([4000, 2500, 900], [3, 1, 9]), ([5000, 800], [180, 64])])
def test_every_head_width_over_shared_keys(dev, lens, news, hd, t):
    """One token (four waves join a row), prompts of 32 rows a wave, and few rows."""
    cache, table = filled(lens, 2, 64, hd, 32, dev)
    run(cache, table, lens, news, 4, TYPES[t], dev)
    run(cache, table, lens, news, 4, TYPES[t], dev, window=1111, one=True)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("heads,hq", [(1, 1), (1, 40), (2, 132), (8, 8)])
def test_head_groups_over_shared_keys(dev, heads, hq, t):
    """Down to one query head a key head, and up to more of them than a tile has rows."""
    lens = [2300, 1400]
    cache, table = filled(lens, heads, 16, 64, 33, dev)
    run(cache, table, lens, [1, 1], hq, TYPES[t], dev)
    run(cache, table, lens, [7, 3], hq, TYPES[t], dev, window=700)


@pytest.mark.parametrize("one", [False, True])
def test_rows_that_see_nothing_beside_shared_keys(dev, one):
    lens, news = [0, 3, 5000, 0, 2000], [1, 5, 2, 4, 2100]
    cache, table = filled(lens, 1, 64, 64, 34, dev)
    out, lse, _ = run(cache, table, lens, news, 2, torch.float16, dev, one=one)
    for rows in (slice(0, 3), slice(8, 112)):
        assert not bool(out[rows].any()) and bool((lse[rows] == (0 if one else -math.inf)).all())


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("new", [1, 220])
@pytest.mark.parametrize("token", [3, 2600, 4700, 4999])
def test_bad_pages_and_nan_in_a_part(dev, token, new, one):
    """A page outside the cache, a key or a value that is not a number, in the first, a middle and the last part of shared keys:
    NaN in the rows that see it, the others as they should be."""
    lens, news = [5000, 3000], [new, 1]
    cache, table = filled(lens, 2, 16, 64, 35, dev)
    q = torch.randn(new + 1, 4, 64, device=dev)
    start, kv_len = ints([0, new, new + 1], dev), ints(lens, dev)
    want = oracle.attention(q, cache, table, start, kv_len, 0.125, parts=2, one=one)
    pos = torch.cat((torch.arange(5000 - new, 5000, device=dev), torch.full((1,), -1, device=dev)))  # in sequence 0

    def holds(table, seen, lse_too):  # seen: [rows, heads]
        out, lse = cache.attention(q, table, start, kv_len, lse=True, one=one)
        assert bool(out[seen].isnan().all()) and (not lse_too or bool(lse[seen].isnan().all()))
        check(torch.where(seen[..., None], want[0].float(), out), torch.where(seen, want[1].float(), lse) if lse_too else lse, want)

    nothing = torch.zeros(new + 1, 4, dtype=torch.bool, device=dev)
    holds(table, nothing, True)
    bad = table.clone()
    bad[0, token // 16] = cache.k_codes.shape[0]
    holds(bad, nothing | (pos >= token // 16 * 16)[:, None], True)
    at = (int(table[0, token // 16]), 1, token % 16)
    for scales in (cache.k_scales, cache.v_scales):
        old = scales[at].clone()
        scales[at] = math.nan
        holds(table, (pos >= token)[:, None] & (torch.arange(4, device=dev) >= 2), scales is cache.k_scales)
        scales[at] = old


def test_a_captured_call_follows_lengths_across_the_sharing(dev):
    """One captured call replayed at lengths that share the keys among workgroups in other ways, against the eager call."""
    cache, table = filled([6000, 6000, 6000], 2, 64, 64, 36, dev)
    q = torch.randn(3, 8, 64, device=dev)
    start, kv_len = ints([0, 1, 2, 3], dev), ints([1, 1, 1], dev)
    cache.attention(q, table, start, kv_len, lse=True, one=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = cache.attention(q, table, start, kv_len, lse=True, one=True)
    for lens in ([6000, 1, 0], [700, 5999, 6000], [1, 2, 3], [6000, 6000, 6000], [0, 0, 4097]):
        kv_len.copy_(ints(lens, dev))
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        again = cache.attention(q, table, start, kv_len, lse=True, one=True)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
        check(*got, oracle.attention(q, cache, table, start, kv_len, 0.125, parts=2, one=True))

"""Attention over the paged 4-bit cache where the arithmetic inside has to reach far: values of all sizes beside one another,
rows that see nothing beside rows that do, more rows than usual.  Against 64 bits (quant4_oracle)."""
import math

import pytest
import torch

import quant4_oracle as oracle
from scratchtape_amd.kv4 import KvCache4bit
from test_kv4_gpu import TYPES, check, filled, ints, run

pytestmark = pytest.mark.gpu


def place(table, page, s, at):
    """Pages and slots of the tokens `at` (a tensor) of sequence s."""
    return table[s].long()[at // page], at % page


def set_pairs(scales, table, s, at, scale, lo):
    """(scale, lo) of tokens `at` of sequence s, all heads; numbers or tensors of one a token."""
    p, slot = place(table, scales.shape[2], s, at)
    pair = torch.stack([torch.as_tensor(x, dtype=torch.float32, device=scales.device).expand(len(at)) for x in (scale, lo)], -1)
    scales[p, :, slot] = pair[:, None, :].expand(-1, scales.shape[1], -1)


# ---- values that are far from 0 and all alike --------------------------------------------------------------------

@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("length", [1, 40, 500, 6000])
@pytest.mark.parametrize("value", [3e10, 1e11, -1e25, 1e35, 3e38])
def test_constant_values_of_any_size(dev, value, length, t):
    """A vector of equal values has scale 0 and stands for lo, however large: alone, and beside ordinary vectors."""
    lens = [length, 33]
    at = torch.arange(length, device=dev)
    for which in (at, at[::3]):
        cache, table = filled(lens, 2, 32, 64, 21, dev)
        set_pairs(cache.v_scales, table, 0, which, 0.0, value)
        run(cache, table, lens, [1, 1], 4, TYPES[t], dev)
        run(cache, table, lens, [min(length, 70), 30], 4, TYPES[t], dev, one=True)


def test_constant_values_of_opposite_sign(dev):
    lens = [300, 7]
    cache, table = filled(lens, 1, 16, 128, 22, dev)
    at = torch.arange(300, device=dev)
    set_pairs(cache.v_scales, table, 0, at, 0.0, torch.where(at % 2 == 0, 1e30, -1e30))
    run(cache, table, lens, [1, 1], 2, torch.float32, dev)
    run(cache, table, lens, [40, 1], 2, torch.float32, dev)


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("signs", [1, -1])
def test_scores_that_rise_over_constant_values(dev, signs, new):
    """Weights grow by up to 2^100 from a tile to the next, over values whose components are equal; one of the last tokens' is NaN,
    and some rows see it."""
    lens = [400, 400]
    cache, table = filled(lens, 1, 16, 64, 28, dev)
    at = torch.arange(400, device=dev)
    for s in (0, 1):
        set_pairs(cache.k_scales, table, s, at, 0.0, (at // 32).float() * (70 / 8 if s else 30 / 8))  # scores of 70, 30 a tile
        set_pairs(cache.v_scales, table, s, at, 0.0, torch.where(at % 2 == 0, 1e11, signs * 1.1e11))
    q = torch.ones(2 * new, 2, 64, device=dev)
    start, kv_len = ints([0, new, 2 * new], dev), ints(lens, dev)
    out, lse = cache.attention(q, table, start, kv_len, lse=True)
    want = oracle.attention(q, cache, table, start, kv_len, 0.125, parts=2)
    check(out, lse, want)
    p, slot = place(table, 16, 0, at[390:391])
    cache.v_scales[p, :, slot] = math.nan
    out = cache.attention(q, table, start, kv_len)
    seen = torch.zeros(2 * new, dtype=torch.bool, device=dev)
    seen[max(0, new - 10):new] = True
    assert bool(out[seen].isnan().all())
    check(torch.where(seen[:, None, None], want[0].float(), out), None, want)


# ---- sums that are joined ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("exponent", [20, 45, 80])
@pytest.mark.parametrize("length,new,hd", [(300, 1, 64), (300, 40, 32), (5000, 1, 64), (5000, 200, 128)])
def test_zero_values_weigh_as_much_beside_large_ones(dev, length, new, hd, exponent):
    """Tokens whose values are all 0, in tiles and stretches of their own, beside tokens of large values."""
    lens = [length, 17]
    for run_of in (32, 1024):
        cache, table = filled(lens, 1, 32, hd, 25, dev)
        at = torch.arange(length, device=dev)
        zero = at // run_of % 2 == 0
        set_pairs(cache.v_scales, table, 0, at, torch.where(zero, 0.0, 2.0 ** exponent), torch.where(zero, 0.0, -7.0 * 2.0 ** exponent))
        run(cache, table, lens, [new, 1], 2, torch.float32, dev, spread=0.1)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("length,new", [(64, 1), (300, 33), (3000, 1), (3000, 200)])
def test_softmax1_of_low_scores_and_equal_values(dev, length, new, t):
    """Weights of 2^-43 beside the phantom's: the output is as small, not 0."""
    lens = [length, 17]
    cache, table = filled(lens, 1, 32, 64, 26, dev)
    at = torch.arange(length, device=dev)
    set_pairs(cache.k_scales, table, 0, at, 0.0, -30.0 / 8)  # scores of -30 for a q of ones
    set_pairs(cache.v_scales, table, 0, at, 0.0, 1.0)
    q = torch.ones(new + 1, 2, 64, device=dev).to(TYPES[t])
    start, kv_len = ints([0, new, new + 1], dev), ints(lens, dev)
    out, lse = cache.attention(q, table, start, kv_len, lse=True, one=True)
    check(out, lse, oracle.attention(q, cache, table, start, kv_len, 64 ** -0.5, parts=2 if t == "f32" else 1, one=True))


# ---- large values ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [30, 50, 90, 115, 120])
@pytest.mark.parametrize("length,new", [(512, 1), (512, 90), (4000, 1), (4000, 300)])
def test_small_weights_of_large_values_count(dev, length, new, exponent, t):
    """One token weighs 2^15 times as much as any other: the others together make up what only their sum shows."""
    lens = [length, 60]
    cache, table = filled(lens, 1, 32, 64, 23, dev)
    at = torch.arange(length, device=dev)
    set_pairs(cache.k_scales, table, 0, at, 0.0, torch.where(at == 3, 15 * math.log(2) / 8, 0.0))  # scores 8 times that for a q of ones
    set_pairs(cache.v_scales, table, 0, at, 2.0 ** exponent, -7 * 2.0 ** exponent)
    q = torch.ones(new + 1, 2, 64, device=dev).to(TYPES[t])
    start, kv_len = ints([0, new, new + 1], dev), ints(lens, dev)
    for one in (False, True):
        out, lse = cache.attention(q, table, start, kv_len, lse=True, one=one)
        check(out, lse, oracle.attention(q, cache, table, start, kv_len, 64 ** -0.5, parts=2 if t == "f32" else 1, one=one))


@pytest.mark.parametrize("new", [1, 150])
def test_large_values_behind_and_before_ordinary_ones(dev, new):
    """Values of 2^100 at one end of the keys and small ones at the other: rows that do not see the large ones, and rows whose
    large ones weigh next to nothing, are as exact as without them."""
    for first in (False, True):
        for small in (1.0, 2.0 ** -30):
            lens = [400, 400]
            cache, table = filled(lens, 1, 16, 64, 24, dev)
            at = torch.arange(400, device=dev)
            for s in (0, 1):
                big = (at < 64) == first if s == 0 else at >= 330  # sequence 1's last rows see large ones, the others none
                set_pairs(cache.v_scales, table, s, at, torch.where(big, 2.0 ** 100, small), torch.where(big, -7.4 * 2.0 ** 100, -7.6 * small))
                if s == 0:  # q is ones: scores of the large ones -160 nats below the others
                    set_pairs(cache.k_scales, table, s, at, 0.0, torch.where(big, -20.0, 0.0))
            q = torch.ones(2 * new, 2, 64, device=dev)
            start, kv_len = ints([0, new, 2 * new], dev), ints(lens, dev)
            out, lse = cache.attention(q, table, start, kv_len, lse=True)
            check(out, lse, oracle.attention(q, cache, table, start, kv_len, 64 ** -0.5, parts=2))


# ---- all of it at once -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("news,kw", [([1, 1], {}), ([150, 40], {}), ([1, 7], dict(one=True, window=900)), ([300, 200], dict(one=True)),
                                     ([3, 90], dict(window=65))], ids=str)
@pytest.mark.parametrize("lengths", [[400, 330], [3000, 1500]])
def test_values_of_all_sizes_at_once(dev, lengths, news, kw, t):
    """Scales and lowest values from 2^-80 to 2^123 in neighbouring tokens, some vectors zero, some of equal components, in runs and
    scattered, over scores as far apart as 30."""
    for seed in range(3):
        cache, table = filled(lengths, 2, 16, 64, 40 + seed, dev, spread=0.6)
        g = torch.Generator(device=dev).manual_seed(seed)
        for s, n in enumerate(lengths):
            at = torch.arange(n, device=dev)
            low, high = ((-80, 123), (-80, 0), (-20, 60))[(seed + s) % 3]
            exponent = torch.randint(low, high, (n,), generator=g, device=dev).float()
            if seed == 1:
                exponent = exponent[at // 48 * 48]
            scale = 2.0 ** exponent.double()
            kind = torch.randint(0, 4, (n,), generator=g, device=dev)
            lo = torch.where(kind == 0, scale * 100, -scale * 7.3)
            scale = torch.where(kind == 1, 0.0, scale)
            lo = torch.where(kind == 2, 0.0, lo).clamp(-3e38, 3e38)
            set_pairs(cache.v_scales, table, s, at, scale.float(), lo.float())
        run(cache, table, lengths, news, 4, TYPES[t], dev, seed=seed, spread=2.0, **kw)


@pytest.mark.parametrize("new", [1, 100])
def test_values_over_the_whole_range_of_f32(dev, new):
    """Vectors from -3.3e38 to 3.3e38: their scale times 15 passes f32, their values do not."""
    lens = [300, 64]
    cache, table = filled(lens, 1, 16, 64, 44, dev)
    at = torch.arange(300, device=dev)
    set_pairs(cache.v_scales, table, 0, at, 6.6e38 / 15, -3.3e38)
    run(cache, table, lens, [new, 1], 2, torch.float32, dev)
    run(cache, table, lens, [new, 1], 2, torch.float32, dev, one=True)


# ---- caches without pages, many rows -----------------------------------------------------------------------------

@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("width", [0, 3])
def test_rows_that_see_nothing_of_a_cache_without_pages(dev, width, one):
    """More rows than tokens: those at negative positions see nothing (0, and -inf or 0), the others a token that is nowhere."""
    cache = KvCache4bit.empty(0, 2, 16, 64, dev)
    table = torch.zeros(2, width, dtype=torch.int32, device=dev)
    x = torch.randn(45, 4, 64, device=dev)
    out, lse = cache.attention(x, table, ints([0, 5, 45], dev), ints([1, 20], dev), lse=True, one=one)
    nothing = torch.zeros(45, dtype=torch.bool, device=dev)
    nothing[:4] = nothing[5:25] = True
    assert not bool(out[nothing].any()) and bool((lse[nothing] == (0 if one else -math.inf)).all())
    assert bool(out[~nothing].isnan().all()) and bool(lse[~nothing].isnan().all())


def test_more_than_2_to_the_23_rows_of_heads(dev):
    """A batch of prompts whose rows and heads together pass 2^23, as a batch's append takes them."""
    seqs, length, hq, hd = 70, 2000, 64, 32
    cache, table = filled([length] * seqs, 1, 64, hd, 27, dev)
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn(seqs * length, hq, hd, generator=g, device=dev, dtype=torch.float16)
    start, kv_len = ints([length * s for s in range(seqs + 1)], dev), ints([length] * seqs, dev)
    out, lse = cache.attention(q, table, start, kv_len, lse=True, window=100)
    for s in (0, 33, seqs - 1):  # those sequences alone, some of their heads
        rows, heads = slice(length * s, length * (s + 1)), slice(0, hq, 21)
        want = oracle.attention(q[rows, heads].contiguous(), cache, table[s:s + 1], ints([0, length], dev), ints([length], dev), hd ** -0.5, window=100)
        check(out[rows, heads], lse[rows, heads], want)


# ---- appends of more and fewer tokens ----------------------------------------------------------------------------

@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("tokens", [255, 256, 257, 600])
def test_an_append_in_pieces_writes_the_same(dev, tokens, t):
    """Tokens at once and 100 at a time, whichever way the vectors are dealt out."""
    hq, heads, hd, page = 10, 5, 128, 16
    g = torch.Generator(device=dev).manual_seed(tokens)
    q, k, v = (torch.randn(tokens, h, hd, generator=g, device=dev).to(TYPES[t]) for h in (hq, heads, heads))
    pages = -(-tokens // page)
    table = torch.randperm(pages, generator=g, device=dev).to(torch.int32)[None]
    pos, seq = torch.arange(tokens, dtype=torch.int32, device=dev), torch.zeros(tokens, dtype=torch.int32, device=dev)
    freq = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], device=dev)
    caches = [KvCache4bit.empty(pages, heads, page, hd, dev) for _ in range(2)]
    whole = caches[0].append(q, k, v, seq, pos, table, inv_freq=freq, values=True)
    parts = [caches[1].append(*(x[i:i + 100] for x in (q, k, v, seq, pos)), table, inv_freq=freq, values=True) for i in range(0, tokens, 100)]
    for got, pieces in zip(whole, zip(*parts)):
        assert torch.equal(got, torch.cat(pieces))
    for (a, _), (b, _) in zip(caches[0]._buffers(), caches[1]._buffers()):
        assert torch.equal(a, b)

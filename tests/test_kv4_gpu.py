"""The paged 4-bit cache on the GPU against 64-bit arithmetic: what append writes bit for bit, attention within the error
that f32 sums allow (quant4_oracle)."""
import math

import pytest
import torch

import quant4_oracle as oracle
from scratchtape_amd import quant4
from scratchtape_amd.kv4 import KvCache4bit

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ints = lambda v, dev: torch.tensor(v, dtype=torch.int32, device=dev)


def frequencies(rot, dev):
    return torch.tensor([10000.0 ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float32, device=dev)


def poison(cache):
    """Codes of all ones, and scales that spoil whatever reads them."""
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(255)
    for t, v in ((cache.k_scales, math.nan), (cache.v_scales, math.inf)):
        t.fill_(v)


def tables(seqs, per_seq, extra, seed, dev):
    g = torch.Generator().manual_seed(seed)
    pages = seqs * per_seq + extra
    return torch.randperm(pages, generator=g)[:seqs * per_seq].view(seqs, per_seq).to(torch.int32).to(dev), pages


def filled(lens, heads, page, hd, seed, dev, extra=2, spread=1.0, shift=0.0):
    """A cache that holds normal keys and values for sequences of these lengths and poison everywhere else, and its table."""
    g = torch.Generator().manual_seed(seed)
    per = max(1, -(-max(lens) // page))
    table, pages = tables(len(lens), per, extra, seed, dev)
    cache = KvCache4bit.empty(pages, heads, page, hd, dev)
    poison(cache)
    for s, n in enumerate(lens):
        if n == 0:
            continue
        at = torch.arange(n, device=dev)
        p, slot = table[s].long()[at // page], at % page
        for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
            x = (torch.randn(n * heads, hd, generator=g) * spread + shift).to(dev)
            c, sc, lo = oracle.quantise(x)
            codes[p, :, slot] = oracle.pack(c).view(n, heads, -1)
            scales[p, :, slot] = torch.cat((sc, lo), -1).float().view(n, heads, 2)
    return cache, table


def check(got, lse, want):
    out, want_lse, tol, tol_lse = want
    rows = ~out.isnan().all(-1).all(-1)
    big = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    got, out, tol = got.double()[rows], out[rows], tol[rows]
    off = (got - out).abs()
    # Beyond its largest value a type's nearest is infinity: from half a step past it on (f16: 65504 + 16), less the error.
    past = got.isinf() & (got.sign() == out.sign()) & (out.abs() + tol >= big)
    assert bool(((off <= tol) | past).all()), float((off / tol)[~past].nan_to_num(math.inf).max())
    if lse is not None:
        same = lse.double()[rows] == want_lse[rows]  # both -inf
        off = (lse.double() - want_lse).abs()[rows]
        assert bool((same | (off <= tol_lse[rows])).all()), float((off / tol_lse[rows])[~same].max())


def run(cache, table, lens, news, hq, t, dev, seed=0, spread=1.0, scale=None, **kw):
    hd = 2 * cache.k_codes.shape[3]
    start = [0]
    for c in news:
        start.append(start[-1] + c)
    g = torch.Generator().manual_seed(seed + 77)
    q = (torch.randn(start[-1], hq, hd, generator=g) * spread).to(t).to(dev)
    q_start, kv_len = ints(start, dev), ints(lens, dev)
    out, lse = cache.attention(q, table, q_start, kv_len, scale=scale, lse=True, **kw)
    want = oracle.attention(q, cache, table, q_start, kv_len, hd ** -0.5 if scale is None else scale,
                            parts=2 if t == torch.float32 else 1, **kw)
    check(out, lse, want)
    return out, lse, want


# ---- append ----------------------------------------------------------------------------------------------------

def check_append(cache, before, q, k, v, seq, pos, table, inv_freq, interleaved, outs):
    """Every written place against the oracle, and every other place against what was there."""
    page = cache.k_codes.shape[2]
    want = [t.clone() for t in before]
    used = []
    for t, (s, p) in enumerate(zip(seq.tolist(), pos.tolist())):
        if 0 <= s < table.shape[0] and 0 <= p < table.shape[1] * page and 0 <= int(table[s, p // page]) < cache.k_codes.shape[0]:
            used.append(t)
    used = torch.tensor(used, dtype=torch.long, device=k.device)
    if not used.numel():
        for got, w in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), want):
            assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))
        return used
    at_page = table[seq[used].long(), (pos[used] // page).long()].long()
    slot = (pos[used] % page).long()
    turned = oracle.rotate(k[used], pos[used], inv_freq, interleaved).float()
    held = []
    for i, x in ((0, turned), (2, v[used].float())):
        c, scale, lo = oracle.quantise(x)
        want[i][at_page, :, slot] = oracle.pack(c)
        want[i + 1][at_page, :, slot] = torch.cat((scale, lo), -1).float()
        held.append((c * scale + lo, c * scale + lo.abs()))
    for got, w in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), want):
        assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))
    eps = torch.finfo(k.dtype).eps / 2
    if q is not None:
        y = oracle.rotate(q[used], pos[used], inv_freq, interleaved)
        size = q[used].double().abs().amax(-1, keepdim=True)
        # one rounding; the f32 rotation before it: two products, a sum, the cosine and sine
        assert bool(((outs[0][used].double() - y).abs() <= eps * y.abs() + 2.0 ** -21 * size + 2.0 ** -25).all())
    for got, (y, size) in zip(outs[1:], held):
        if got is not None:
            assert bool(((got[used].double() - y).abs() <= eps * y.abs() + 2.0 ** -23 * size + 2.0 ** -25).all())
    return used


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("heads,hq,hd,page,rot,interleaved,tokens", [
    (4, 4, 64, 16, 64, False, 1), (8, 32, 128, 64, 128, False, 70), (3, 15, 96, 32, 96, True, 33), (1, 7, 32, 16, 30, False, 50),
    (2, 2, 256, 256, 128, True, 129), (2, 10, 192, 16, 0, False, 40), (5, 5, 64, 1024, 2, True, 17),
    (3, 15, 96, 64, 96, False, 1100), (1, 4, 32, 256, 30, False, 1024)])
def test_append_is_exact(dev, heads, hq, hd, page, rot, interleaved, tokens, t):
    """Tokens of several sequences at scattered places, some of them padding or nowhere, from views of a fused projection."""
    t = TYPES[t]
    g = torch.Generator().manual_seed(tokens + hd)
    seqs, per = 5, 3
    table, pages = tables(seqs, per, 2, 1, dev)
    table[3, 1], table[4, 0] = -1, pages
    cache = KvCache4bit.empty(pages, heads, page, hd, dev)
    poison(cache)
    before = [x.clone() for x in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    places = torch.randperm((seqs + 1) * (per + 1) * page, generator=g)[:tokens]
    seq = (places // ((per + 1) * page)).to(torch.int32)
    pos = (places % ((per + 1) * page)).to(torch.int32)
    if tokens > 3:
        seq[1], pos[2], seq[3] = -1, -1, 2 ** 31 - 1
    fused = (torch.randn(tokens, (hq + 2 * heads) * hd, generator=g) * 3).to(t).to(dev)
    q, k, v = (x.unflatten(-1, (-1, hd)) for x in fused.split([hq * hd, heads * hd, heads * hd], -1))
    freq = frequencies(rot, dev) if rot else None
    seq, pos = seq.to(dev), pos.to(dev)
    outs = [torch.full((tokens, h, hd), 9.0, dtype=t, device=dev) for h in (hq, heads, heads)]
    got = cache.append(q, k, v, seq, pos, table, inv_freq=freq, interleaved=interleaved, values=True, out=outs)
    assert all(a is b for a, b in zip(got, outs))
    used = check_append(cache, before, q, k, v, seq, pos, table, freq, interleaved, outs)
    idle = torch.ones(tokens, dtype=torch.bool, device=dev)
    idle[used] = False
    for o in outs:
        assert bool((o[idle] == 9).all())


def test_append_without_queries_or_outputs(dev):
    table, pages = tables(2, 4, 1, 2, dev)
    for with_q in (False, True):
        cache = KvCache4bit.empty(pages, 2, 16, 64, dev)
        before = [x.clone() for x in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
        k, v, q = (torch.randn(6, h, 64, device=dev) for h in (2, 2, 6))
        seq, pos = ints([0, 0, 1, 1, 1, -1], dev), ints([0, 63, 16, 17, 31, 0], dev)
        got = cache.append(q if with_q else None, k, v, seq, pos, table, inv_freq=frequencies(64, dev))
        assert (got is not None) == with_q
        check_append(cache, before, q if with_q else None, k, v, seq, pos, table, frequencies(64, dev), False, [got, None, None])


def test_append_far_positions_and_odd_rows(dev):
    """Positions up to the last of a long table (angles in 64 bits), rows that are not 16-byte aligned, values that are not
    finite, and no tokens at all."""
    page, per = 1024, 2048
    table = torch.full((2, per), -1, dtype=torch.int32, device=dev)
    table[0, per - 1], table[1, 1000], table[1, 0] = 0, 1, 2
    cache = KvCache4bit.empty(3, 2, page, 128, dev)
    before = [x.clone() for x in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    seq = ints([0, 0, 1, 1, 1, 1], dev)
    pos = ints([per * page - 1, per * page - 77, 1000 * page, 1000 * page + 1023, 0, 1], dev)
    for t in TYPES.values():
        rows = torch.randn(6, 4 * 128 + 3, device=dev).to(t)
        k, v = rows[:, 1:257].unflatten(-1, (2, 128)), rows[:, 258:514].unflatten(-1, (2, 128))
        freq = frequencies(128, dev)
        got = cache.append(k, k, v, seq, pos, table, inv_freq=freq, values=True)
        check_append(cache, before, k, k, v, seq, pos, table, freq, False, got)
        cache.append(None, k[:0], v[:0], seq[:0], pos[:0], table)
    k = torch.randn(6, 2, 128, device=dev)
    k[0, 0, 5], k[1, 1, 127], k[2, 0, 64] = math.nan, math.inf, -math.inf
    got = cache.append(None, k, k, seq, pos, table, values=True)
    check_bad = [(0, 0), (1, 1), (2, 0)]
    for held in got[1:]:
        for i in range(6):
            for h in range(2):
                assert bool(held[i, h].isnan().all()) == ((i, h) in check_bad)
                assert bool(held[i, h].isnan().any()) == ((i, h) in check_bad)


# ---- attention -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 192, 256])
def test_single_tokens_of_ragged_sequences(dev, hd, t):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 500, 777]
    cache, table = filled(lens, 2, 32, hd, hd, dev)
    run(cache, table, lens, [1] * len(lens), 6, TYPES[t], dev, spread=2.0)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("heads,hq", [(1, 1), (1, 5), (3, 15), (2, 32), (1, 40), (4, 4), (7, 7)])
def test_head_groups(dev, heads, hq, t):
    lens = [40, 333, 1]
    cache, table = filled(lens, heads, 16, 64, hq, dev)
    run(cache, table, lens, [1, 1, 1], hq, TYPES[t], dev)
    run(cache, table, lens, [4, 7, 1], hq, TYPES[t], dev)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("page", [16, 32, 64, 256, 1024])
@pytest.mark.parametrize("news", [[3, 0, 9, 1], [40, 33, 64, 100], [1, 200, 0, 16]])
def test_ragged_prompts_and_pages(dev, news, page, t):
    lens = [max(c, n) for c, n in zip(news, (70, 0, 1100, 200))]
    cache, table = filled(lens, 2, page, 64, page, dev)
    run(cache, table, lens, news, 6, TYPES[t], dev, spread=1.5)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("hd", [32, 96, 128, 192, 256])
def test_prompts_of_every_head_width(dev, hd, t):
    lens, news = [150, 90], [150, 37]
    cache, table = filled(lens, 2, 16, hd, hd, dev)
    run(cache, table, lens, news, 4, TYPES[t], dev)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=7), dict(window=64), dict(window=100000), dict(causal=False),
                                dict(one=True), dict(one=True, window=33), dict(scale=0.5), dict(scale=-0.3), dict(scale=0.0)])
def test_masks_softmax1_and_scales(dev, kw, t):
    lens, news = [300, 64, 33, 5], [1, 20, 33, 5]
    cache, table = filled(lens, 2, 32, 64, 5, dev)
    run(cache, table, lens, news, 8, TYPES[t], dev, **kw)
    run(cache, table, lens, [1, 1, 1, 1], 8, TYPES[t], dev, **kw)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("one", [False, True])
def test_rows_that_see_nothing(dev, one, t):
    """Sequences without tokens, and more rows than cached tokens: 0 and -inf (softmax1: 0)."""
    lens, news = [0, 3, 20, 0], [1, 5, 2, 4]
    cache, table = filled(lens, 2, 16, 64, 3, dev)
    out, lse, _ = run(cache, table, lens, news, 4, TYPES[t], dev, one=one)
    for row in (0, 1, 2, 8, 9, 10, 11):
        assert bool((out[row] == 0).all()) and bool((lse[row] == (0 if one else -math.inf)).all())


@pytest.mark.parametrize("t", sorted(TYPES))
def test_extreme_scores_and_values(dev, t):
    """Scores far apart (weights that underflow), scores all far below and above zero, values of very different sizes, far
    from zero and constant."""
    lens = [200, 130]
    for spread, shift, big in ((6.0, 0.0, 20.0), (0.5, 30.0, 3.0), (0.5, -30.0, -3.0), (1e-3, 0.0, 1.0), (0.0, 2.0, 1.0)):
        cache, table = filled(lens, 2, 32, 64, 11, dev, spread=spread, shift=shift)
        factor = torch.tensor([2.0 ** (4 * (i % 9) - 20) for i in range(cache.v_scales.shape[2])], device=dev)
        used = torch.isfinite(cache.v_scales)
        cache.v_scales.copy_(torch.where(used, cache.v_scales * factor[:, None], cache.v_scales))
        run(cache, table, lens, [1, 1], 4, TYPES[t], dev, spread=abs(big))
        run(cache, table, lens, [64, 40], 4, TYPES[t], dev, spread=abs(big))


def test_bad_pages_and_lengths_give_nan(dev):
    """A page outside the cache, or a length past the table, spoils the rows that see it and no other; a bad page that no row
    sees spoils nothing."""
    lens, news = [100, 100, 100, 40], [1, 40, 1, 1]
    cache, table = filled(lens, 2, 16, 64, 3, dev)
    good = table.clone()
    q = torch.randn(43, 4, 64, device=dev)
    start = ints([0, 1, 41, 42, 43], dev)
    want, want_lse = cache.attention(q, good, start, ints(lens, dev), lse=True)
    for bad in (-1, cache.k_codes.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = good.clone()
        table[1, 4] = bad        # tokens 64..79: rows 5.. of sequence 1 (positions 60..99) see them
        table[3, 3:] = bad       # behind sequence 3's 40 tokens
        out, lse = cache.attention(q, table, start, ints(lens, dev), lse=True)
        seen = torch.zeros(43, dtype=torch.bool, device=dev)
        seen[1 + 4:41] = True
        assert bool(out[seen].isnan().all()) and bool(lse[seen].isnan().all())
        assert torch.equal(out[~seen], want[~seen]) and torch.equal(lse[~seen], want_lse[~seen])
        out = cache.attention(q[2:3], table[1:2], ints([0, 1], dev), ints([100], dev), window=20)
        assert bool(torch.isfinite(out).all())
    out = cache.attention(q, good, start, ints([100, 100, good.shape[1] * 16 + 1, 40], dev))
    assert bool(out[41].isnan().all()) and torch.equal(out[:41], want[:41]) and torch.equal(out[42:], want[42:])


def test_values_that_are_not_finite_spoil_only_rows_that_see_them(dev):
    lens, news = [90, 64], [30, 1]
    cache, table = filled(lens, 2, 16, 64, 4, dev)
    q = torch.randn(31, 4, 64, device=dev)
    start, kv_len = ints([0, 30, 31], dev), ints(lens, dev)
    want = cache.attention(q, table, start, kv_len)
    at = 75  # of sequence 0, head 1: rows 15.. see it
    for scales in (cache.k_scales, cache.v_scales):
        old = scales.clone()
        scales[int(table[0, at // 16]), 1, at % 16] = math.nan
        out = cache.attention(q, table, start, kv_len)
        assert bool(out[15:30, 2:].isnan().all())
        assert torch.equal(out[:15], want[:15]) and torch.equal(out[:, :2], want[:, :2]) and torch.equal(out[30], want[30])
        scales.copy_(old)
    q[3, 1, 7], q[9, 0, 0] = math.nan, math.inf
    out = cache.attention(q, table, start, kv_len)
    assert bool(out[3, 1].isnan().all()) and bool(out[9, 0].isnan().all())
    out[3, 1], out[9, 0] = want[3, 1], want[9, 0]
    assert torch.equal(out, want)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_views_and_rows_of_no_sequence(dev, t):
    """Rows at strides of their own; rows before, behind and between the sequences' are left as they were."""
    t = TYPES[t]
    lens = [50, 31]
    cache, table = filled(lens, 2, 16, 64, 6, dev)
    fused = torch.randn(12, 4 * 64 + 3, device=dev).to(t)
    for shift in (0, 3):
        q = fused[:, shift:shift + 256].unflatten(-1, (4, 64))
        start = ints([2, 5, 6], dev)
        out = torch.full((12, 4, 64), 8.0, dtype=t, device=dev)
        assert cache.attention(q, table, start, ints(lens, dev), out=out) is out
        assert bool((out[:2] == 8).all()) and bool((out[6:] == 8).all())
        # (Which kernel runs goes by rows a sequence, n / sequences, so that a call of the four rows alone may add in another order:
        # against 64 bits, not against its bits.)
        part = 2 if t == torch.float32 else 1
        check(out[2:6], None, oracle.attention(q[2:6], cache, table, ints([0, 3, 4], dev), ints(lens, dev), 64 ** -0.5, parts=part))
    assert cache.attention(fused[:0, :256].unflatten(-1, (4, 64)), table, ints([0, 0, 0], dev), ints(lens, dev)).shape == (0, 4, 64)


@pytest.mark.parametrize("t,hq,new,length", [("bf16", 8, 1, 70000), ("f32", 2, 3, 33333), ("f16", 4, 300, 9000)])
def test_long_sequences(dev, t, hq, new, length):
    lens = [length, 129]
    cache, table = filled(lens, 2, 64, 64, 9, dev)
    run(cache, table, lens, [new, 1], hq, TYPES[t], dev, spread=2.0)


def test_caches_and_tables_without_pages(dev):
    """Nothing is written; rows without tokens get 0, rows that should see one NaN."""
    x = torch.randn(2, 2, 64, device=dev)
    for pages, width in ((0, 3), (4, 0), (0, 0)):
        cache = KvCache4bit.empty(pages, 2, 16, 64, dev)
        table = torch.zeros(2, width, dtype=torch.int32, device=dev)
        outs = [torch.full_like(x, 9.0) for _ in range(3)]
        cache.append(x, x, x, ints([0, 1], dev), ints([0, 5], dev), table, inv_freq=frequencies(64, dev), values=True, out=outs)
        assert all(bool((o == 9).all()) for o in outs) and not any(bool(b.any()) for b, _ in cache._buffers())
        out, lse = cache.attention(x, table, ints([0, 1, 2], dev), ints([0, 1], dev), lse=True)
        assert not bool(out[0].any()) and bool((lse[0] == -math.inf).all())
        assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all())


def test_calls_on_two_streams_at_once(dev):
    """Calls that overlap have workspaces of their own."""
    lens = [9000, 4000]
    cache, table = filled(lens, 2, 64, 64, 15, dev)
    q = [torch.randn(2, 8, 64, device=dev) for _ in range(2)]
    args = (table, ints([0, 1, 2], dev), ints(lens, dev))
    want = [cache.attention(x, *args) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [cache.attention(q[i % 2], *args, stream=streams[i % 2]) for i in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("lens,news,heads,hq", [([3000, 9000], [1, 90], 1, 1), ([700] * 5 + [6000], [1] * 5 + [150], 2, 8)])
def test_one_sequence_of_many_rows_among_single_tokens(dev, lens, news, heads, hq, t):
    """Parts of units with far more rows than the sequences have on average."""
    cache, table = filled(lens, heads, 64, 64, 14, dev)
    run(cache, table, lens, news, hq, TYPES[t], dev, spread=2.0)


def test_many_sequences(dev):
    g = torch.Generator().manual_seed(12)
    lens = torch.randint(0, 90, (700,), generator=g).tolist()
    cache, table = filled([max(lens)] * 700, 1, 16, 32, 12, dev)
    run(cache, table, lens, [min(1 + i % 3, max(1, n)) for i, n in enumerate(lens)], 2, torch.bfloat16, dev)


def test_a_cache_past_4_gib(dev):
    """Pages whose codes and scales lie more than 2^32 bytes into their tensors."""
    hd, page, heads = 256, 1024, 8
    pages = 4300  # 4.5 GiB of codes, and as much again
    codes = [torch.empty(pages, heads, page, hd // 2, dtype=torch.uint8, device=dev) for _ in range(2)]
    scales = [torch.empty(pages, heads, page, 2, device=dev) for _ in range(2)]
    cache = KvCache4bit(codes[0], scales[0], codes[1], scales[1])
    small = KvCache4bit.empty(3, heads, page, hd, dev)
    table, low = ints([[pages - 1, 2, pages - 2]], dev), ints([[0, 1, 2]], dev)
    x = torch.randn(2500, heads, hd, device=dev)
    seq, pos = torch.zeros(2500, dtype=torch.int32, device=dev), torch.arange(2500, dtype=torch.int32, device=dev)
    for c, tab in ((cache, table), (small, low)):
        c.append(None, x, x * 2, seq, pos, tab, inv_freq=frequencies(hd, dev))
    for a, b in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), (small.k_codes, small.k_scales, small.v_codes, small.v_scales)):
        assert torch.equal(a[pages - 1], b[0]) and torch.equal(a[2], b[1]) and torch.equal(a[pages - 2][:, :452], b[2][:, :452])
    q = torch.randn(1, 16, hd, device=dev)
    got = cache.attention(q, table, ints([0, 1], dev), ints([2500], dev))
    assert torch.equal(got, small.attention(q, low, ints([0, 1], dev), ints([2500], dev)))


def test_the_same_call_twice_gives_the_same_bits(dev):
    lens = [5000, 123, 40]
    cache, table = filled(lens, 2, 64, 128, 2, dev)
    q = torch.randn(3, 16, 128, device=dev)
    first = cache.attention(q, table, ints([0, 1, 2, 3], dev), ints(lens, dev), lse=True)
    for _ in range(5):
        again = cache.attention(q, table, ints([0, 1, 2, 3], dev), ints(lens, dev), lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---- as they are used -------------------------------------------------------------------------------------------

def decode_step(x, w_qkv, w_out, cache, table, seq, pos, q_start, kv_len, freq, hq, heads, hd, **kw):
    qkv = quant4.matvec_4bit(x, *w_qkv, **kw)
    q, k, v = (y.unflatten(-1, (-1, hd)) for y in qkv.split([hq * hd, heads * hd, heads * hd], -1))
    q = cache.append(q, k, v, seq, pos, table, inv_freq=freq, **kw)
    ctx = cache.attention(q, table, q_start, kv_len, **kw)
    return quant4.matvec_4bit(ctx.flatten(1), *w_out, **kw)


def test_a_run_of_decoding_steps(dev):
    """Prompts taken in at once, then tokens one by one: every step against the same steps in 64 bits over the cache that
    the kernels filled; the prompt's rows against the same tokens appended one at a time."""
    hq, heads, hd, d, seqs = 6, 2, 64, 256, 3
    g = torch.Generator().manual_seed(31)
    w_qkv = quant4.quantize_4bit((torch.randn((hq + 2 * heads) * hd, d, generator=g) / 16).to(dev), 64)
    w_out = quant4.quantize_4bit((torch.randn(d, hq * hd, generator=g) / 16).to(dev), 128)
    freq = frequencies(hd, dev)
    table, pages = tables(seqs, 8, 1, 3, dev)
    cache = KvCache4bit.empty(pages, heads, 16, hd, dev)
    one = KvCache4bit.empty(pages, heads, 16, hd, dev)
    prompt = [20, 1, 37]
    xs = [torch.randn(n + 6, d, generator=g).to(dev) for n in prompt]
    step = lambda c, x, seq, pos, start, lens: decode_step(x, w_qkv, w_out, c, table, ints(seq, dev), ints(pos, dev),
                                                           ints(start, dev), ints(lens, dev), freq, hq, heads, hd)
    seq = [s for s in range(seqs) for _ in range(prompt[s])]
    pos = [p for s in range(seqs) for p in range(prompt[s])]
    y = step(cache, torch.cat([x[:n] for x, n in zip(xs, prompt)]), seq, pos, [0, 20, 21, 58], prompt)
    got = {(s, p): y[i] for i, (s, p) in enumerate(zip(seq, pos))}
    for i in range(6):
        lens = [n + i + 1 for n in prompt]
        y = step(cache, torch.stack([x[n + i] for x, n in zip(xs, prompt)]), [0, 1, 2], [n - 1 for n in lens], [0, 1, 2, 3], lens)
        got.update({(s, prompt[s] + i): y[s] for s in range(seqs)})
    for s in range(seqs):
        for p in range(prompt[s] + 6):
            y = step(one, xs[s][p:p + 1], [s], [p], [0] * (s + 1) + [1] * (seqs - s), [p + 1 if r == s else 0 for r in range(seqs)])
            # f32 throughout: the same sums in another order
            assert bool(((got[s, p] - y[0]).abs() <= 2e-5 * y.abs().max()).all()), (s, p)
    for a, b in zip((cache.k_codes, cache.v_codes), (one.k_codes, one.v_codes)):
        assert torch.equal(a, b)


def test_a_captured_step_follows_lengths_and_pages(dev):
    """One captured decoding step replayed as its sequences grow past where it was captured and change pages, with eager
    calls in between, equals the eager step each time; on a stream of its own it gives the same."""
    hq, heads, hd, d, seqs = 4, 2, 64, 128, 4
    g = torch.Generator().manual_seed(5)
    w_qkv = quant4.quantize_4bit((torch.randn((hq + 2 * heads) * hd, d, generator=g) / 11).to(dev), 64)
    w_out = quant4.quantize_4bit((torch.randn(d, hq * hd, generator=g) / 16).to(dev), 64)
    freq = frequencies(hd, dev)
    cache, table = filled([4000] * seqs, heads, 16, hd, 8, dev, extra=40)
    x = torch.randn(seqs, d, device=dev)
    seq, pos, kv_len = ints(range(seqs), dev), ints([0] * seqs, dev), ints([1] * seqs, dev)
    q_start = ints(range(seqs + 1), dev)
    args = (w_qkv, w_out, cache, table, seq, pos, q_start, kv_len, freq, hq, heads, hd)
    decode_step(x, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = decode_step(x, *args)
    side = torch.cuda.Stream()
    for lens in ([5, 17, 64, 1], [1000, 3999, 2, 3000], [33, 33, 33, 33], [0, 900, 3999, 12]):
        x.copy_(torch.randn(seqs, d, generator=g))
        pos.copy_(ints(lens, dev))
        kv_len.copy_(pos + 1)
        table.copy_(table.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        replayed = y.clone()
        assert torch.equal(replayed, decode_step(x, *args))
        torch.cuda.synchronize()
        other = decode_step(x, *args, stream=side)
        side.synchronize()
        assert torch.equal(replayed, other)

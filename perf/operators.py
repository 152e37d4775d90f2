"""A decoding step held in 4 bits, as cases that can be timed and compared: the plain forms in torch operations
(`own` false) and the package's entry points (`own` true).

- quantize:   f32 / f16 / bf16 weights to 4-bit codes with a scale and a minimum per group, and the values they stand for
- matvec:     a Linear layer of 4-bit weights on a few rows, with bias and ReLU
- append:     rotation of the new tokens' queries and keys by their positions, keys and values quantised into the paged cache
- attention:  ragged causal attention of the new tokens over the paged 4-bit cache

The 4-bit format: a group x (a run of `group` weights along k; a token's head vector in the cache) has lo = min x,
hi = max x, scale = (hi - lo) / 15, code = round_half_even((x - lo) * 15 / (hi - lo)), and stands for
scale * code + lo; code i is in byte i / 2, bits 4 (i % 2).  Codes are decided in 64 bits, so that a value next to
a border has one answer.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # The fused QKV projection of the d_model-256 model (768 x 256): the smallest weight worth quantising.
        dict(name="quantize_qkv_256", kind="quantize", n=768, k=256, group=64, type="f32"),
        # A large layer's weight, as a checkpoint is converted.
        dict(name="quantize_large", kind="quantize", n=16384, k=8192, group=128, type="bf16"),
        # The d_model-256 model's feed-forward layer on one token, f32 as its tape computes: latency.
        dict(name="matvec_ffn_256", kind="matvec", m=1, k=256, n=1024, group=64, type="f32", bias=True, relu=True),
        # One token through a wide layer: every weight byte read for one row.
        dict(name="matvec_wide", kind="matvec", m=1, k=8192, n=32768, group=128, type="bf16", bias=False, relu=False),
        # Sixteen sequences decoding together, a width no tile divides, small groups.
        dict(name="matvec_batch_odd", kind="matvec", m=16, k=4096, n=11003, group=32, type="f16", bias=True, relu=False),
        # One new token of each of 64 sequences.
        dict(name="append_decode", kind="append", seqs=64, longest=8192, tokens=64, hq=32, hkv=8, hd=128, rot=128,
             interleaved=False, page=64, type="bf16"),
        # The prompts of a few sequences taken in together, ragged, with padding at the end.
        dict(name="append_prompts", kind="append", seqs=9, longest=6000, tokens=8191, hq=32, hkv=8, hd=128, rot=128,
             interleaved=False, page=64, type="f16"),
        # The d_model-256 model (4 heads of 64) one token after a window of 128: the smallest attention.
        dict(name="attn_window_128", kind="attention", seqs=1, shortest=128, longest=128, new=1, hq=4, hkv=4, hd=64,
             page=16, window=0, one=False, type="f32"),
        # One sequence with a long context: few heads, the keys split over the card.
        dict(name="attn_long", kind="attention", seqs=1, shortest=131072, longest=131072, new=1, hq=32, hkv=8, hd=128,
             page=64, window=0, one=False, type="bf16"),
        # A serving batch: 64 sequences of all lengths, one token each.
        dict(name="attn_batch", kind="attention", seqs=64, shortest=200, longest=8192, new=1, hq=32, hkv=8, hd=128,
             page=64, window=0, one=False, type="bf16"),
        # A chunk of a long prompt against what is cached already.
        dict(name="attn_prompt", kind="attention", seqs=1, shortest=8192, longest=8192, new=2048, hq=32, hkv=8, hd=128,
             page=64, window=0, one=False, type="f16"),
        # Five drafted tokens of a dozen sequences checked at once, odd groups of heads, a sliding window, softmax1, f32.
        dict(name="attn_drafts_odd", kind="attention", seqs=12, shortest=700, longest=5000, new=5, hq=15, hkv=3, hd=96,
             page=16, window=1000, one=True, type="f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "matvec", "matvec", "append", "attention", "attention", "attention"])
    t = rng.choice(["f32", "f16", "bf16"])
    if kind == "quantize":
        group = rng.choice([32, 64, 128])
        return dict(kind=kind, n=_log_int(rng, 1, 8192), k=group * _log_int(rng, 1, 8192 // group), group=group, type=t)
    if kind == "matvec":
        group = rng.choice([32, 64, 128])
        return dict(kind=kind, m=_log_int(rng, 1, 32), k=group * _log_int(rng, 1, 8192 // group), n=_log_int(rng, 16, 16384),
                    group=group, type=t, bias=rng.random() < 0.5, relu=rng.random() < 0.3)
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 1, 2, 4, 5, 7, 8])
    hd = rng.choice([32, 64, 64, 96, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        longest = _log_int(rng, 16, 8192)
        seqs = _log_int(rng, 1, 64)
        return dict(kind=kind, seqs=seqs, longest=longest, tokens=_log_int(rng, 1, min(4096, seqs * longest)), hq=hq, hkv=hkv,
                    hd=hd, rot=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.4, page=page, type=t)
    while True:
        seqs, longest = _log_int(rng, 1, 96), _log_int(rng, 1, 65536)
        new = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 1024)])
        # No more keys than attn_batch has, and no more products than attn_prompt (f32 products cost more).
        if seqs * longest * hkv * hd <= 2.6e8 and seqs * new * hq * longest * hd <= (3e10 if t == "f32" else 6e10):
            return dict(kind=kind, seqs=seqs, shortest=max(1, int(longest * rng.choice([0.02, 0.5, 1.0]))), longest=longest,
                        new=min(new, longest), hq=hq, hkv=hkv, hd=hd, page=page,
                        window=rng.choice([0, 0, 0, _log_int(rng, 1, longest)]), one=rng.random() < 0.2, type=t)


# ---- inputs ---------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _group_values(x):
    """The 4-bit form of the groups in x's last dimension: codes (uint8, one each), scale and lo (float32)."""
    y = x.double()
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    d = hi - lo
    codes = torch.round((y - lo) * 15 / d)
    codes = torch.where(d > 0, codes, torch.zeros_like(codes))
    return codes.to(torch.uint8), (d / 15).float(), lo.float()


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _bell_codes(g, *shape):
    """Packed codes with the frequencies that normally distributed values give."""
    return _pack(_randn(g, *shape).mul_(2.8).add_(7.5).round_().clamp_(0, 15).to(torch.uint8))


def _lengths(case, seed):
    """Host lengths of the sequences from shortest to longest (one of each at least), reproducible from the seed."""
    r = torch.Generator().manual_seed(int(seed) * 104729 + 7)
    lens = torch.randint(case["shortest"], case["longest"] + 1, (case["seqs"],), generator=r)
    lens[0] = case["longest"]
    return [int(v) for v in lens]


def _table(g, seqs, per_seq):
    """A page table over a shuffled pool with a few pages to spare."""
    pages = seqs * per_seq + 3
    return torch.randperm(pages, generator=g, device=DEV)[:seqs * per_seq].reshape(seqs, per_seq).to(torch.int32), pages


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prepare_append(case, seed):
    g, t = _gen(seed), TYPES[case["type"]]
    n, seqs, hq, hkv, hd = case["tokens"], case["seqs"], case["hq"], case["hkv"], case["hd"]
    # As even a share of the tokens as their number allows, each sequence's at the end of some length of its own.
    share = [n // seqs + (1 if s < n % seqs else 0) for s in range(seqs)]
    r = torch.Generator().manual_seed(int(seed) * 104729 + 7)
    seq, pos = [], []
    for s, c in enumerate(share):
        start = int(torch.randint(0, case["longest"] - c + 1, (1,), generator=r)) if c < case["longest"] else 0
        seq += [s] * c
        pos += range(start, start + c)
    pad = -n % 8 if n > seqs else 0  # a batch of prompts is padded to a multiple of 8 tokens
    seq, pos, rows = seq + [-1] * pad, pos + [0] * pad, n + pad
    table, pages = _table(g, seqs, -(-case["longest"] // case["page"]))
    qkv = _randn(g, rows, (hq + 2 * hkv) * hd).mul_(1.5).to(t)  # the fused projection's output
    split = [hq * hd, hkv * hd, hkv * hd]
    q, k, v = (x.unflatten(-1, (-1, hd)) for x in qkv.split(split, -1))
    freq = torch.tensor([10000.0 ** (-2 * i / case["rot"]) for i in range(case["rot"] // 2)], dtype=torch.float32, device=DEV)
    cache = dict(k_codes=torch.zeros(pages, hkv, case["page"], hd // 2, dtype=torch.uint8, device=DEV),
                 k_scales=torch.zeros(pages, hkv, case["page"], 2, device=DEV))
    cache.update(v_codes=cache["k_codes"].clone(), v_scales=cache["k_scales"].clone())
    outs = [torch.zeros(rows, h, hd, dtype=t, device=DEV) for h in (hq, hkv, hkv)]
    return dict(case=case, q=q, k=k, v=v, seq=_ints(seq), pos=_ints(pos), table=table, freq=freq, cache=cache, outs=outs)


def _prepare_attention(case, seed):
    g, t = _gen(seed), TYPES[case["type"]]
    hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
    lens = _lengths(case, seed)
    news = [min(case["new"], n) for n in lens]
    table, pages = _table(g, len(lens), -(-max(lens) // page))
    cache = {}
    for name in "kv":
        cache[name + "_codes"] = torch.cat([_bell_codes(g, min(512, pages - p), hkv, page, hd) for p in range(0, pages, 512)])
        s = torch.rand(pages, hkv, page, 1, generator=g, device=DEV).mul_(0.1).add_(0.31)
        cache[name + "_scales"] = torch.cat((s, s * -7.5 + _randn(g, pages, hkv, page, 1).mul_(0.1)), -1)
    start = [0]
    for c in news:
        start.append(start[-1] + c)
    rows = [s * max(news) + i for s, c in enumerate(news) for i in range(c)]
    q = _randn(g, start[-1], hq, hd).mul_(2.0).to(t)
    return dict(case=case, q=q, cache=cache, table=table, q_start=_ints(start), kv_len=_ints(lens), lens=lens, news=news,
                rows=torch.tensor(rows, device=DEV))


def prepare(case, seed):
    kind = case["kind"]
    if kind == "quantize":
        return dict(case=case, x=_randn(_gen(seed), case["n"], case["k"]).mul_(0.02).to(TYPES[case["type"]]))
    if kind == "matvec":
        g = _gen(seed)
        n, k, group = case["n"], case["k"], case["group"]
        codes, scale, lo = _group_values(_randn(g, n, k // group, group).mul_(0.02))
        return dict(case=case, x=_randn(g, case["m"], k).to(TYPES[case["type"]]), codes=_pack(codes).flatten(1),
                    scales=torch.cat((scale, lo), -1), bias=_randn(g, n).mul_(0.1) if case["bias"] else None)
    return _prepare_append(case, seed) if kind == "append" else _prepare_attention(case, seed)


# ---- one pass -------------------------------------------------------------------------------------------------

def _plain_quantize(state):
    x, group = state["x"], state["case"]["group"]
    codes, scale, lo = _group_values(x.unflatten(-1, (-1, group)))
    return dict(scales=torch.cat((scale, lo), -1), values=(scale * codes + lo).flatten(1).to(x.dtype), packed=_pack(codes).flatten(1))


def _plain_matvec(state):
    x, scales = state["x"], state["scales"]
    w = _unpack(state["codes"]).unflatten(-1, (scales.shape[1], -1)).float() * scales[..., :1] + scales[..., 1:]
    y = x.float() @ w.flatten(1).t()
    if state["bias"] is not None:
        y = y + state["bias"]
    return (y.clamp(min=0) if state["case"]["relu"] else y).to(x.dtype)


def _plain_rotate(x, pos, freq, interleaved):
    """x [n, heads, hd] with its first 2 * len(freq) components rotated by pos * freq, in 64 bits."""
    x, half = x.double(), freq.numel()
    angle = (pos.double()[:, None] * freq.double())[:, None, :]
    cos, sin = angle.cos(), angle.sin()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_append(state):
    c, cache, seq, pos = state["case"], state["cache"], state["seq"], state["pos"]
    used = (seq >= 0)[:, None, None]
    # A padding token's write goes to a page that no table names.
    page = torch.where(seq >= 0, state["table"][seq.clamp(min=0).long(), (pos // c["page"]).long()].long(),
                       cache["k_codes"].shape[0] - 1)
    spare = torch.ones(cache["k_codes"].shape[0], dtype=torch.bool, device=DEV)
    spare[state["table"].long().flatten()] = False
    page = torch.where(seq >= 0, page, spare.int().argmax())
    slot = (pos % c["page"]).long()
    q_out, k_out, v_out = state["outs"]
    outs = [torch.where(used, _plain_rotate(state["q"], pos, state["freq"], c["interleaved"]).to(q_out.dtype), q_out)]
    turned = _plain_rotate(state["k"], pos, state["freq"], c["interleaved"]).float()
    for name, x, old in (("k", turned, k_out), ("v", state["v"].float(), v_out)):
        codes, scale, lo = _group_values(x)
        cache[name + "_codes"][page, :, slot] = _pack(codes)
        cache[name + "_scales"][page, :, slot] = torch.cat((scale, lo), -1)
        outs.append(torch.where(used, (scale * codes + lo).to(old.dtype), old))
    return outs


def _plain_cached(cache, name, table):
    """The named half of the cache as f32 [seqs, heads, tokens, hd], pages in the tables' order."""
    scales = cache[name + "_scales"][table]
    x = _unpack(cache[name + "_codes"][table]).float() * scales[..., :1] + scales[..., 1:]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(state):
    c, q, rows = state["case"], state["q"], state["rows"]
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    seqs, new, longest = len(state["lens"]), max(state["news"]), max(state["lens"])
    table = state["table"][:, :-(-longest // c["page"])].long()
    k, v = (_plain_cached(state["cache"], name, table)[:, :, :longest] for name in "kv")
    padded = torch.zeros(seqs * new, hq, hd, device=DEV)
    padded[rows] = q.float()
    # [seqs, hkv, new * (hq / hkv), hd]: a key head's query heads side by side.
    padded = padded.view(seqs, new, hkv, hq // hkv, hd).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, hd)
    s = (padded @ k.transpose(-1, -2).contiguous()).mul_(hd ** -0.5).view(seqs, hkv, new, hq // hkv, longest)
    start, length = state["q_start"].long(), state["kv_len"].long()
    at = (length - (start[1:] - start[:-1]))[:, None] + torch.arange(new, device=DEV)  # [seqs, new] positions
    key = torch.arange(longest, device=DEV)
    seen = (key <= at[..., None]) & (key < length[:, None, None])
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    s.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=0.0 if c["one"] else -1e30)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    if c["one"]:
        total = total + (-m).exp()
    out = (p.view(seqs, hkv, -1, longest) @ v).view(seqs, hkv, new, hq // hkv, hd) / torch.where(total > 0, total, 1.0)
    lse = (m + total.log())[..., 0]
    out, lse = (x.transpose(1, 2).reshape(seqs * new, hq, -1)[rows] for x in (out, lse.unsqueeze(-1)))
    return dict(out=out.to(q.dtype), lse=lse[..., 0])


def _own_pass(state):
    from scratchtape_amd import kv4, quant4

    c = state["case"]
    if c["kind"] == "quantize":
        _, scales, values = quant4.quantize_4bit(state["x"], c["group"], values=True)
        return dict(scales=scales, values=values)
    if c["kind"] == "matvec":
        return quant4.matvec_4bit(state["x"], state["codes"], state["scales"], bias=state["bias"], relu=c["relu"])
    cache = kv4.KvCache4bit(**state["cache"])
    if c["kind"] == "append":
        return cache.append(state["q"], state["k"], state["v"], state["seq"], state["pos"], state["table"],
                            inv_freq=state["freq"], interleaved=c["interleaved"], values=True, out=state["outs"])
    out, lse = cache.attention(state["q"], state["table"], state["q_start"], state["kv_len"], window=c["window"], one=c["one"],
                               lse=True)
    return dict(out=out, lse=lse)


def run(state):
    if own:
        return _own_pass(state)
    kind = state["case"]["kind"]
    if kind == "quantize":
        got = _plain_quantize(state)
        return dict(scales=got["scales"], values=got["values"])  # what the packed codes stand for
    return {"matvec": _plain_matvec, "append": _plain_append, "attention": _plain_attention}[kind](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _visible(case):
    """Expected (keys read per key head, query-key pairs per query head) summed over the sequences."""
    mean = case["longest"] if case["seqs"] == 1 else \
        (case["longest"] + (case["seqs"] - 1) * (case["shortest"] + case["longest"]) / 2) / case["seqs"]
    new = min(case["new"], mean)
    w = case["window"] or math.inf
    keys = min(mean, w + new - 1)
    pairs = new * (min(mean - (new - 1) / 2, w))
    return case["seqs"] * keys, case["seqs"] * pairs


def work(case):
    kind, e = case["kind"], SIZE[case["type"]]
    if kind == "quantize":
        n = case["n"] * case["k"]
        return dict(bytes=n * (2 * e + 0.5 + 8 / case["group"]), flops=8 * n)
    if kind == "matvec":
        n, m = case["n"] * case["k"], case["m"]
        return dict(bytes=n * (0.5 + 8 / case["group"]) + m * e * (case["k"] + case["n"]) + 4 * case["n"] * case["bias"],
                    flops=2 * m * n)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if kind == "append":
        per_token = 2 * (hq + 2 * hkv) * hd * e + hkv * (hd + 16) + 8
        return dict(bytes=case["tokens"] * per_token, flops=case["tokens"] * hd * (3 * (hq + hkv) + 16 * hkv))
    keys, pairs = _visible(case)
    rows = case["seqs"] * case["new"] * hq
    return dict(bytes=keys * hkv * (hd + 16) + rows * (2 * hd * e + 4), flops=4 * hd * hq * pairs)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _exact_groups(x):
    """What the 4-bit form of each group along x's last dimension stands for, its step and its lowest value."""
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    step = (high - low) / 15
    level = torch.where(step > 0, ((x - low) * 15 / (high - low)).round(), 0.0)
    return low + level * step, step, low


def _exact_attention(state):
    c = state["case"]
    hkv, share, page = c["hkv"], c["hq"] // c["hkv"], c["page"]
    outs, lses, first = [], [], 0
    for s, (length, new) in enumerate(zip(state["lens"], state["news"])):
        out = torch.empty(new, c["hq"], c["hd"], dtype=torch.float64, device=DEV)
        lse = torch.empty(new, c["hq"], dtype=torch.float64, device=DEV)
        where = torch.arange(length, device=DEV)
        pages, slots = state["table"][s].long()[where // page], where % page
        back = (length - new + torch.arange(new, device=DEV))[:, None] - where[None, :]
        hidden = (back < 0) | (back >= c["window"]) if c["window"] else back < 0
        for h in range(hkv):
            kv = []
            for name in "kv":
                raw = state["cache"][name + "_codes"][pages, h, slots]
                x = torch.empty(length, c["hd"], dtype=torch.float64, device=DEV)
                x[:, 0::2], x[:, 1::2] = (raw % 16).double(), (raw // 16).double()
                step = state["cache"][name + "_scales"][pages, h, slots].double()
                kv.append(x * step[:, :1] + step[:, 1:])
            for i in range(h * share, (h + 1) * share):
                logits = (state["q"][first:first + new, i].double() @ kv[0].t()) / math.sqrt(c["hd"])
                logits.masked_fill_(hidden, -math.inf)
                if c["one"]:  # the phantom logit 0
                    logits = torch.cat((logits, torch.zeros(new, 1, dtype=torch.float64, device=DEV)), 1)
                lse[:, i] = torch.logsumexp(logits, 1)
                out[:, i] = torch.exp(logits - lse[:, i:i + 1])[:, :length] @ kv[1]
        outs.append(out)
        lses.append(lse)
        first += new
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        values, step, low = _exact_groups(state["x"].double().view(case["n"], -1, case["group"]))
        return dict(scales=torch.cat((step, low), -1), values=values.view(case["n"], -1))
    if kind == "matvec":
        raw = state["codes"]
        w = torch.empty(case["n"], case["k"], dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = (raw % 16).double(), (raw // 16).double()
        per = state["scales"].double().repeat_interleave(case["group"], 1)
        w = w.mul_(per[..., 0]).add_(per[..., 1])
        y = torch.matmul(w, state["x"].double().t().contiguous()).t()
        if state["bias"] is not None:
            y = y + state["bias"].double()
        return torch.relu(y) if case["relu"] else y
    if kind == "attention":
        return _exact_attention(state)
    half = case["rot"] // 2
    i = torch.arange(half, device=DEV)
    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), state["pos"].double()[:, None] * state["freq"].double()[None, :])
    used = (state["seq"] >= 0)[:, None, None]
    outs = []
    for x, old in zip((state["q"], state["k"], state["v"]), state["outs"]):
        y = x.double()
        if x is not state["v"]:
            z = torch.complex(y[..., a], y[..., b]) * turn[:, None, :]
            y[..., a], y[..., b] = z.real, z.imag
        if x is not state["q"]:  # a code is decided for the f32 value, so that one next to a border has one answer
            y = _exact_groups(y.float().double())[0]
        outs.append(torch.where(used, y, old.double()))
    return outs

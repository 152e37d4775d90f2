"""A transformer layer's step in 8 bits and the norm it is trained with, as cases that can be timed and compared: the
plain forms in torch operations (`own` false) and the package's entry points (`own` true).

- norm:     the residual's addition and the root-mean-square norm; rows for training, or 8-bit rows for a product
- back:     its backward pass: the gradients of the rows and of the weight
- quantize: rows of weights (a scale per channel) or activations (a scale per token) to 8 bits
- linear:   a product of 8-bit rows and 8-bit weights with both scales, bias and ReLU
- gated:    both projections of a gated feed-forward layer in 8 bits, the activation and the product

The 8-bit format: a row x has a = max |x| and scale = f32(a / 127); value i is held as code = round_half_even(127 x / a),
decided in 64 bits, so that a value next to a border has one answer, and stands for scale * code.  The norm's 8-bit rows
are those of t = h w: the row's 1 / rms is a factor of the scale alone.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # One window of 128 tokens of the d_model-256 model in training: latency.
        dict(name="norm_window_256", kind="norm", rows=128, d=256, type="f32", weight="f32", residual=True, bits8=False),
        # 64 sequences decoding together, a wide model: the norm in front of an 8-bit product.
        dict(name="norm8_decode", kind="norm", rows=64, d=8192, type="bf16", weight="bf16", residual=True, bits8=True),
        # Prompts taken in together, a number of tokens that nothing divides.
        dict(name="norm8_prompts", kind="norm", rows=8191, d=8192, type="bf16", weight="bf16", residual=True, bits8=True),
        # The d_model-256 model's training step: 32 windows of 128 tokens.
        dict(name="back_step_256", kind="back", rows=4096, d=256, type="f32", weight="f32", dh=True),
        # A training step of a wide model, the weights kept in f32.
        dict(name="back_large", kind="back", rows=16384, d=4096, type="bf16", weight="f32", dh=True),
        # A large layer's weight, as a checkpoint is converted.
        dict(name="quantize_weight", kind="quantize", n=16384, k=8192, type="bf16"),
        # A feed-forward layer's activations on their way into its second product, odd in both sizes.
        dict(name="quantize_acts_odd", kind="quantize", n=515, k=11003, type="f16"),
        # One token through a wide layer: every weight byte read for one row.
        dict(name="linear_token", kind="linear", m=1, k=8192, n=32768, type="bf16", bias=False, relu=False),
        # 48 sequences decoding together, a width that no tile divides.
        dict(name="linear_batch_odd", kind="linear", m=48, k=4096, n=11003, type="f16", bias=True, relu=True),
        # A long prompt through a square layer: the largest product.
        dict(name="linear_prompt", kind="linear", m=8192, k=8192, n=8192, type="bf16", bias=False, relu=False),
        # Sixteen sequences decoding together, both projections.
        dict(name="gated_decode", kind="gated", m=16, k=4096, n=12288, type="bf16", act="silu", bias=False),
        # Ragged prompts, both projections.
        dict(name="gated_prompts", kind="gated", m=4095, k=4096, n=12288, type="f16", act="gelu", bias=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "back", "quantize", "linear", "linear", "linear", "gated", "gated"])
    t = rng.choice(["f32", "f16", "bf16"])
    if kind in ("norm", "back", "quantize"):
        while True:
            rows, d = _log_int(rng, 1, 32768), _log_int(rng, 1, 16384)
            if rng.random() < 0.6:
                d = -(-d // 8) * 8
            if rows * d * SIZE[t] <= 1.3e8:
                break
        if kind == "quantize":
            return dict(kind=kind, n=rows, k=d, type=t)
        w = rng.choice([t, t, "f32"])
        if kind == "back":
            return dict(kind=kind, rows=rows, d=d, type=t, weight=w, dh=rng.random() < 0.7)
        return dict(kind=kind, rows=rows, d=d, type=t, weight=w, residual=rng.random() < 0.7, bits8=rng.random() < 0.6)
    while True:
        m, k, n = _log_int(rng, 1, 8192), _log_int(rng, 16, 16384), _log_int(rng, 16, 16384)
        if rng.random() < 0.6:
            k, n = -(-k // 64) * 64, -(-n // 32) * 32
        if m * k * n <= 2e11 and n * k <= 1e8:
            break
    bias = rng.random() < 0.5
    if kind == "linear":
        return dict(kind=kind, m=m, k=k, n=n, type=t, bias=bias, relu=rng.random() < 0.3)
    return dict(kind=kind, m=m, k=k, n=-(-n // 2), type=t, act=rng.choice(["silu", "silu", "gelu"]), bias=bias)


# ---- inputs ---------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 6007 + 31)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _activations(g, rows, d):
    """Rows of a residual stream: tokens of unlike sizes, a few channels far larger than the rest."""
    x = _randn(g, rows, d).mul_(_randn(g, rows, 1).mul_(0.3).exp_())
    return x.mul_(torch.where(torch.rand(d, generator=g, device=DEV) < 0.004, 20.0, 1.0))


def _row_codes(x):
    """The 8-bit form of x's rows: codes (int8, rows 16 bytes apart or a multiple of it) and scales (float32)."""
    n, k = x.shape
    codes = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device=DEV)[:, :k]
    scales = torch.empty(n, device=DEV)
    for i in range(0, n, 4096):
        y = x[i:i + 4096].double()
        top = y.abs().amax(-1, keepdim=True)
        codes[i:i + 4096] = torch.where(top > 0, torch.round(y * 127 / top), 0.0).to(torch.int8)
        scales[i:i + 4096] = (top[:, 0] / 127).float()
    return codes, scales


def prepare(case, seed):
    g, kind, t = _gen(seed), case["kind"], TYPES[case["type"]]
    if kind == "quantize":
        return dict(case=case, x=_activations(g, case["n"], case["k"]).to(t))
    if kind in ("norm", "back"):
        rows, d = case["rows"], case["d"]
        state = dict(case=case, w=(1 + 0.2 * _randn(g, d)).to(TYPES[case["weight"]]), x=_activations(g, rows, d).to(t))
        if kind == "norm":
            state["residual"] = _activations(g, rows, d).to(t) if case["residual"] else None
        else:
            state["dy"] = _randn(g, rows, d).mul_(0.1).to(t)
            state["dh"] = _randn(g, rows, d).mul_(0.1).to(t) if case["dh"] else None
            state["rstd"] = torch.rsqrt(state["x"].double().square().mean(-1) + EPS).float()
        return state
    width = case["n"] * (2 if kind == "gated" else 1)
    x, x_scales = _row_codes(_activations(g, case["m"], case["k"]))
    w, w_scales = _row_codes(_randn(g, width, case["k"]).mul_(0.02))
    return dict(case=case, x=x, x_scales=x_scales, w=w, w_scales=w_scales, bias=_randn(g, width).mul_(0.1) if case["bias"] else None)


# ---- one pass -------------------------------------------------------------------------------------------------

def _plain_row_values(t, scale, dtype):
    """What the 8-bit form of the rows t (64 bits) stands for, scale [rows] f32."""
    top = t.abs().amax(-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(t * 127 / top), 0.0)
    return (codes.float() * scale[:, None]).to(dtype)


def _plain_quantize(state):
    x = state["x"].double()
    scales = (x.abs().amax(-1) / 127).float()
    return dict(scales=scales, values=_plain_row_values(x, scales, state["x"].dtype))


def _plain_norm(state):
    c, x = state["case"], state["x"]
    h = x if state["residual"] is None else (x.float() + state["residual"].float()).to(x.dtype)
    rstd = 1 / torch.sqrt(h.double().square().mean(-1) + EPS)
    if c["bits8"]:
        t = h.double() * state["w"].double()
        scales = (t.abs().amax(-1) * rstd / 127).float()
        return dict(h=h, scales=scales, values=_plain_row_values(t, scales, x.dtype))
    rstd = rstd.float()
    return dict(h=h, rstd=rstd, y=(h.float() * rstd[:, None] * state["w"].float()).to(x.dtype))


def _plain_back(state):
    x, rstd = state["x"], state["rstd"][:, None]
    g, xh = state["dy"].float(), state["x"].float() * rstd
    dw = (g * xh).sum(0, dtype=torch.float64).float()
    g = g * state["w"].float()
    dx = rstd * (g - xh * (g * xh).mean(-1, keepdim=True))
    if state["dh"] is not None:
        dx = dx + state["dh"].float()
    return dict(dx=dx.to(x.dtype), dw=dw)


def _plain_product(state):
    y = state["x"].float() @ state["w"].float().t()
    y = y * state["x_scales"][:, None] * state["w_scales"]
    return y if state["bias"] is None else y + state["bias"]


def _plain_linear(state):
    y = _plain_product(state)
    return (y.clamp(min=0) if state["case"]["relu"] else y).to(TYPES[state["case"]["type"]])


def _plain_gated(state):
    gate, up = _plain_product(state).chunk(2, -1)
    if state["case"]["act"] == "silu":
        act = gate / (1 + torch.exp(-gate))
    else:  # gate Phi(gate)
        act = gate * 0.5 * torch.special.erfc(gate * -math.sqrt(0.5))
    return (act * up).to(TYPES[state["case"]["type"]])


def _own_pass(state):
    from scratchtape_amd import quant8, rows

    c = state["case"]
    if c["kind"] == "norm":
        out = rows.rms_norm(state["x"], state["w"], residual=state["residual"], eps=EPS, y=not c["bits8"],
                            eight_bit=c["bits8"], values=c["bits8"])
        if c["bits8"]:
            return dict(h=out.h, scales=out.scales, values=out.values)
        return dict(h=out.h, rstd=out.rstd, y=out.y)
    if c["kind"] == "back":
        dx, dw = rows.rms_norm_backward(state["dy"], state["x"], state["rstd"], state["w"], dh=state["dh"])
        return dict(dx=dx, dw=dw)
    if c["kind"] == "quantize":
        _, scales, values = quant8.quantize_8bit(state["x"], values=True)
        return dict(scales=scales, values=values)
    operands = [state[name] for name in ("x", "x_scales", "w", "w_scales")]
    if c["kind"] == "linear":
        return quant8.matmul_8bit(*operands, bias=state["bias"], relu=c["relu"], dtype=TYPES[c["type"]])
    return quant8.gated_8bit(*operands, bias=state["bias"], activation=c["act"], dtype=TYPES[c["type"]])


def run(state):
    if own:
        return _own_pass(state)
    return {"norm": _plain_norm, "back": _plain_back, "quantize": _plain_quantize, "linear": _plain_linear,
            "gated": _plain_gated}[state["case"]["kind"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    kind, e = case["kind"], SIZE[case["type"]]
    if kind == "quantize":
        n = case["n"] * case["k"]
        return dict(bytes=n * (2 * e + 1) + 4 * case["n"], flops=4 * n)
    if kind in ("norm", "back"):
        n, w = case["rows"] * case["d"], case["d"] * SIZE[case["weight"]]
        if kind == "back":
            return dict(bytes=n * e * (3 + case["dh"]) + 4 * case["rows"] + w + 4 * case["d"], flops=11 * n)
        streams = (3 if case["residual"] else 1) * e  # x, and the residual and the sum
        return dict(bytes=n * (streams + e + case["bits8"]) + 4 * case["rows"] + w, flops=(9 if case["bits8"] else 5) * n)
    m, k, n = case["m"], case["k"], case["n"]
    width = n * (2 if kind == "gated" else 1)
    return dict(bytes=(m + width) * (k + 4) + 4 * width * case["bias"] + m * n * e, flops=2 * m * width * k)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _exact_codes(t):
    """Codes of the rows t by their distance from zero, and the rows' largest values."""
    size = t.abs()
    top = size.max(-1, keepdim=True).values
    level = torch.where(top > 0, (size * 127 / top).round(), 0.0)
    return torch.copysign(level, t), top


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        codes, top = _exact_codes(state["x"].double())
        return dict(scales=top[:, 0] / 127, values=codes * (top / 127))
    if kind in ("norm", "back"):
        x, w = state["x"].double(), state["w"].double()
        if kind == "norm":
            h = x if state["residual"] is None else x + state["residual"].double()
            kept = h.to(state["x"].dtype).double()  # the norm is of the sum as it is kept
            rms = (kept.pow(2).sum(-1, keepdim=True) / case["d"] + EPS).sqrt()
            if not case["bits8"]:
                return dict(h=h, rstd=1 / rms[:, 0], y=kept / rms * w)
            codes, top = _exact_codes(kept * w)
            scales = top / rms / 127
            return dict(h=h, scales=scales[:, 0], values=codes * scales)
        r, dy = state["rstd"].double()[:, None], state["dy"].double()
        along = ((dy * w) * x).sum(-1, keepdim=True) * r.pow(3) / case["d"]
        dx = dy * w * r - along * x
        if state["dh"] is not None:
            dx += state["dh"].double()
        return dict(dx=dx, dw=torch.einsum("rd,r->d", dy * x, state["rstd"].double()))
    w = state["w"].double().mul_(state["w_scales"].double()[:, None])
    y = torch.matmul(state["x"].double().mul_(state["x_scales"].double()[:, None]), w.t())
    if state["bias"] is not None:
        y += state["bias"].double()
    if kind == "linear":
        return y.relu() if case["relu"] else y
    gate, up = y[:, :case["n"]], y[:, case["n"]:]
    if case["act"] == "silu":
        return gate * torch.sigmoid(gate) * up
    return gate * torch.special.ndtr(gate) * up

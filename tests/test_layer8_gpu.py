"""A transformer layer's step in 8 bits on the package's operators together: norm and residual into 8-bit rows, products, the 4-bit
paged cache's attention between them, the gated feed-forward.  Each operator's output is checked against 64-bit arithmetic on its
own inputs, and a captured step against the eager one; the norm is trained through its backward."""
import pytest
import torch

from scratchtape_amd import kv4, quant8, rows
import quant4_oracle
import quant8_oracle as oracle

pytestmark = pytest.mark.gpu
T = torch.bfloat16


class Layer:
    """Width d, hq query heads over hkv key heads of 64, feed-forward width ff."""

    def __init__(self, d, hq, hkv, ff, seed, dev):
        g = torch.Generator(device=dev).manual_seed(seed)
        make = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.hq, self.hkv = hq, hkv
        self.norms = [(1 + 0.1 * make(d)).to(T) for _ in range(2)]
        self.qkv, self.out, self.both, self.down = (quant8.quantize_8bit(make(n, k) / k ** 0.5) for n, k in
                                                    (((hq + 2 * hkv) * 64, d), (d, hq * 64), (2 * ff, d), (d, ff)))
        self.freq = 10000.0 ** (-torch.arange(32, device=dev) / 32.0)

    def step(self, x, residual, cache, table, seq, pos, q_start, kv_len, keep=None):
        """The layer's two outputs: what to add to the residual stream, and the stream; `keep` takes every call's inputs and
        output."""
        say = (lambda *a: None) if keep is None else (lambda *a: keep.append(a))
        a = rows.rms_norm(x, self.norms[0], residual=residual, y=False, eight_bit=True)
        say("norm", x, residual, self.norms[0], a)
        qkv = quant8.matmul_8bit(a.codes, a.scales, *self.qkv)
        say("linear", a.codes, a.scales, *self.qkv, qkv)
        q, k, v = (t.unflatten(-1, (-1, 64)) for t in qkv.split([self.hq * 64, self.hkv * 64, self.hkv * 64], -1))
        q = cache.append(q, k, v, seq, pos, table, inv_freq=self.freq)
        attended = cache.attention(q, table, q_start, kv_len)
        codes, scales = quant8.quantize_8bit(attended.flatten(1))
        say("quantize", attended.flatten(1), codes, scales)
        y = quant8.matmul_8bit(codes, scales, *self.out)
        say("linear", codes, scales, *self.out, y)
        b = rows.rms_norm(y, self.norms[1], residual=a.h, y=False, eight_bit=True)
        say("norm", y, a.h, self.norms[1], b)
        h = quant8.gated_8bit(b.codes, b.scales, *self.both)
        say("gated", b.codes, b.scales, *self.both, h)
        codes, scales = quant8.quantize_8bit(h)
        say("quantize", h, codes, scales)
        y = quant8.matmul_8bit(codes, scales, *self.down)
        say("linear", codes, scales, *self.down, y)
        return y, b.h


def check(kind, *args):
    if kind == "norm":
        x, residual, weight, out = args
        h, rstd, _, t = oracle.norm(x, residual, weight, 1e-5)
        codes, a = oracle.quantise(t)
        assert torch.equal(out.h.cpu(), h) and torch.equal(out.codes.cpu().long(), codes)
        oracle.close(out.scales, a * rstd / 127, 2.0 ** -50 * a * rstd)
    elif kind == "quantize":
        x, codes, scales = args
        want, a = oracle.quantise(x.cpu().double())
        assert torch.equal(codes.cpu().long(), want) and torch.equal(scales.cpu(), (a / 127).float())
    else:
        *ops, got = args
        y, tol = oracle.product(*ops)
        if kind == "gated":
            n = y.shape[1] // 2
            y, tol = oracle.gated((y[:, :n], tol[:, :n]), (y[:, n:], tol[:, n:]), "silu")
        oracle.close(got, y, tol)


@pytest.mark.parametrize("d,hq,hkv,ff,seqs,new", [(256, 4, 4, 512, 1, 1), (256, 4, 2, 500, 5, 1), (512, 8, 2, 1000, 3, 40)])
def test_layer_step(dev, d, hq, hkv, ff, seqs, new):
    layer = Layer(d, hq, hkv, ff, d + ff, dev)
    g = torch.Generator(device=dev).manual_seed(1)
    page, before = 16, 37
    per = -(-(before + new) // page)
    cache = kv4.KvCache4bit.empty(seqs * per, hkv, page, 64, dev)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    table = torch.randperm(seqs * per, generator=g, device=dev).view(seqs, per).to(torch.int32)
    for first, count in ((0, before), (before, new)):  # a prompt, then the step that is checked and captured
        n = seqs * count
        x, residual = (torch.randn(n, d, generator=g, device=dev).to(T) for _ in range(2))
        plan = (ints([s for s in range(seqs) for _ in range(count)]), ints([first + i for _ in range(seqs) for i in range(count)]),
                ints([s * count for s in range(seqs + 1)]), ints([first + count] * seqs))
        call = lambda keep=None: layer.step(x, residual, cache, table, plan[0], plan[1], plan[2], plan[3], keep)
        seen = []
        y, h = call(seen)
        for args in seen:
            check(*args)
        assert bool(y.isfinite().all()) and len(seen) == 8
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for _ in range(3):
        for t in captured:
            t.zero_()
        graph.replay()
        again = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, (y, h))) and all(torch.equal(a, b) for a, b in zip(again, (y, h)))


def test_norm_trains(dev):
    """Two norms with a residual between them, forward and backward in f32, against torch's differentiation in 64 bits."""
    g = torch.Generator().manual_seed(6)
    x, r, dy = (torch.randn(40, 200, generator=g) for _ in range(3))
    w1, w2 = (torch.rand(200, generator=g) + 0.5 for _ in range(2))
    leaves = [t.double().requires_grad_() for t in (x, r, w1, w2)]
    norm = lambda h, w: h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5) * w
    h1 = leaves[0] + leaves[1]
    h2 = h1 + norm(h1, leaves[2])
    want = torch.autograd.grad((norm(h2, leaves[3]) * dy.double()).sum(), leaves)
    x, r, dy, w1, w2 = (t.to(dev) for t in (x, r, dy, w1, w2))
    a = rows.rms_norm(x, w1, residual=r)
    b = rows.rms_norm(a.y, w2, residual=a.h)
    dh2, dw2 = rows.rms_norm_backward(dy, b.h, b.rstd, w2)
    dx, dw1 = rows.rms_norm_backward(dh2, a.h, a.rstd, w1, dh=dh2)
    # chains of two norms of f32 values up to 5 and gradients up to 5: some ten roundings of 2^-24 of terms up to 25, sums of 200 and of 40
    for got, exact in ((dx, want[0]), (dx, want[1]), (dw1, want[2]), (dw2, want[3])):
        assert float((got.cpu().double() - exact).abs().max()) < 10 * 25 * 40 * 2.0 ** -24

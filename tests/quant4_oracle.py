"""The 4-bit format, the products over it and attention over a paged 4-bit cache in 64 bits, for the tests: written from
the definitions, one sequence and head at a time, on the device of its inputs."""
import math

import torch


def quantise(x):
    """Groups along x's last dimension -> codes (int64), scale and lo (float64 values of f32)."""
    y = x.double()
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    bad = ~torch.isfinite(y).all(-1, keepdim=True)
    d = hi - lo
    codes = torch.where((d > 0) & ~bad, torch.round((y - lo) * 15 / d), torch.zeros_like(y))
    nan = torch.full_like(lo, math.nan)
    return codes.nan_to_num(0).long(), torch.where(bad, nan, (d / 15).float().double()), torch.where(bad, nan, lo)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2).double()


def rotate(x, pos, inv_freq, interleaved):
    """x [n, heads, hd], its first 2 len(inv_freq) components rotated by pos * inv_freq, in 64 bits."""
    y = x.double().clone()
    half = 0 if inv_freq is None else inv_freq.numel()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        t = pos.double() * inv_freq[i].double()
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        u, v = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    return y


def cached(codes, scales, table_row, length, head):
    """The first `length` tokens of one sequence and head: codes and (scale, lo) as float64 [length, hd], [length, 2]."""
    at = torch.arange(length, device=codes.device)
    page = table_row.long()[at // codes.shape[2]]
    slot = at % codes.shape[2]
    return unpack(codes[page, head, slot]), scales[page, head, slot].double()


def attention(q, cache, table, q_start, kv_len, scale, causal=True, window=0, one=False, parts=1):
    """(out, lse, tolerance of out, tolerance of lse) for rows q [n, hq, hd]; rows of no sequence are NaN in all four.

    The tolerances follow from how the sums may be taken: scores and outputs in f32 in any order whose longest chain of
    additions is as long as the key's components and the row's keys / 32 allow (plus 64); weights rounded to 11 bits
    (parts = 1: half- and bfloat16 rows) or 22 (parts = 2: f32 rows), the codes exact; exp2 to 4 units in the last place;
    the output rounded once."""
    n, hq, hd = q.shape
    heads = cache.k_codes.shape[1]
    share = hq // heads
    dev = q.device
    out, tol = (torch.full((n, hq, hd), math.nan, dtype=torch.float64, device=dev) for _ in range(2))
    lse, tol_lse = (torch.full((n, hq), math.nan, dtype=torch.float64, device=dev) for _ in range(2))
    u = 2.0 ** -24
    half_step = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    starts, lens = q_start.tolist(), kv_len.tolist()
    for s in range(len(lens)):
        first, rows, length = starts[s], starts[s + 1] - starts[s], lens[s]
        if rows <= 0:
            continue
        at = torch.arange(length, device=dev)
        pos = length - rows + torch.arange(rows, device=dev)
        seen = at[None, :] <= pos[:, None] if causal else torch.ones(rows, length, dtype=torch.bool, device=dev)
        if window:
            seen &= at[None, :] > pos[:, None] - window
        for h in range(heads):
            kc, ks = cached(cache.k_codes, cache.k_scales, table[s], length, h)
            vc, vs = cached(cache.v_codes, cache.v_scales, table[s], length, h)
            k, v = kc * ks[:, :1] + ks[:, 1:], vc * vs[:, :1] + vs[:, 1:]
            k_abs, v_abs = kc * ks[:, :1] + ks[:, 1:].abs(), (vc + 8) * vs[:, :1] + vs[:, 1:].abs()
            for i in range(h * share, (h + 1) * share):
                qi = q[first:first + rows, i].double()
                z = (qi @ k.t()) * scale
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
                size = torch.where(seen, (qi.abs() @ k_abs.t()) * abs(scale), torch.zeros_like(z))
                top = z.amax(-1, keepdim=True) if length else torch.full((rows, 1), -math.inf, dtype=torch.float64, device=dev)
                if one:
                    top = top.clamp(min=0)
                top = torch.where(top == -math.inf, torch.zeros_like(top), top)
                p = torch.where(seen, torch.exp(z - top), torch.zeros_like(z))
                total = p.sum(-1, keepdim=True) + (torch.exp(-top) if one else 0)
                some = total > 0
                weights = torch.where(seen, p / torch.where(some, total, torch.ones_like(total)), torch.zeros_like(p))
                w_v = torch.where(weights[:, :, None] > 0, weights[:, :, None] * v[None], torch.zeros((), dtype=torch.float64, device=dev)).sum(1) \
                    if rows * length * hd < 1 << 24 else weights @ v
                out[first:first + rows, i] = w_v
                lse[first:first + rows, i] = torch.where(some, top + torch.log(total), torch.full_like(top, -math.inf))[:, 0]
                # Scores: hd products and as many additions, the f32 score's own roundings with it.
                most = size.amax(-1, keepdim=True) if length else torch.zeros_like(top)
                d_score = (hd + 64) * u * most
                chain = (64 + length / 32) * u
                rounding = 2.0 ** -11 if parts == 1 else 2.0 ** -21
                rel = 2 * d_score + chain + rounding + 2.0 ** -20
                w_abs = torch.where(weights > 0, weights, torch.zeros_like(weights)) @ v_abs.nan_to_num(0)
                tol[first:first + rows, i] = rel * w_abs + half_step * w_v.abs() + tiny
                tol_lse[first:first + rows, i] = (2 * d_score + chain + 2.0 ** -20 + 4 * u * (top.abs() + 1))[:, 0]
    return out, lse, tol, tol_lse

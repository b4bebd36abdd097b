"""The mixture of experts from its definition, in 64 bits: the router's choice on the host, products expert by expert."""
import math

import numpy as np
import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half of the smallest step


def route(z, top_k, bias=None, scores="softmax", groups=1, top_groups=1, group_best=2, renormalise=False, scale=1.0):
    """z [tokens, experts] float64 -> (chosen, weights), token by token."""
    z, out = np.asarray(z, dtype=np.float64), []
    bias = None if bias is None else np.asarray(bias, dtype=np.float64)
    for row in z:
        with np.errstate(invalid="ignore", over="ignore"):
            if scores == "sigmoid":
                s = 1.0 / (1.0 + np.exp(-row))
            else:
                top = np.nanmax(row) if not np.isnan(row).all() else 0.0
                e = np.exp(row - (0.0 if top == -np.inf else top))
                s = e / e.sum() if e.sum() != 0.0 else e
        c = s if bias is None else s + bias
        c = np.where(np.isnan(c), -np.inf, c)
        order = c if bias is not None or scores == "sigmoid" else np.where(np.isnan(row), -np.inf, row)
        size = len(c) // groups
        kept = range(groups)
        if top_groups < groups:
            worth = [np.sort(c[g * size:(g + 1) * size])[::-1][:group_best].sum() for g in range(groups)]
            kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:top_groups]
        allowed = [e for g in sorted(kept) for e in range(g * size, (g + 1) * size)]
        best = sorted(allowed, key=lambda e: (-order[e], e))[:top_k]
        w = s[best]
        if renormalise:
            w = w / (w.sum() if w.sum() != 0.0 else 1.0)
        out.append((best, w * scale))
    return np.array([b for b, _ in out], dtype=np.int32).reshape(-1, top_k), np.array([w for _, w in out]).reshape(-1, top_k)


def problem(tokens, top_k, experts, n, k, group, dtype, scales, seed, device="cuda", absent=0.0, distinct=True):
    """(x [tokens, k], chosen, q [experts, n, k] int8, scale): activations with loud channels, popular experts among the chosen."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, k, generator=g)
    x[:, ::97] *= 8.0
    q = torch.randint(-8, 8, (experts, n, k), dtype=torch.int8, generator=g)
    s = ((torch.rand(experts, n, -(-k // group), generator=g) + 0.1) * (1.0 / (4.0 * math.sqrt(max(k, 1))))).to(scales)
    liked = torch.randn(experts, generator=g)
    if distinct:
        chosen = (torch.randn(tokens, experts, generator=g) + liked).argsort(dim=1, descending=True)[:, :top_k].to(torch.int32)
    else:
        chosen = torch.randint(0, experts, (tokens, top_k), dtype=torch.int32, generator=g)
    chosen = torch.where(torch.rand(tokens, top_k, generator=g) < absent, torch.full_like(chosen, -1), chosen).contiguous()
    return x.to(dtype).to(device), chosen.to(device), q.to(device), s.to(device)


def pack(q):
    u = q.view(torch.uint8)
    return ((u[..., 0::2] & 15) | ((u[..., 1::2] & 15) << 4)).view(torch.int8).contiguous()


def values(q, s, group):
    return q.double() * s.double().repeat_interleave(group, dim=-1)[..., :q.shape[-1]]


def product(x, w, scales):
    """x [rows, k] float64 times w [n, k], and how far float32 may be off: errors of at most half a unit of each of K terms, 6 standard deviations of their
    sum; for bf16 up to 64 rows the weights take part as 136 more than they are, which is taken off: 272 times the scale to a term's size."""
    size = x.abs() @ (w.abs() + scales).T
    return x @ w.T, 6.0 * math.sqrt(max(x.shape[1], 1)) * 2.0 ** -24 * size


def spread(s, group, k, dtype):
    return 272.0 * s.double().repeat_interleave(group, dim=-1)[..., :k] if dtype == torch.bfloat16 else 0.0 * s.double().repeat_interleave(group, dim=-1)[..., :k]


def near_product(x, q, s, group, dtype, tiles):
    """x [rows, k] float64 times w = q * s of one expert, and how far the kernels' sums may be off, for checks that would see one wrong scale among hundreds.

    A product of 16 bits and four is exact in float32. The sum over a part of a group (the largest common divisor of its size and 128) has a rounding of half a unit to each
    product, of a partial sum that is no larger than the sum of sizes; such errors of all parts are independent: 6 standard deviations. Parts times their scales are added up one
    after the other, over waves and runs of K: a rounding to each. Few rows of bf16 use 136 + q, and take 136 sum(x) off: as many roundings again, of sums that are that much larger. Many
    rows of bf16 (``tiles``) are float16 numbers under a power of two of their row: each element off by 2^-39 of the row's largest at most."""
    s = s.double()
    k, part = x.shape[1], math.gcd(group, 128)
    shift = 136.0 if dtype == torch.bfloat16 and not tiles else 0.0
    want, size = torch.zeros(x.shape[0], q.shape[0], dtype=torch.float64, device=x.device), 0.0
    variance = torch.zeros_like(want)
    for c in range(0, k, part):
        a, w = x[:, c:c + part], q[:, c:c + part].double()
        scale = s[:, c // group].abs()
        part_size = a.abs() @ w.abs().T * scale
        want += a @ w.T * s[:, c // group]
        size = size + part_size
        variance += 2.0 * part * (part_size + shift * a.abs().sum(dim=1)[:, None] * scale) ** 2
    off = 6.0 * 2.0 ** -24 * (variance.sqrt() + math.sqrt(k // part + 32) * size)
    if dtype == torch.bfloat16 and tiles:
        off = off + 2.0 ** -39 * x.abs().amax(dim=1)[:, None] * (q.double().abs() * s.repeat_interleave(group, dim=-1)[:, :k].abs()).sum(dim=1) if k else off
    return want, off


def check_product(x, chosen, q, s, group, bias, y, near=False):
    """y [tokens, top_k, n] of gemm_experts against 64 bits; x [tokens, k] or [tokens, top_k, k]. ``near``: within near_product's bounds."""
    rows = (x if x.dim() == 3 else x[:, None].expand(-1, chosen.shape[1], -1)).flatten(0, 1).double()
    which, got = chosen.flatten(), y.flatten(0, 1).double()
    assert y.dtype == x.dtype and y.shape == (*chosen.shape, q.shape[1])
    none = (which < 0) | (which >= q.shape[0])
    assert not got[none].any()
    for e in torch.unique(which[~none]).tolist():
        mine = which == e
        if near:  # (a mean of 32 rows and more is always in tiles)
            want, off = near_product(rows[mine], q[e], s[e], group, x.dtype, which.numel() >= 32 * q.shape[0])
        else:
            want, off = product(rows[mine], values(q[e], s[e], group), spread(s[e], group, q.shape[2], x.dtype))
        if bias is not None:
            want, off = want + bias[e].double(), off + 2.0 ** -24 * bias[e].double().abs()
        bound = off + UNIT[x.dtype] * (want.abs() + off) + TINY[x.dtype]
        bad = (got[mine] - want).abs() - bound
        assert bool((bad <= 0).all()), (e, float(bad.max()))


def check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, group, y, near=False):
    """y of mlp against 64 bits. What the gates are off by, the rounding of h (independent errors of at most half a step, 6 standard deviations), the sums in
    float32, one rounding at the end."""
    unit, tiny, xs, inner = UNIT[x.dtype], TINY[x.dtype], x.double(), q_down.shape[2]
    want, off = torch.zeros_like(xs), torch.zeros_like(xs)
    variance = torch.zeros_like(xs)
    for e in torch.unique(chosen).tolist():
        if not 0 <= e < q_up.shape[0]:
            continue
        for j in range(chosen.shape[1]):
            who = chosen[:, j] == e
            if not who.any():
                continue
            share = weights[who, j].double()[:, None]
            tiles = chosen.numel() >= 32 * q_up.shape[0]
            if near:
                a, da = near_product(xs[who], q_up[e], s_up[e], group, x.dtype, tiles)
            else:
                a, da = product(xs[who], values(q_up[e], s_up[e], group), spread(s_up[e], group, q_up.shape[2], x.dtype))
            gate, value, dg, dv = a[:, :inner], a[:, inner:], da[:, :inner], da[:, inner:]
            silu = gate * torch.sigmoid(gate)
            h = silu * value
            # (|silu'| is below 1.1; exp and the division in float32: (|gate| + 8) units)
            dh = 1.1 * value.abs() * dg + silu.abs() * dv + 1.1 * dg * dv + (gate.abs() + 8.0) * 2.0 ** -23 * h.abs()
            w = values(q_down[e], s_down[e], group)
            if near:
                part, dpart = near_product(h, q_down[e], s_down[e], group, x.dtype, tiles)
            else:
                part, dpart = product(h, w, spread(s_down[e], group, inner, x.dtype))
            want[who] += share * part
            off[who] += share.abs() * (dpart + (dh + tiny) @ w.abs().T) + chosen.shape[1] * 2.0 ** -24 * (share * part).abs()
            variance[who] += share ** 2 * (((unit * (h.abs() + dh)) ** 2) @ (w ** 2).T)
    off += 6.0 * variance.sqrt()
    bound = off + unit * (want.abs() + off) + tiny
    assert y.dtype == x.dtype and y.shape == x.shape
    bad = (y.double() - want).abs() - bound
    assert bool((bad <= 0).all()), float(bad.max())

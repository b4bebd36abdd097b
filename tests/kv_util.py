"""Plain implementations of the paged 8-bit cache on the CPU, shared by its tests: storing in the definition's own 32-bit
operations and in 64 bits, attention in 64 bits."""
import math

import torch


def make_cache(pages, kv_heads, dim, page, seed, scale=0.02):
    """Random codes everywhere (what earlier sequences left), positive scales."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(-127, 128, (pages, kv_heads, page, dim), dtype=torch.int8, generator=g)
    v = torch.randint(-127, 128, (pages, kv_heads, dim, page), dtype=torch.int8, generator=g)
    scales = (torch.rand((pages, kv_heads, 2), generator=g) + 0.25) * scale
    return k, v, scales


def make_table(lengths, page, pages, seed, spare=1):
    """A block table with pages in any order; -1 behind a sequence's last one."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-max(n, 0) // page) for n in lengths]
    order = torch.randperm(pages, generator=g).to(torch.int32)
    assert sum(held) <= pages
    table = torch.full((len(lengths), max(held + [0]) + spare), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def starts(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)


def rotate(x, positions, cos, sin, interleaved):
    """x [tokens, heads, dim] float32 or float64; every operation in x's type."""
    if cos is None:
        return x
    pairs = cos.shape[1]
    c, s = (t[positions].to(x.dtype)[:, None] for t in (cos, sin))
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        out[..., :pairs], out[..., pairs:2 * pairs] = a * c - b * s, b * c + a * s
    return out


def append_plain(k, v, cache_k, cache_v, scales, table, lengths, counts, cos, sin, interleaved, q=None, wide=False):
    """The definition, on copies: (codes of k, codes of v, scales, q). ``wide``: in 64 bits, codes as float64."""
    real = torch.float64 if wide else torch.float32
    page = cache_k.shape[2]
    ck, cv, sc = cache_k.to(real), cache_v.transpose(2, 3).to(real), scales.to(real).clone()
    qo = None if q is None else torch.zeros(q.shape, dtype=real)
    row = 0
    for s, (length, count) in enumerate(zip(lengths, counts)):
        length, begin = max(length, 0), max(length, 0) - count
        keep = [i for i in range(count) if begin + i >= 0]
        pos = torch.tensor([begin + i for i in keep], dtype=torch.long)
        rows = torch.tensor([row + i for i in keep], dtype=torch.long)
        row += count
        if not keep:
            continue
        if qo is not None:
            qo[rows] = rotate(q[rows].to(real), pos, cos, sin, interleaved)
        for side, new in ((0, rotate(k[rows].to(real), pos, cos, sin, interleaved)), (1, v[rows].to(real))):
            codes = (ck, cv)[side]
            for number in range(int(pos[0]) // page, int(pos[-1]) // page + 1):
                if number >= table.shape[1] or not 0 <= table[s, number] < cache_k.shape[0]:
                    continue
                p, mine = int(table[s, number]), (pos // page == number).nonzero()[:, 0]
                first = int(pos[mine[0]]) % page
                amax = new[mine].abs().amax(dim=(0, 2))
                step = amax / 127 if wide else amax * torch.tensor(1.0 / 127.0, dtype=torch.float32)
                before = sc[p, :, side] if first > 0 else torch.zeros_like(step)
                after = torch.maximum(before, step)
                after = torch.where(after < 2.0 ** -100, torch.zeros_like(after), after)
                some = after > 0
                ratio = torch.where(some, before / torch.where(some, after, torch.ones_like(after)), torch.zeros_like(after))
                inverse = torch.where(some, 1.0 / torch.where(some, after, torch.ones_like(after)), torch.zeros_like(after))
                if first == 0 or bool((after != before).any()):
                    codes[p] = torch.round(codes[p] * ratio[:, None, None]).clamp(-127, 127)
                codes[p][:, first:first + len(mine)] = torch.round(new[mine] * inverse[None, :, None]).clamp(-127, 127).transpose(0, 1)
                sc[p, :, side] = after
    cv = cv.transpose(2, 3).contiguous()
    return (ck, cv, sc, qo) if wide else (ck.to(torch.int8), cv.to(torch.int8), sc, qo)


def attend_plain(q, cache_k, cache_v, scales, table, lengths, counts, scale=None, causal=True, window=0):
    """(out, sum of weight * |value|, largest sum of |q| |key| * scale a row), float64."""
    tokens, heads, dim = q.shape
    page, shared = cache_k.shape[2], heads // cache_k.shape[1]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    out, spread, size = (torch.zeros(tokens, heads, n, dtype=torch.float64) for n in (dim, dim, 1))
    row = 0
    for s, (length, count) in enumerate(zip(lengths, counts)):
        length = max(length, 0)
        ids = [int(i) for i in table[s, :-(-length // page)]] + [-1] * max(0, -(-length // page) - table.shape[1])
        there = torch.tensor([0 <= i < cache_k.shape[0] for i in ids], dtype=torch.bool).repeat_interleave(page)[:length]
        safe = torch.tensor([i if 0 <= i < cache_k.shape[0] else 0 for i in ids], dtype=torch.long)
        k = (cache_k[safe].double() * scales[safe][..., 0, None, None].double()).transpose(1, 2).reshape(-1, cache_k.shape[1], dim)[:length]
        v = (cache_v[safe].transpose(2, 3).double() * scales[safe][..., 1, None, None].double()).transpose(1, 2).reshape(-1, cache_k.shape[1], dim)[:length]
        j = torch.arange(length)
        for i in range(count):
            position = length - count + i
            seen = there.clone()
            if position < 0:
                seen[:] = False
            if causal:
                seen &= j <= position
            if window:
                seen &= j > position - window
            if not seen.any():
                continue
            for h in range(heads):
                keys, values, x = k[seen][:, h // shared], v[seen][:, h // shared], q[row + i, h].double()
                w = torch.softmax(keys @ x * scale, dim=0)
                out[row + i, h], spread[row + i, h] = w @ values, w @ values.abs()
                size[row + i, h] = (keys.abs() @ x.abs()).max() * abs(scale)
        row += count
    return out, spread, size


UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a unit in the last place, relative


def check_attention(got, want, dtype):
    """|got - want| within: the rounding of the result; weights rounded to 11 bits, relative to the sum of weight * |value| (and a quarter more for the
    sums); scores whose float32 sums are off by 2^-20 of the sum of |q| |key|, which multiplies every weight by as much; half of
    float16's smallest step."""
    out, spread, size = want
    bound = UNIT[dtype] * out.abs() + (1.25 * 2.0 ** -11 + 2.0 * 2.0 ** -20 * size) * spread + 2.0 ** -24
    off = (got.double().cpu() - out).abs()
    assert bool((off <= bound).all()), float((off - bound).max())

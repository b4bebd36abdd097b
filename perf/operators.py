"""The operators of a quantised model's attention block, for timing and for comparing results.

Four kinds of case, the last of them the other three together:

* ``linear``  -- ``quadmul_amd.gemm_grouped``: 16-bit activations times packed int4 weights with a scale per group of K.
* ``append``  -- ``quadmul_amd.kv_cache.append``: new keys and values rotated to their positions and stored in a paged
  cache of 8-bit codes with one scale per page, head and side; the queries rotated in the same call. What is stored
  comes back as values through ``kv_cache.read``.
* ``attend``  -- ``quadmul_amd.kv_cache.attend``: attention of one or more new tokens per sequence over that cache.
* ``block``   -- a whole attention block of a decode step: the query / key / value projection, ``append``, ``attend``, the
  output projection.

Layouts: codes of the keys ``[pages, kv_heads, page_size, head_dim]`` and of the values ``[pages, kv_heads, head_dim, page_size]``, int8;
scales ``[pages, kv_heads, 2]`` float32 (keys, values); ``block_table`` ``[sequences, most pages]`` int32, -1 where there is no page;
``lengths`` ``[sequences]`` int32, the tokens that a sequence has with its new ones. Tokens are packed one sequence after the other,
``query_start`` ``[sequences + 1]`` int32 says where each begins.

(N, K) of the weights are those of the repository's shape table; its (6144, 4096) is a query / key / value projection of 32 query heads and 8 heads of
keys and values, 128 wide.
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}

# (N, K) of the weight matrices in the repository's shape table and benchmark
WEIGHTS = ((4096, 4096), (11008, 4096), (4096, 11008), (12288, 4096), (8192, 8192), (10240, 8192), (28672, 4096), (6144, 4096),
           (4096, 14336), (8192, 28672))


def listed():
    return [
        # one token through the smallest weight of the table: latency, and 8 MiB of weights
        {"name": "linear_1", "kind": "linear", "m": 1, "n": 4096, "k": 4096, "group": 128, "dtype": "float16", "scales": "float16", "bias": False},
        # one token through a wide projection, the finest groups, as its scales come from the quantiser (float32)
        {"name": "linear_1_wide_g32", "kind": "linear", "m": 1, "n": 28672, "k": 4096, "group": 32, "dtype": "bfloat16", "scales": "float32", "bias": False},
        # a batch of thirteen sequences against the longest K of the table
        {"name": "linear_13_long_k", "kind": "linear", "m": 13, "n": 8192, "k": 28672, "group": 128, "dtype": "bfloat16", "scales": "bfloat16", "bias": True},
        # a prefill of 2048 tokens through an MLP's projection
        {"name": "linear_2048", "kind": "linear", "m": 2048, "n": 11008, "k": 4096, "group": 128, "dtype": "float16", "scales": "float16", "bias": False},
        # one new token for each of 64 sequences of a serving batch
        {"name": "append_decode_64", "kind": "append", "sequences": 64, "longest": 4096, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bfloat16", "interleaved": False, "mix": 1},
        # prompts of up to 2048 tokens, each of another length, one of them the continuation of a shorter one
        {"name": "append_prompts_4", "kind": "append", "sequences": 4, "longest": 3001, "new": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "float16", "interleaved": False, "mix": 2},
        # one sequence of a few hundred tokens: the smallest attention that there is, latency counts
        {"name": "attend_1_short", "kind": "attend", "sequences": 1, "longest": 517, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "float16", "window": 0, "mix": 3},
        # a serving batch of 32 sequences, lengths from one token to 8192
        {"name": "attend_32_ragged", "kind": "attend", "sequences": 32, "longest": 8192, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bfloat16", "window": 0, "mix": 4},
        # one very long sequence: the work has to be split over it
        {"name": "attend_1_long", "kind": "attend", "sequences": 1, "longest": 131072, "new": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bfloat16", "window": 0, "mix": 5},
        # chunks of four prompts, each with its own history
        {"name": "attend_prompts_4", "kind": "attend", "sequences": 4, "longest": 4096, "new": 512, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "float16", "window": 0, "mix": 6},
        # small heads without sharing, seven tokens a sequence to verify a draft, a sliding window
        {"name": "attend_16_draft", "kind": "attend", "sequences": 16, "longest": 2000, "new": 7, "heads": 12, "kv_heads": 12, "dim": 64, "page": 32,
         "dtype": "bfloat16", "window": 1024, "mix": 7},
        # the attention block of a decode step for eight sequences
        {"name": "block_8", "kind": "block", "sequences": 8, "longest": 2048, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "float16", "group": 128, "hidden": 4096, "mix": 8},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("linear", "append", "attend", "block"), weights=(4, 2, 4, 1))[0]
    dtype = rng.choice(("float16", "bfloat16"))
    if kind == "linear":
        group = rng.choice((32, 64, 128, 128, 256))
        if rng.random() < 0.6:  # a weight of the table
            n, k = rng.choice(WEIGHTS)
        else:                   # any N, any number of whole groups
            n, k = _log_between(rng, 100, 16000), group * max(1, _log_between(rng, 256, 16384) // group)
        most = max(1, min(4096, int(2048 * 11008 * 4096 / (n * k))))  # no more work than the largest listed
        return {"kind": kind, "m": _log_between(rng, 1, most) if rng.random() < 0.6 else rng.randint(1, min(most, 40)), "n": n, "k": k,
                "group": group, "dtype": dtype, "scales": rng.choice((dtype, "float32")), "bias": rng.random() < 0.3}
    heads, kv_heads, dim = rng.choice(((32, 8, 128), (32, 32, 128), (64, 8, 128), (28, 4, 128), (12, 12, 64), (16, 1, 256), (8, 2, 64)))
    page = rng.choice((16, 32, 64, 128))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "mix": rng.randrange(10, 1 << 20)}
    if kind == "block":
        kv_heads = rng.choice((8, 32))
        case |= {"heads": 32, "kv_heads": kv_heads, "dim": 128, "sequences": rng.randint(1, 40), "longest": _log_between(rng, 64, 4096 * 8 // kv_heads), "new": 1,
                 "group": rng.choice((64, 128)), "hidden": 4096}
    else:
        most = 131072 * 8 * 128 // (kv_heads * dim)  # no larger a cache than the largest listed
        longest = _log_between(rng, 16, 8192) if kind == "append" else _log_between(rng, 32, min(most, 65536))
        sequences = _log_between(rng, 1, max(1, min(128, most // longest)))
        new = 1
        if kind == "append":
            sequences = min(sequences, max(1, most // (8 * page)))
            if rng.random() < 0.5:
                new = _log_between(rng, 1, max(1, min(longest, most // (20 * sequences))))
            case["interleaved"] = rng.random() < 0.3
        else:
            if rng.random() < 0.35:
                new = _log_between(rng, 1, max(1, min(longest, 512, int(3e8 * 128 / (sequences * longest * heads * dim)))))
            case["window"] = rng.choice((0, 0, 0, _log_between(rng, 16, 4096)))
        case |= {"longest": longest, "sequences": sequences, "new": new}
    return case


def _sizes(case):
    """(tokens, of them new) of each sequence: fixed by the case. The first one is the longest; of several, one has a single token."""
    rng = random.Random(case["mix"])
    count, longest, new = case["sequences"], case["longest"], case["new"]
    total = [longest] + [_log_between(rng, max(1, longest // 32), longest) for _ in range(count - 1)]
    fresh = [new] + [new if new < 16 else rng.randint(max(1, new // 4), new) for _ in range(count - 1)]
    if count > 2:
        total[count // 2] = 1
    return [(t, min(t, f)) for t, f in zip(total, fresh)]


def _packed_weight(gen, n, k, group, dtype, scales):
    """Normal weights, quantised group by group as ``quadmul_amd.quantize_groups`` does: amax / 7, two nibbles to a byte, even k low."""
    w = (torch.randn(n, k, device="cuda", generator=gen) * (1.0 / math.sqrt(k))).to(dtype).float().reshape(n, k // group, group)
    amax = w.abs().amax(dim=2)
    q = torch.round(w * (7.0 / amax)[..., None]).clamp(-7, 7).to(torch.int16).reshape(n, k) & 15
    return (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8).view(torch.int8), (amax / 7.0).to(scales)


def _activations(gen, rows, k, dtype):
    """Normal values with a few large channels, as the hidden states of a transformer have."""
    x = torch.randn(rows, k, device="cuda", generator=gen)
    loud = torch.randint(0, k, (max(1, k // 512),), device="cuda", generator=gen)
    x[:, loud] *= 6.0
    return x.to(dtype)


def _cache(gen, case):
    """A cache that has been served from: pages in any order, more of them than are in use, every page full of codes."""
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    sizes = _sizes(case)
    held = [-(-total // page) for total, _ in sizes]
    pages = sum(held) + 7
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    ends = [sum(held[:i + 1]) for i in range(len(held))]
    table = torch.stack([torch.nn.functional.pad(order[end - n:end], (0, max(held) + 1 - n), value=-1) for n, end in zip(held, ends)])
    codes, scales = [], []
    for shape, tokens in (((pages, heads, page, dim), 2), ((pages, heads, dim, page), 3)):
        channel = torch.ones(dim, device="cuda")
        channel[torch.randint(0, dim, (3,), device="cuda", generator=gen)] = 4.0 if tokens == 2 else 1.5  # keys have louder channels
        values = torch.randn(shape, device="cuda", generator=gen).mul_(channel if tokens == 2 else channel[:, None])
        amax = values.abs().amax(dim=(2, 3))
        codes.append(torch.round(values.mul_((127.0 / amax)[..., None, None])).to(torch.int8))
        scales.append(amax / 127.0)
        del values
    return {"k": codes[0], "v": codes[1], "scales": torch.stack(scales, dim=-1).contiguous(), "table": table,
            "lengths": torch.tensor([t for t, _ in sizes], dtype=torch.int32, device="cuda"),
            "start": torch.tensor([0] + [sum(f for _, f in sizes[:i + 1]) for i in range(len(sizes))], dtype=torch.int32, device="cuda"),
            "tokens": sum(f for _, f in sizes), "most_new": max(f for _, f in sizes), "longest": max(t for t, _ in sizes)}


def _rotation(positions, dim):
    """cos and sin of the rotation, [positions, dim / 2] float32."""
    inverse = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inverse
    return angle.cos().float(), angle.sin().float()


def _touched(case, table):
    """The pages that the new tokens fall into, [pages] int32."""
    page = case["page"]
    found = [table[i, (t - f) // page:-(-t // page)] for i, (t, f) in enumerate(_sizes(case))]
    return torch.cat(found).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "linear":
        n, k = case["n"], case["k"]
        weight, scale = _packed_weight(gen, n, k, case["group"], dtype, DTYPES[case["scales"]])
        bias = (torch.randn(n, device="cuda", generator=gen) * 0.1).to(dtype) if case["bias"] else None
        return {"kind": kind, "x": _activations(gen, case["m"], k, dtype), "weight": weight, "scale": scale, "bias": bias, "group": case["group"]}
    state = {"kind": kind, "heads": case["heads"], "kv_heads": case["kv_heads"], "dim": case["dim"], "page": case["page"]} | _cache(gen, case)
    heads, kv_heads, dim, tokens = case["heads"], case["kv_heads"], case["dim"], state["tokens"]
    if kind == "attend":
        state |= {"q": torch.randn(tokens, heads, dim, device="cuda", generator=gen).mul_(1.5).to(dtype), "window": case["window"]}
        return state
    state["cos"], state["sin"] = _rotation(state["table"].shape[1] * case["page"], dim)
    state["touched"] = _touched(case, state["table"])
    state["interleaved"], state["window"] = case.get("interleaved", False), 0
    if kind == "append":  # one row of the projection's output holds a token's queries, keys and values
        state["qkv"] = _activations(gen, tokens, (heads + 2 * kv_heads) * dim, dtype)
        return state
    hidden, group = case["hidden"], case["group"]
    state |= {"x": _activations(gen, tokens, hidden, dtype), "group": group, "into": _packed_weight(gen, (heads + 2 * kv_heads) * dim, hidden, group, dtype, dtype),
              "out": _packed_weight(gen, hidden, heads * dim, group, dtype, dtype)}
    return state


def _split(state, qkv):
    """Queries, keys and values of the tokens: views of the projection's rows."""
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    q, k, v = qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1)
    return q.unflatten(1, (heads, dim)), k.unflatten(1, (kv_heads, dim)), v.unflatten(1, (kv_heads, dim))


# ---- the framework's operators -----------------------------------------------------------------------------------------------------


def _own_linear(x, weight, scale, bias, group):
    import quadmul_amd

    return quadmul_amd.gemm_grouped(x, weight, scale, group, bias)


def _own_append(s, qkv):
    from quadmul_amd import kv_cache

    q, k, v = _split(s, qkv)
    q = kv_cache.append(k, v, s["k"], s["v"], s["scales"], s["table"], s["lengths"], s["start"], q=q, cos=s["cos"], sin=s["sin"],
                        interleaved=s["interleaved"], max_query=s["most_new"])
    return q, kv_cache.read(s["k"], s["v"], s["scales"], s["touched"], qkv.dtype)


def _own_attend(s, q):
    from quadmul_amd import kv_cache

    return kv_cache.attend(q, s["k"], s["v"], s["scales"], s["table"], s["lengths"], s["start"], window=s["window"], max_query=s["most_new"],
                           max_length=s["longest"])


# ---- their plain form: elementary operations in 32 bits ----------------------------------------------------------------------------


def _plain_linear(x, weight, scale, bias, group):
    u = weight.view(torch.uint8)
    q = torch.stack((u & 15, u >> 4), dim=-1).reshape(u.shape[0], -1).float()
    q = torch.where(q > 7, q - 16, q)
    w = (q.unflatten(1, (-1, group)) * scale.float()[..., None]).flatten(1)
    y = x.float() @ w.T
    return (y if bias is None else y + bias.float()).to(x.dtype)


def _places(s):
    """(sequence, position) of every new token."""
    start, lengths = s["start"].long(), s["lengths"].long()
    token = torch.arange(s["tokens"], device="cuda")
    sequence = torch.searchsorted(start, token, right=True) - 1
    return sequence, lengths[sequence] - (start[sequence + 1] - token)


def _plain_rotate(x, cos, sin, interleaved):
    """x [tokens, heads, dim] float32, cos and sin [tokens, dim / 2]."""
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    c, s = cos[:, None], sin[:, None]
    a, b = a * c - b * s, b * c + a * s
    return torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)


def _plain_store(new, codes, scale, pages, inside, touched):
    """new [tokens, heads, dim]; codes [pages, heads, page, dim] and scale [pages, heads], written in place; inside: places in a page. The scale of a
    page that held tokens before grows with its largest value, and its codes follow; any other page begins anew."""
    lowest = torch.full((codes.shape[0],), codes.shape[2], device="cuda").scatter_reduce_(0, pages, inside, "amin")
    amax = torch.zeros_like(scale).index_reduce_(0, pages, new.abs().amax(dim=2), "amax")
    before = torch.where(lowest[touched, None] > 0, scale[touched], torch.zeros_like(scale[touched]))
    after = torch.maximum(before, amax[touched] * (1.0 / 127.0))
    ratio = torch.where(after > 0, before / after, torch.zeros_like(after))
    codes[touched] = torch.round(codes[touched].float() * ratio[..., None, None]).to(torch.int8)
    scale[touched] = after
    inverse = torch.where(scale[pages] > 0, 1.0 / scale[pages], torch.zeros_like(scale[pages]))
    codes[pages, :, inside] = torch.round(new * inverse[..., None]).clamp(-127, 127).to(torch.int8)


def _plain_append(s, qkv):
    q, k, v = _split(s, qkv)
    sequence, position = _places(s)
    pages, inside = s["table"][sequence, position // s["page"]].long(), position % s["page"]
    cos, sin, touched = s["cos"][position], s["sin"][position], s["touched"].long()
    _plain_store(_plain_rotate(k.float(), cos, sin, s["interleaved"]), s["k"], s["scales"][..., 0], pages, inside, touched)
    _plain_store(v.float(), s["v"].transpose(2, 3), s["scales"][..., 1], pages, inside, touched)
    return _plain_rotate(q.float(), cos, sin, s["interleaved"]).to(qkv.dtype), _plain_read(s, qkv.dtype)


def _plain_read(s, dtype):
    pages = s["touched"].long()
    scale = s["scales"][pages]
    k = s["k"][pages].float() * scale[..., 0, None, None]
    v = s["v"][pages].transpose(2, 3).float() * scale[..., 1, None, None]
    return k.to(dtype), v.to(dtype)


def _plain_attend(s, q):
    heads, kv_heads, dim, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    count, most, width = s["lengths"].numel(), s["most_new"], -(-s["longest"] // page)
    table = s["table"][:, :width].long().clamp(min=0)
    scale = s["scales"][table]
    k = (s["k"][table].float() * scale[..., 0, None, None]).transpose(1, 2).reshape(count, kv_heads, width * page, dim)
    v = (s["v"][table].transpose(3, 4).float() * scale[..., 1, None, None]).transpose(1, 2).reshape(count, kv_heads, width * page, dim)
    sequence, position = _places(s)
    row = torch.arange(s["tokens"], device="cuda") - s["start"].long()[sequence]
    padded = torch.zeros(count, most, heads, dim, device="cuda")
    padded[sequence, row] = q.float()
    limit = torch.full((count, most), -1, dtype=torch.long, device="cuda")
    limit[sequence, row] = position
    # [sequences, kv heads, new tokens x heads that share them, tokens]
    shared = heads // kv_heads
    grouped = padded.reshape(count, most, kv_heads, shared, dim).permute(0, 2, 1, 3, 4).reshape(count, kv_heads, most * shared, dim)
    scores = torch.matmul(grouped, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim))
    token = torch.arange(width * page, device="cuda")
    seen = token <= limit[..., None]
    if s["window"]:
        seen &= token > limit[..., None] - s["window"]
    seen = seen[:, None, :, None].expand(count, 1, most, shared, width * page).reshape(count, 1, most * shared, width * page)
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp_(scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(count, kv_heads, most, shared, dim).permute(0, 2, 1, 3, 4).reshape(count, most, heads, dim)
    return o[sequence, row].to(q.dtype)


def run(state):
    kind = state["kind"]
    linear, append, attend = (_own_linear, _own_append, _own_attend) if own else (_plain_linear, _plain_append, _plain_attend)
    if kind == "linear":
        return linear(state["x"], state["weight"], state["scale"], state["bias"], state["group"])
    if kind == "attend":
        return attend(state, state["q"])
    if kind == "append":
        q, (k, v) = append(state, state["qkv"])
        return {"q": q, "k": k, "v": v}
    q, (k, v) = append(state, linear(state["x"], *state["into"], None, state["group"]))
    return {"y": linear(attend(state, q).flatten(1), *state["out"], None, state["group"]), "k": k, "v": v}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------------------


def _exact_linear(x, weight, scale, bias, group):
    low, high = weight.to(torch.int32) & 15, (weight.to(torch.int32) >> 4) & 15
    q = torch.empty(weight.shape[0], 2 * weight.shape[1], dtype=torch.float64, device="cuda")
    q[:, 0::2], q[:, 1::2] = low, high
    q -= 16.0 * (q >= 8)
    q *= scale.double().repeat_interleave(group, dim=1)
    y = torch.zeros(x.shape[0], q.shape[0], dtype=torch.float64, device="cuda") if bias is None else bias.double().expand(x.shape[0], -1)
    return torch.addmm(y, x.double(), q.T)


def _exact_append(case, s, q, k, v):
    """Page by page. The codes and scales become float64: what is stored is what they stand for."""
    dim, page, half = case["dim"], case["page"], case["dim"] // 2
    frequency = torch.complex(s["cos"].double(), s["sin"].double())
    pair = (lambda x: (x[..., 0::2], x[..., 1::2])) if s["interleaved"] else (lambda x: (x[..., :half], x[..., half:]))

    def turned(x, positions):
        z = torch.complex(*pair(x.double())) * frequency[positions][:, None]
        out = torch.empty(*x.shape[:2], dim, dtype=torch.float64, device="cuda")
        a, b = pair(out)
        a.copy_(z.real), b.copy_(z.imag)
        return out

    queries, stored = [], {"k": [], "v": []}
    table, at = s["table"].tolist(), 0
    for i, (total, fresh) in enumerate(_sizes(case)):
        begin, rows = total - fresh, slice(at, at + fresh)
        positions = torch.arange(begin, total, device="cuda")
        queries.append(turned(q[rows], positions))
        new = {"k": turned(k[rows], positions), "v": v[rows].double()}
        at += fresh
        for number in range(begin // page, -(-total // page)):
            name = table[i][number]
            lo, hi = max(begin, number * page), min(total, (number + 1) * page)
            for side, which in (("k", 0), ("v", 1)):
                codes = (s["k"][name] if side == "k" else s["v"][name].transpose(1, 2)).double()  # [heads, page, dim]
                here = new[side][lo - begin:hi - begin].transpose(0, 1)
                old = s["scales"][name, :, which].double() if lo > number * page else torch.zeros(case["kv_heads"], dtype=torch.float64, device="cuda")
                scale = torch.maximum(old, here.abs().amax(dim=(1, 2)) / 127)[:, None, None]
                codes = torch.round(codes * (old[:, None, None] / scale))
                codes[:, lo % page:lo % page + hi - lo] = torch.round(here / scale).clamp(-127, 127)
                stored[side].append(codes * scale)
    return torch.cat(queries), torch.stack(stored["k"]), torch.stack(stored["v"])


def _exact_attend(case, s, q, replaced=None):
    """Head by head. ``replaced``: the values of the pages in ``touched``, where they are not what the cache holds."""
    dim, page, shared = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    out, at, taken = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0, 0
    for i, (total, fresh) in enumerate(_sizes(case)):
        held = -(-total // page)
        pages = s["table"][i, :held].long()
        scale = s["scales"][pages].double()
        k = s["k"][pages].double() * scale[..., 0, None, None]
        v = s["v"][pages].transpose(2, 3).double() * scale[..., 1, None, None]
        if replaced is not None:
            last = held - (total - fresh) // page
            k[held - last:], v[held - last:] = replaced[0][taken:taken + last], replaced[1][taken:taken + last]
            taken += last
        j = torch.arange(total, device="cuda")
        limit = torch.arange(total - fresh, total, device="cuda")[:, None]
        hidden = (j > limit) | ((j <= limit - s["window"]) if s["window"] else torch.zeros_like(j > limit))
        for h in range(case["heads"]):
            keys, values = (x[:, h // shared].reshape(held * page, dim)[:total] for x in (k, v))
            scores = (q[at:at + fresh, h].double() @ keys.T) / math.sqrt(dim)
            weights = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=1)
            out[at:at + fresh, h] = weights @ values
        at += fresh
    return out


def exact(case, seed):
    """What ``run`` returns, in 64 bits from the same inputs."""
    s, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        return _exact_linear(s["x"], s["weight"], s["scale"], s["bias"], s["group"])
    if kind == "attend":
        return _exact_attend(case, s, s["q"])
    if kind == "append":
        return dict(zip("qkv", _exact_append(case, s, *_split(s, s["qkv"]))))
    q, k, v = _exact_append(case, s, *_split(s, _exact_linear(s["x"], *s["into"], None, s["group"])))
    y = _exact_linear(_exact_attend(case, s, q, (k, v)).flatten(1), *s["out"], None, s["group"])
    return {"y": y, "k": k, "v": v}


def work(case):
    def linear(m, n, k, group, scale_bytes, bias=False):
        return n * k / 2 + n * (k // group) * scale_bytes + 2 * m * (k + n) + (2 * n if bias else 0), 2 * m * n * k

    kind = case["kind"]
    if kind == "linear":
        b, f = linear(case["m"], case["n"], case["k"], case["group"], 4 if case["scales"] == "float32" else 2, case["bias"])
        return {"bytes": b, "flops": f}
    heads, kv_heads, dim, page, sizes = case["heads"], case["kv_heads"], case["dim"], case["page"], _sizes(case)
    tokens = sum(f for _, f in sizes)
    touched = sum(-(-t // page) - (t - f) // page for t, f in sizes)
    # the new tokens in, the queries out and one byte for each value stored; then the pages that they are in, read back
    append = 2 * tokens * (2 * heads + 2 * kv_heads) * dim + 4 * tokens * dim + 2 * tokens * kv_heads * dim + touched * kv_heads * (6 * page * dim + 24)
    window = case.get("window", 0)
    seen = [min(t, f - 1 + window) if window else t for t, f in sizes]  # tokens that some new token attends to
    pairs = sum(sum(min(p + 1, window) if window else p + 1 for p in range(t - f, t)) for t, f in sizes)
    attend = 2 * kv_heads * dim * sum(seen) + 8 * kv_heads * sum(-(-t // page) for t in seen) + 4 * tokens * heads * dim
    if kind == "append":
        return {"bytes": append, "flops": 3 * tokens * (heads + kv_heads) * dim}
    if kind == "attend":
        return {"bytes": attend, "flops": 4 * pairs * heads * dim}
    parts = [linear(tokens, (heads + 2 * kv_heads) * dim, case["hidden"], case["group"], 2), linear(tokens, case["hidden"], heads * dim, case["group"], 2)]
    return {"bytes": append + attend + sum(b for b, _ in parts), "flops": 4 * pairs * heads * dim + sum(f for _, f in parts)}

"""The operators of a model whose MLP is a choice of experts, for timing and for comparing results.

Four kinds of case, the last of them the first and the third together:

* ``route``  -- ``quadmul_amd.moe.route``: each token's experts and their weights, from the router's logits.
* ``linear`` -- ``quadmul_amd.moe.gemm_experts``: each token's row (or a row for each of its experts) times the packed int4
  weights of each of its experts.
* ``mlp``    -- ``quadmul_amd.moe.mlp``: the gated MLP of each token's experts, their outputs added up by weight.
* ``layer``  -- ``route`` and ``mlp`` one after the other, from a batch's logits and hidden states.

Layouts: logits ``[tokens, experts]``; a token's experts ``[tokens, top_k]`` int32 (-1: an expert that this GPU does not hold) and their weights, float32;
packed weights ``[experts, n, k / 2]`` int8, two nibbles to a byte, with a scale per group of k ``[experts, n, ceil(k / group)]``. Rows 0 to inner - 1 of the
first matrix of an MLP are the gate, as many further ones what it is multiplied with.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}

# (hidden, inner) of experts: few wide ones, with the sizes of the repository's shape table, and many narrow ones
WIDE = ((4096, 14336), (4096, 11008))
NARROW = ((2048, 1024), (2048, 1408), (4096, 1024), (1024, 512), (2880, 2880), (2080, 1376))


def listed():
    return [
        # one token's choice in a decode step: latency
        {"name": "route_1", "kind": "route", "tokens": 1, "experts": 64, "top_k": 6, "scores": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_best": 1,
         "renormalise": False, "scale": 1.0, "logits": "bfloat16"},
        # a serving batch; sigmoid scores, a bias that balances the experts' loads, half of the groups
        {"name": "route_64_groups", "kind": "route", "tokens": 64, "experts": 256, "top_k": 8, "scores": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_best": 2,
         "renormalise": True, "scale": 2.5, "logits": "float32"},
        # a prefill of 16384 tokens
        {"name": "route_16384", "kind": "route", "tokens": 16384, "experts": 128, "top_k": 8, "scores": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_best": 1,
         "renormalise": True, "scale": 1.0, "logits": "float32"},
        # five tokens through one matrix of a few wide experts
        {"name": "linear_5_wide", "kind": "linear", "tokens": 5, "top_k": 2, "experts": 8, "all_experts": 8, "n": 11008, "k": 4096, "group": 128, "dtype": "float16",
         "scales": "float16", "bias": True, "per_choice": False, "mix": 1},
        # the second matrix by itself: a row for each expert of each of 300 tokens, finer groups, scales as the quantiser gives them
        {"name": "linear_300_per_choice", "kind": "linear", "tokens": 300, "top_k": 4, "experts": 32, "all_experts": 32, "n": 2048, "k": 1024, "group": 64, "dtype": "bfloat16",
         "scales": "float32", "bias": False, "per_choice": True, "mix": 2},
        # one token of a decode step: eight of many narrow experts, 25 MB of weights
        {"name": "mlp_1_narrow", "kind": "mlp", "tokens": 1, "top_k": 8, "experts": 128, "all_experts": 128, "hidden": 2048, "inner": 1024, "group": 128, "dtype": "float16",
         "scales": "float16", "mix": 3},
        # one token, two of eight wide experts, 176 MB of weights
        {"name": "mlp_1_wide", "kind": "mlp", "tokens": 1, "top_k": 2, "experts": 8, "all_experts": 8, "hidden": 4096, "inner": 14336, "group": 128, "dtype": "bfloat16",
         "scales": "bfloat16", "mix": 4},
        # odd sizes, the finest groups, and a third of the experts on another GPU
        {"name": "mlp_13_odd", "kind": "mlp", "tokens": 13, "top_k": 3, "experts": 10, "all_experts": 15, "hidden": 2080, "inner": 1376, "group": 32, "dtype": "float16",
         "scales": "float32", "mix": 5},
        # a serving batch of 32 sequences: nearly every expert has a token or a few
        {"name": "mlp_32_narrow", "kind": "mlp", "tokens": 32, "top_k": 8, "experts": 128, "all_experts": 128, "hidden": 2048, "inner": 1024, "group": 128, "dtype": "bfloat16",
         "scales": "bfloat16", "mix": 6},
        # chunks of prompts: some tens of rows to an expert
        {"name": "mlp_600_narrow", "kind": "mlp", "tokens": 600, "top_k": 8, "experts": 128, "all_experts": 128, "hidden": 2048, "inner": 1024, "group": 128, "dtype": "bfloat16",
         "scales": "bfloat16", "mix": 7},
        # a prefill of 4096 tokens through wide experts
        {"name": "mlp_4096_wide", "kind": "mlp", "tokens": 4096, "top_k": 2, "experts": 8, "all_experts": 8, "hidden": 4096, "inner": 11008, "group": 128, "dtype": "float16",
         "scales": "float16", "mix": 8},
        # a decode step of 48 sequences from the logits to the output
        {"name": "layer_48", "kind": "layer", "tokens": 48, "top_k": 6, "experts": 64, "all_experts": 64, "hidden": 2048, "inner": 1408, "group": 64, "dtype": "bfloat16",
         "scales": "bfloat16", "mix": 9},
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("route", "linear", "mlp", "layer"), weights=(3, 3, 5, 1))[0]
    if kind == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * rng.randint(max(2, 8 // groups), 256 // groups)
        top_groups = rng.randint(max(1, groups // 2), groups)
        top_k = rng.randint(1, min(10, experts // groups * top_groups))
        tokens = _log_between(rng, 1, 16384) if rng.random() < 0.7 else rng.randint(1, 64)
        return {"kind": kind, "tokens": max(1, min(tokens, 16384 * 128 // experts)), "experts": experts, "top_k": top_k, "scores": rng.choice(("softmax", "sigmoid")),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "group_best": rng.choice((1, 2)), "renormalise": rng.random() < 0.6,
                "scale": rng.choice((1.0, 2.5)), "logits": rng.choice(("float32", "bfloat16", "float16"))}
    dtype = rng.choice(("float16", "bfloat16"))
    case = {"kind": kind, "group": rng.choice((32, 64, 128, 128, 256)), "dtype": dtype, "scales": rng.choice((dtype, "float32")), "mix": rng.randrange(10, 1 << 20)}
    if rng.random() < 0.35:  # few wide experts
        experts, top_k = rng.choice((4, 8, 16)), rng.choice((1, 2, 2, 4))
        hidden, inner = rng.choice(WIDE)
        experts = min(experts, 8)
    else:
        experts, top_k = rng.choice((16, 40, 64, 128, 160)), rng.choice((2, 4, 6, 8))
        hidden, inner = rng.choice(NARROW) if rng.random() < 0.6 else (32 * rng.randint(16, 128), 32 * rng.randint(8, 64))
    total = experts + (rng.randint(1, experts) if kind == "mlp" and rng.random() < 0.2 else 0)
    most = max(1, min(4096, int(8192 * 11008 * 4096 / (top_k * hidden * inner))))  # no more work than the largest listed
    tokens = _log_between(rng, 1, most) if rng.random() < 0.5 else rng.randint(1, min(most, 64))
    case |= {"tokens": tokens, "top_k": top_k, "experts": experts, "all_experts": total}
    if kind == "linear":
        n, k = rng.choice(((inner, hidden), (hidden, inner)))
        return case | {"n": n, "k": k, "bias": rng.random() < 0.3, "per_choice": rng.random() < 0.4}
    return case | {"hidden": hidden, "inner": inner}


def _logits(case):
    """Router's logits of tokens that like some experts more than others, [tokens, all_experts] float64: fixed by the case."""
    rng = np.random.RandomState(case["mix"])
    return rng.randn(case["tokens"], case["all_experts"]) * 1.5 + rng.randn(case["all_experts"]) * 0.7


def _choices(case):
    """Each token's experts, best first; -1 for those from number `experts` on."""
    best = np.argsort(-_logits(case), axis=1, kind="stable")[:, :case["top_k"]]
    return np.where(best < case["experts"], best, -1)


def _packed_weights(gen, experts, n, k, group, dtype, scales):
    """Normal weights, quantised group by group as ``quadmul_amd.quantize_groups`` does: amax / 7, two nibbles to a byte, even k low."""
    groups = -(-k // group)
    packed = torch.empty(experts, n, k // 2, dtype=torch.int8, device="cuda")
    scale = torch.empty(experts, n, groups, dtype=scales, device="cuda")
    for e in range(experts):
        w = (torch.randn(n, k, device="cuda", generator=gen) * (1.0 / math.sqrt(k))).to(dtype).float()
        w = torch.nn.functional.pad(w, (0, groups * group - k)).reshape(n, groups, group)
        amax = w.abs().amax(dim=2)
        q = torch.round(w * (7.0 / amax)[..., None]).clamp(-7, 7).to(torch.int8).reshape(n, -1)[:, :k] & 15
        packed[e] = q[:, 0::2] | (q[:, 1::2] << 4)
        scale[e] = amax / 7.0
    return packed, scale


def _activations(gen, shape, dtype):
    """Normal values with a few large channels, as the hidden states of a transformer have."""
    x = torch.randn(shape, device="cuda", generator=gen)
    loud = torch.randint(0, shape[-1], (max(1, shape[-1] // 512),), device="cuda", generator=gen)
    x[..., loud] *= 6.0
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, tokens, top_k, experts = case["kind"], case["tokens"], case["top_k"], case["experts"]
    if kind == "route":
        logits = (torch.randn(tokens, experts, device="cuda", generator=gen) * 1.5 + torch.randn(experts, device="cuda", generator=gen) * 0.5).to(DTYPES[case["logits"]])
        bias = torch.randn(experts, device="cuda", generator=gen) * 0.05 if case["bias"] else None
        return {"kind": kind, "logits": logits, "top_k": top_k,
                "rule": {"bias": bias} | {name: case[name] for name in ("scores", "groups", "top_groups", "group_best", "renormalise", "scale")}}
    dtype, scales, group = DTYPES[case["dtype"]], DTYPES[case["scales"]], case["group"]
    state = {"kind": kind, "group": group, "top_k": top_k}
    # the case says how many tokens each expert has; the seed, which expert that is and which tokens they are
    names, order = torch.randperm(experts, device="cuda", generator=gen), torch.randperm(tokens, device="cuda", generator=gen)
    if kind == "layer":
        state["logits"] = torch.from_numpy(_logits(case)).cuda()[order][:, names].float()
    else:
        chosen = torch.from_numpy(_choices(case)).cuda()[order]
        state["chosen"] = torch.where(chosen < 0, chosen, names[chosen.clamp(min=0)]).to(torch.int32)
    if kind == "linear":
        n, k = case["n"], case["k"]
        state["weight"], state["scale"] = _packed_weights(gen, experts, n, k, group, dtype, scales)
        state["bias"] = (torch.randn(experts, n, device="cuda", generator=gen) * 0.1).to(dtype) if case["bias"] else None
        state["x"] = _activations(gen, (tokens, top_k, k) if case["per_choice"] else (tokens, k), dtype)
        return state
    hidden, inner = case["hidden"], case["inner"]
    state["up"], state["down"] = _packed_weights(gen, experts, 2 * inner, hidden, group, dtype, scales), _packed_weights(gen, experts, hidden, inner, group, dtype, scales)
    state["x"] = _activations(gen, (tokens, hidden), dtype)
    if kind == "mlp":
        weights = torch.rand(tokens, top_k, device="cuda", generator=gen) + 0.2
        state["weights"] = weights / weights.sum(dim=1, keepdim=True)
    return state


# ---- the framework's operators -----------------------------------------------------------------------------------------------------


def _own_route(logits, top_k, rule):
    from quadmul_amd import moe

    return moe.route(logits, top_k, **rule)


def _own_linear(s):
    from quadmul_amd import moe

    return moe.gemm_experts(s["x"], s["chosen"], s["weight"], s["scale"], s["group"], s["bias"])


def _own_mlp(s, chosen, weights):
    from quadmul_amd import moe

    return moe.mlp(s["x"], chosen, weights, *s["up"], *s["down"], s["group"])


# ---- their plain form: elementary operations in 32 bits, the router's in 64, for what it chooses lies next to a border ---------------


def _plain_route(logits, top_k, rule):
    z = logits.double()
    if rule["scores"] == "softmax":
        top = z.amax(dim=1, keepdim=True)
        p = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = p.sum(dim=1, keepdim=True)
        s = p / torch.where(total > 0, total, torch.ones_like(total))
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    c = s if rule["bias"] is None else s + rule["bias"].double()
    if rule["top_groups"] < rule["groups"]:
        parts = c.unflatten(1, (rule["groups"], -1))
        best = torch.sort(parts, dim=2, descending=True).values[..., :rule["group_best"]].sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :rule["top_groups"]]
        inside = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        c = torch.where(inside[..., None], parts, torch.full_like(parts, -math.inf)).flatten(1)
    chosen = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :top_k]
    w = torch.gather(s, 1, chosen)
    if rule["renormalise"]:
        total = w.sum(dim=1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    return chosen.to(torch.int32), (w * rule["scale"]).float()


def _plain_weight(packed, scale, group):
    u = packed.view(torch.uint8)
    q = torch.stack((u & 15, u >> 4), dim=-1).reshape(u.shape[0], -1).float()
    q = torch.where(q > 7, q - 16, q)
    return q * scale.float().repeat_interleave(group, dim=1)[:, :q.shape[1]]


def _plain_linear(s):
    x, chosen, weight = s["x"], s["chosen"], s["weight"]
    y = torch.zeros(*chosen.shape, weight.shape[1], device="cuda")
    for e in range(weight.shape[0]):
        token, choice = (chosen == e).nonzero(as_tuple=True)
        if token.numel():
            rows = (x[token, choice] if x.dim() == 3 else x[token]).float() @ _plain_weight(weight[e], s["scale"][e], s["group"]).T
            y[token, choice] = rows if s["bias"] is None else rows + s["bias"][e].float()
    return y.to(x.dtype)


def _plain_mlp(s, chosen, weights):
    x, (up, up_scale), (down, down_scale) = s["x"], s["up"], s["down"]
    y = torch.zeros(x.shape, device="cuda")
    for e in range(up.shape[0]):
        token, choice = (chosen == e).nonzero(as_tuple=True)
        if token.numel():
            gate, value = (x[token].float() @ _plain_weight(up[e], up_scale[e], s["group"]).T).chunk(2, dim=1)
            h = gate / (1.0 + torch.exp(-gate)) * value
            y[token] += weights[token, choice][:, None] * (h @ _plain_weight(down[e], down_scale[e], s["group"]).T)
    return y.to(x.dtype)


def run(state):
    route, linear, mlp = (_own_route, _own_linear, _own_mlp) if own else (_plain_route, _plain_linear, _plain_mlp)
    kind = state["kind"]
    if kind == "route":
        chosen, weights = route(state["logits"], state["top_k"], state["rule"])
        return {"chosen": chosen, "weights": weights}
    if kind == "linear":
        return linear(state)
    if kind == "mlp":
        return mlp(state, state["chosen"], state["weights"])
    chosen, weights = route(state["logits"], state["top_k"], {"bias": None, "scores": "softmax", "groups": 1, "top_groups": 1, "group_best": 1, "renormalise": True, "scale": 1.0})
    return {"chosen": chosen, "weights": weights, "y": mlp(state, chosen, weights)}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------------------


def _exact_route(logits, top_k, bias, scores, groups, top_groups, group_best, renormalise, scale):
    """Token by token on the host: scores, then the order of (score downwards, number upwards)."""
    z = logits.double().cpu().numpy()
    e = np.exp(z - z.max(axis=1, keepdims=True))
    s = e / e.sum(axis=1, keepdims=True) if scores == "softmax" else 1.0 / (1.0 + np.exp(-z))
    c = s if bias is None else s + bias.double().cpu().numpy()
    experts, size = c.shape[1], c.shape[1] // groups
    chosen, weights = np.empty((len(c), top_k), dtype=np.int32), np.empty((len(c), top_k))
    for t, row in enumerate(c):
        allowed = np.arange(experts)
        if top_groups < groups:
            worth = [np.sort(row[g * size:(g + 1) * size])[::-1][:group_best].sum() for g in range(groups)]
            kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:top_groups]
            allowed = np.concatenate([np.arange(g * size, (g + 1) * size) for g in sorted(kept)])
        best = allowed[np.argsort(-row[allowed], kind="stable")[:top_k]]
        chosen[t], w = best, s[t, best]
        weights[t] = (w / w.sum() if renormalise else w) * scale
    return torch.from_numpy(chosen).cuda(), torch.from_numpy(weights).cuda()


def _exact_weight(packed, scale, group):
    low, high = packed.to(torch.int32) & 15, (packed.to(torch.int32) >> 4) & 15
    q = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=torch.float64, device="cuda")
    q[:, 0::2], q[:, 1::2] = low, high
    q -= 16.0 * (q >= 8)
    for g in range(scale.shape[1]):
        q[:, g * group:(g + 1) * group] *= scale[:, g, None].double()
    return q


def _exact_linear(s):
    x = s["x"] if s["x"].dim() == 3 else s["x"][:, None].expand(-1, s["top_k"], -1)
    x, which = x.flatten(0, 1), s["chosen"].flatten()
    y = torch.zeros(which.shape[0], s["weight"].shape[1], dtype=torch.float64, device="cuda")
    for e in torch.unique(which).tolist():
        if e >= 0:
            y[which == e] = x[which == e].double() @ _exact_weight(s["weight"][e], s["scale"][e], s["group"]).T + (0.0 if s["bias"] is None else s["bias"][e].double())
    return y.unflatten(0, s["chosen"].shape)


def _exact_mlp(s, chosen, weights):
    inner = s["down"][0].shape[2] * 2
    y = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    for e in torch.unique(chosen).tolist():
        if e < 0:
            continue
        share = (weights.double() * (chosen == e)).sum(dim=1)
        who = (chosen == e).any(dim=1)
        first = s["x"][who].double() @ _exact_weight(s["up"][0][e], s["up"][1][e], s["group"]).T
        h = first[:, :inner] * torch.sigmoid(first[:, :inner]) * first[:, inner:]
        y[who] += share[who, None] * (h @ _exact_weight(s["down"][0][e], s["down"][1][e], s["group"]).T)
    return y


def exact(case, seed):
    """What ``run`` returns, in 64 bits from the same inputs."""
    s, kind = prepare(case, seed), case["kind"]
    if kind == "route":
        return dict(zip(("chosen", "weights"), _exact_route(s["logits"], s["top_k"], **s["rule"])))
    if kind == "linear":
        return _exact_linear(s)
    if kind == "mlp":
        return _exact_mlp(s, s["chosen"], s["weights"])
    chosen, weights = _exact_route(s["logits"], s["top_k"], None, "softmax", 1, 1, 1, True, 1.0)
    return {"chosen": chosen, "weights": weights, "y": _exact_mlp(s, chosen, weights)}


def work(case):
    kind, tokens, top_k = case["kind"], case["tokens"], case["top_k"]
    if kind == "route":
        experts = case["experts"]
        return {"bytes": tokens * (experts * (4 if case["logits"] == "float32" else 2) + 8 * top_k) + (4 * experts if case["bias"] else 0), "flops": tokens * experts * 4}
    chosen = _choices(case)
    slots, touched, scale_bytes = int((chosen >= 0).sum()), len(np.unique(chosen[chosen >= 0])), 4 if case["scales"] == "float32" else 2

    def matrix(n, k):
        return touched * n * (k / 2 + -(-k // case["group"]) * scale_bytes)

    if kind == "linear":
        n, k = case["n"], case["k"]
        rows = slots if case["per_choice"] else int((chosen >= 0).any(axis=1).sum())
        return {"bytes": matrix(n, k) + (2 * touched * n if case["bias"] else 0) + 2 * rows * k + 2 * tokens * top_k * n + 4 * tokens * top_k, "flops": 2 * slots * n * k}
    hidden, inner = case["hidden"], case["inner"]
    routed = tokens * case["experts"] * 4 + 16 * tokens * top_k if kind == "layer" else 8 * tokens * top_k
    return {"bytes": matrix(2 * inner, hidden) + matrix(hidden, inner) + 4 * tokens * hidden + routed, "flops": 6 * slots * hidden * inner}

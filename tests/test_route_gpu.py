"""The router's choice (csrc/qm_route.hpp) against the definition in 64 bits on the host: every number chosen, and the weights to one rounding."""
import numpy as np
import pytest
import torch

import moe_util
import quadmul_amd as qm
from quadmul_amd import moe

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(logits, top_k, bias=None, **rule):
    chosen, weights = moe.route(logits, top_k, bias=bias, **rule)
    z = logits.double().cpu().numpy()
    want, share = moe_util.route(z, top_k, None if bias is None else bias.cpu().numpy(), **rule)
    assert chosen.dtype == torch.int32 and weights.dtype == torch.float32 and chosen.shape == weights.shape == (logits.shape[0], top_k)
    assert np.array_equal(chosen.cpu().numpy(), want)
    got = weights.cpu().double().numpy()
    # one rounding to float32; scores in 64 bits are off by less than a thousandth of that
    assert np.array_equal(np.isnan(got), np.isnan(share))
    assert (np.abs(np.nan_to_num(got) - np.nan_to_num(share)) <= 2.0 ** -24 * 1.001 * np.abs(np.nan_to_num(share)) + 2.0 ** -149).all()
    return chosen, weights


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 8, 2), (3, 64, 6), (5, 65, 7), (64, 128, 8), (7, 200, 64), (130, 256, 8), (9, 512, 10), (4, 1000, 33), (2, 1024, 64), (1029, 40, 3), (2, 5, 5)])
@pytest.mark.parametrize("scores", moe.SCORES)
def test_sizes(tokens, experts, top_k, scores, dtype):
    g = torch.Generator().manual_seed(tokens + experts)
    z = (torch.randn(tokens, experts, generator=g) * 2.0).to(dtype).cuda()
    bias = torch.randn(experts, generator=g).cuda() * 0.1
    check(z, top_k, scores=scores)
    check(z, top_k, scores=scores, renormalise=True, scale=2.5)
    check(z, top_k, bias, scores=scores, renormalise=True)


@pytest.mark.parametrize("group_best", [1, 2])
@pytest.mark.parametrize("tokens,experts,groups,top_groups,top_k", [(33, 256, 8, 4, 8), (5, 64, 64, 7, 7), (17, 60, 3, 2, 9), (4, 1024, 64, 5, 20), (9, 16, 8, 3, 6), (3, 160, 5, 5, 6), (21, 96, 2, 1, 48)])
@pytest.mark.parametrize("scores", moe.SCORES)
def test_groups(tokens, experts, groups, top_groups, top_k, group_best, scores):
    g = torch.Generator().manual_seed(experts + groups)
    z = torch.randn(tokens, experts, generator=g).cuda()
    rule = dict(groups=groups, top_groups=top_groups, group_best=group_best, scores=scores)
    check(z, top_k, **rule)
    check(z, top_k, torch.randn(experts, generator=g).cuda() * 0.2, renormalise=True, scale=0.5, **rule)
    check(z.to(torch.bfloat16), top_k, **rule)


@pytest.mark.parametrize("scores", moe.SCORES)
def test_ties_go_to_the_lower_number(scores):
    z = torch.zeros(6, 128, device="cuda")
    z[1, 5:] = 1.0
    z[2, ::3] = -1.0
    z[3] = torch.randint(-2, 3, (128,), generator=torch.Generator().manual_seed(1)).float()
    z[4, 127] = -0.0
    chosen, _ = check(z, 10, scores=scores)
    assert chosen[0].tolist() == list(range(10)) and chosen[1].tolist() == list(range(5, 15))
    check(z, 10, scores=scores, groups=16, top_groups=3)
    check(z, 8, torch.zeros(128, device="cuda"), scores=scores, groups=8, top_groups=1, group_best=1)


@pytest.mark.parametrize("scores", moe.SCORES)
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
def test_what_is_no_number(scores, dtype):
    """Masked experts, rows that are masked whole, NaN and infinities: always top_k different experts of those there are."""
    inf, nan = float("inf"), float("nan")
    z = torch.randn(12, 70, generator=torch.Generator().manual_seed(3)).to(dtype)
    z[0] = -inf
    z[1, 3:] = -inf
    z[2] = torch.finfo(dtype).min
    z[3, 10] = torch.finfo(dtype).min
    z[4, :69] = -inf
    z[5, 7] = nan
    z[6] = nan
    if scores == "sigmoid":  # (of a softmax NaN)
        z[7, 11] = inf
        z[8] = inf
    z[9] = torch.finfo(dtype).max
    z = z.cuda()
    for rule in ({}, {"renormalise": True}, {"groups": 7, "top_groups": 2}, {"groups": 7, "top_groups": 1, "group_best": 1, "renormalise": True}):
        chosen, weights = check(z, 8, scores=scores, **rule)
        assert all(len(set(row)) == 8 and min(row) >= 0 and max(row) < 70 for row in chosen.tolist())
        assert not weights[0].any()
    bias = torch.zeros(70, device="cuda")
    bias[::2] = -inf  # experts that are switched off
    chosen, _ = check(z, 8, bias, scores=scores)
    assert (chosen[10:] % 2 == 1).all()


def test_plus_infinity_in_a_softmax():
    z = torch.zeros(2, 70, device="cuda")
    z[0, 9] = float("inf")
    chosen, weights = moe.route(z, 4)
    assert len(set(chosen[0].tolist())) == 4 and weights[0].isnan().all() and chosen[1].tolist() == [0, 1, 2, 3] and weights[1].isfinite().all()


def test_scores_next_to_a_border():
    """Scores that 32 bits do not tell apart: sigmoids of neighbouring logits, plus a bias."""
    z = torch.full((4, 256), 9.0, device="cuda")
    z += torch.arange(256, device="cuda") * 2.0 ** -20 * torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")[:, None]
    chosen, _ = check(z, 8, torch.full((256,), 0.25, device="cuda"), scores="sigmoid")
    assert chosen[0].tolist() == list(range(255, 247, -1)) and chosen[1].tolist() == list(range(8))
    check(z * 1e-3, 8)


def test_rows_at_a_distance_and_any_order():
    z = torch.randn(9, 200, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    wide = torch.full((9, 333), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 1:201] = z
    first = check(z, 6)
    for same in (wide[:, 1:201], z.t().contiguous().t(), torch.cat((z, z))[:9]):
        again = moe.route(same, 6)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    one = moe.route(z[:1].expand(5, -1), 6)  # rows at no distance
    assert (one[0] == first[0][:1]).all()
    assert moe.route(z[:0], 6)[0].shape == (0, 6)


def test_many_tokens():
    z = torch.randn(70001, 16, generator=torch.Generator().manual_seed(6)).cuda()
    chosen, weights = moe.route(z, 2, renormalise=True)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(chosen.long(), order)
    want = torch.softmax(torch.gather(z.double(), 1, order), dim=1)
    assert bool(((weights.double() - want).abs() <= 2.0 ** -24 * 1.001 * want).all())


def test_on_another_stream_and_in_a_graph():
    z = torch.randn(40, 256, generator=torch.Generator().manual_seed(7)).cuda()
    rule = dict(scores="sigmoid", groups=8, top_groups=4, renormalise=True)
    first = moe.route(z, 8, **rule)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = moe.route(z, 8, **rule)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = moe.route(z, 8, **rule)
    for seed in range(3):
        z.copy_(torch.randn(40, 256, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        now = moe.route(z, 8, **rule)
        assert torch.equal(held[0], now[0]) and torch.equal(held[1], now[1])


def test_refusals():
    z, bias = torch.zeros(4, 64, device="cuda"), torch.zeros(64, device="cuda")
    assert moe.route(z, 4, bias=bias)[0].shape == (4, 4)
    bad = [((z, 0), {}), ((z, 65), {}), ((z, 4), {"groups": 5}), ((z, 4), {"groups": 0}), ((z, 4), {"groups": 8, "top_groups": 9}), ((z, 4), {"groups": 8, "top_groups": 0}),
           ((z, 9), {"groups": 8, "top_groups": 1}), ((z, 4), {"group_best": 3}), ((z, 4), {"scores": "tanh"}), ((z, 4), {"bias": bias[:63]}), ((z, 4), {"bias": bias.half()}),
           ((z, 4), {"bias": bias.cpu()}), ((z, 4), {"bias": bias[:, None]}), ((z.double(), 4), {}), ((z[0], 4), {}), ((z.cpu(), 4), {}), ((z.int(), 4), {}),
           ((torch.zeros(2, 1025, device="cuda"), 4), {}), ((torch.zeros(2, 0, device="cuda"), 1), {}), ((torch.zeros(2, 130, device="cuda"), 65), {}),
           ((torch.zeros(2, 130, device="cuda"), 2), {"groups": 65})]
    for args, rule in bad:
        with pytest.raises(qm.QuadmulError):
            moe.route(*args, **rule)


def test_without_the_extension_the_same(monkeypatch):
    import types

    z, bias = torch.randn(6, 96, generator=torch.Generator().manual_seed(8)).cuda(), torch.randn(96, generator=torch.Generator().manual_seed(9)).cuda()
    rule = dict(bias=bias, scores="sigmoid", groups=4, top_groups=2, renormalise=True, scale=1.5)
    first = moe.route(z[:, ::1], 5, **rule)
    monkeypatch.setattr(qm, "_ext", types.SimpleNamespace(**dict.fromkeys(qm._EXT_FUNCTIONS, lambda *a: None)))
    again = moe.route(z, 5, **rule)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    test_refusals()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("experts,top_k,groups,top_groups", [(8, 2, 1, 1), (60, 6, 3, 2), (128, 8, 16, 3), (200, 16, 1, 1), (256, 8, 8, 4)])
@pytest.mark.parametrize("scores", moe.SCORES)
def test_so_many_tokens_that_16_lanes_are_enough(scores, experts, top_k, groups, top_groups, dtype):
    """More than 4096 tokens, a workgroup's last ones missing; rows of equal logits, masked ones and NaN among them."""
    z = (torch.randn(4099, experts, generator=torch.Generator().manual_seed(experts)) * 2.0).to(dtype)
    z[5], z[4098], z[77, ::2], z[78, 1:] = 0.5, -float("inf"), -float("inf"), torch.finfo(dtype).min
    z[79, 3] = float("nan")
    z = z.cuda()
    bias = torch.randn(experts, generator=torch.Generator().manual_seed(1)).cuda() * 0.1
    check(z, top_k, scores=scores, renormalise=True)
    check(z, top_k, bias, scores=scores, scale=1.5)
    check(z, top_k, scores=scores, groups=groups, top_groups=top_groups, renormalise=True)

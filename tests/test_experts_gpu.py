"""Products with the int4 weights of each token's experts and their gated MLP (csrc/qm_experts.hpp) against 64 bits: every kernel that the choice leads to, both
types, scales of both kinds, odd sizes, experts that nobody or everybody chose, numbers that are no expert."""
import pytest
import torch

import moe_util
import quadmul_amd as qm
from quadmul_amd import moe

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]
IDS = ["f16", "bf16"]


def product(tokens, top_k, experts, n, k, group, dtype, scales, seed, per_choice=False, with_bias=False, **how):
    x, chosen, q, s = moe_util.problem(tokens, top_k, experts, n, k, group, dtype, scales, seed, **how)
    g = torch.Generator().manual_seed(seed + 1)
    if per_choice:
        x = (torch.randn(tokens, top_k, k, generator=g) * 2.0).to(dtype).cuda()
    bias = torch.randn(experts, n, generator=g).to(dtype).cuda() if with_bias else None
    y = moe.gemm_experts(x, chosen, moe_util.pack(q), s, group, bias)
    moe_util.check_product(x, chosen, q, s, group, bias, y)


SIZES = [  # tokens, top_k, experts, n, k, group
    (1, 1, 1, 16, 32, 32), (1, 2, 8, 64, 128, 128), (1, 8, 128, 100, 256, 64), (2, 3, 5, 257, 1056, 32), (5, 2, 8, 130, 2048, 128), (13, 4, 16, 300, 672, 96),
    (16, 2, 2, 48, 416, 32), (17, 1, 1, 70, 512, 256), (40, 2, 4, 129, 1024, 128), (64, 8, 64, 96, 544, 64), (100, 2, 2, 333, 800, 128), (300, 4, 8, 260, 288, 32),
    (600, 2, 3, 128, 640, 128), (1000, 8, 16, 144, 256, 64), (3, 2, 4, 7, 8192, 128), (2, 2, 4, 40, 14336, 128),
    (4, 2, 3, 33, 2, 32), (6, 3, 7, 65, 130, 64), (20, 2, 4, 9, 1002, 128), (4, 2, 3, 5, 0, 32),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("wide", [False, True], ids=["scales16", "scales32"])
@pytest.mark.parametrize("tokens,top_k,experts,n,k,group", SIZES)
def test_product(tokens, top_k, experts, n, k, group, wide, dtype):
    scales = torch.float32 if wide else dtype
    product(tokens, top_k, experts, n, k, group, dtype, scales, tokens + n + k, with_bias=n % 2 == 0)
    product(tokens, top_k, experts, n, k, group, dtype, scales, tokens + n + k, per_choice=True, with_bias=n % 2 == 1, absent=0.3)


def gated(tokens, top_k, experts, hidden, inner, group, dtype, scales, seed, **how):
    x, chosen, q_up, s_up = moe_util.problem(tokens, top_k, experts, 2 * inner, hidden, group, dtype, scales, seed, **how)
    _, _, q_down, s_down = moe_util.problem(1, 1, experts, hidden, inner, group, dtype, scales, seed + 1)
    weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(seed + 2)).cuda()
    y = moe.mlp(x, chosen, weights, moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, group)
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, group, y)
    return x, chosen, weights, (q_up, s_up, q_down, s_down), y


MLPS = [  # tokens, top_k, experts, hidden, inner, group
    (1, 1, 1, 32, 32, 32), (1, 8, 32, 256, 128, 128), (1, 2, 8, 1056, 352, 32), (2, 6, 64, 512, 192, 64), (3, 2, 4, 2048, 1024, 128), (9, 4, 16, 288, 416, 96),
    (16, 2, 2, 256, 512, 256), (33, 3, 10, 544, 160, 32), (64, 8, 64, 256, 256, 128), (120, 2, 3, 640, 384, 128), (300, 4, 8, 512, 320, 64), (700, 2, 2, 384, 512, 128),
    (1100, 6, 16, 256, 192, 64), (2, 2, 4, 64, 8192, 128), (3, 1, 4, 8192, 64, 128), (5, 2, 4, 34, 6, 32), (21, 3, 5, 130, 66, 64),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("wide", [False, True], ids=["scales16", "scales32"])
@pytest.mark.parametrize("tokens,top_k,experts,hidden,inner,group", MLPS)
def test_mlp(tokens, top_k, experts, hidden, inner, group, wide, dtype):
    scales = torch.float32 if wide else dtype
    gated(tokens, top_k, experts, hidden, inner, group, dtype, scales, tokens + hidden)
    gated(tokens, top_k, experts, hidden, inner, group, dtype, scales, tokens + inner, absent=0.4)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 4, 30, 90, 400])
def test_the_same_expert_twice_and_all_at_one(tokens, dtype):
    """Choices that are not different, and one expert that has every row."""
    product(tokens, 4, 3, 96, 256, 128, dtype, dtype, tokens, distinct=False, with_bias=True)
    gated(tokens, 4, 3, 256, 96, 64, dtype, dtype, tokens, distinct=False)
    x, _, q, s = moe_util.problem(tokens, 2, 9, 80, 512, 128, dtype, dtype, 3)
    for chosen in (torch.full((tokens, 2), 7), torch.tensor([[0, 8]]).expand(tokens, 2)):
        chosen = chosen.to(torch.int32).contiguous().cuda()
        moe_util.check_product(x, chosen, q, s, 128, None, moe.gemm_experts(x, chosen, moe_util.pack(q), s, 128))


@pytest.mark.parametrize("tokens", [1, 5, 70, 300])
def test_numbers_that_are_no_expert(tokens):
    """-1 and everything outside: zeros in the product, nothing in the sum, whatever the weight is; also where nobody has an expert."""
    x, chosen, q, s = moe_util.problem(tokens, 3, 6, 64, 256, 64, torch.float16, torch.float16, 4)
    _, _, q2, s2 = moe_util.problem(1, 1, 6, 256, 32, 64, torch.float16, torch.float16, 5)
    w, w2 = moe_util.pack(q), moe_util.pack(q2)
    for none in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        some = chosen.clone()
        some[:, 1] = none
        moe_util.check_product(x, some, q, s, 64, None, moe.gemm_experts(x, some, w, s, 64))
        weights = torch.rand(tokens, 3, device="cuda")
        weights[:, 1] = float("nan")
        y = moe.mlp(x, some, weights, w, s, w2, s2, 64)
        moe_util.check_mlp(x, some, torch.nan_to_num(weights), q, s, q2, s2, 64, y)
        nobody = torch.full_like(chosen, none)
        assert not moe.gemm_experts(x, nobody, w, s, 64).any() and not moe.mlp(x, nobody, weights, w, s, w2, s2, 64).any()


@pytest.mark.parametrize("tokens,top_k,experts,k", [(1, 2, 4, 512), (9, 2, 4, 512), (80, 2, 4, 512), (400, 2, 4, 256), (7, 2, 3, 66)])
def test_rows_at_a_distance(tokens, top_k, experts, k):
    x, chosen, q, s = moe_util.problem(tokens, top_k, experts, 70, k, 64, torch.bfloat16, torch.bfloat16, 6)
    _, _, q2, s2 = moe_util.problem(1, 1, experts, k, 34, 64, torch.bfloat16, torch.bfloat16, 7)
    up, s_up = torch.cat((q[:, :34], q[:, 34:68]), 1), torch.cat((s[:, :34], s[:, 34:68]), 1)
    weights = torch.rand(tokens, top_k, device="cuda")
    first, y = moe.gemm_experts(x, chosen, moe_util.pack(q), s, 64), moe.mlp(x, chosen, weights, moe_util.pack(up), s_up, moe_util.pack(q2), s2, 64)
    moe_util.check_product(x, chosen, q, s, 64, None, first)
    for pad in (1, 2, 8, 64):
        wide = torch.full((tokens, k + pad), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, :k] = x
        assert torch.equal(first, moe.gemm_experts(wide[:, :k], chosen, moe_util.pack(q), s, 64))
        assert torch.equal(y, moe.mlp(wide[:, :k], chosen, weights, moe_util.pack(up), s_up, moe_util.pack(q2), s2, 64))
        each = torch.full((tokens, top_k, k + pad), float("nan"), dtype=torch.bfloat16, device="cuda")
        each[..., :k] = x[:, None]
        assert torch.equal(first, moe.gemm_experts(each[..., :k], chosen, moe_util.pack(q), s, 64))
    assert torch.equal(first, moe.gemm_experts(x.t().contiguous().t(), chosen, moe_util.pack(q), s, 64))
    assert torch.equal(first, moe.gemm_experts(x[:, None].expand(-1, top_k, -1), chosen, moe_util.pack(q), s, 64))
    same = x[:1].expand(tokens, -1)  # rows at no distance
    moe_util.check_product(same, chosen, q, s, 64, None, moe.gemm_experts(same, chosen, moe_util.pack(q), s, 64))


@pytest.mark.parametrize("tokens", [1, 6, 80, 300])
@pytest.mark.parametrize("x_off,w_off,s_off", [(1, 0, 0), (0, 1, 0), (0, 4, 1), (3, 2, 1), (8, 16, 0)])
def test_any_address(tokens, x_off, w_off, s_off):
    x, chosen, q, s = moe_util.problem(tokens, 2, 5, 48, 256, 32, torch.bfloat16, torch.bfloat16, 8)
    at = lambda t, off: torch.zeros(t.numel() + off, dtype=t.dtype, device="cuda")[off:].view(t.shape).copy_(t)  # noqa: E731
    y = moe.gemm_experts(at(x, x_off), chosen, at(moe_util.pack(q), w_off), at(s, s_off), 32)
    moe_util.check_product(x, chosen, q, s, 32, None, y)
    _, _, q2, s2 = moe_util.problem(1, 1, 5, 256, 64, 32, torch.bfloat16, torch.bfloat16, 9)
    q3, s3 = torch.cat((q, q, q), 1)[:, :128].contiguous(), torch.cat((s, s, s), 1)[:, :128].contiguous()
    weights = torch.rand(tokens, 2, device="cuda")
    y = moe.mlp(at(x, x_off), chosen, weights, at(moe_util.pack(q3), w_off), at(s3, s_off), at(moe_util.pack(q2), w_off), at(s2, s_off), 32)
    moe_util.check_mlp(x, chosen, weights, q3, s3, q2, s2, 32, y)


@pytest.mark.parametrize("tokens", [1, 5, 70, 300])
def test_infinities_and_nans_stay_with_their_token(tokens):
    x, chosen, q, s = moe_util.problem(tokens, 2, 3, 64, 256, 64, torch.float16, torch.float16, 10)
    _, _, q2, s2 = moe_util.problem(1, 1, 3, 256, 32, 64, torch.float16, torch.float16, 11)
    weights = torch.rand(tokens, 2, device="cuda")
    first = moe.gemm_experts(x, chosen, moe_util.pack(q), s, 64), moe.mlp(x, chosen, weights, moe_util.pack(q), s, moe_util.pack(q2), s2, 64)
    for bad in (float("inf"), float("nan")):
        lost = x.clone()
        lost[tokens // 2, 100] = bad
        keep = torch.arange(tokens, device="cuda") != tokens // 2
        for was, now in zip(first, (moe.gemm_experts(lost, chosen, moe_util.pack(q), s, 64), moe.mlp(lost, chosen, weights, moe_util.pack(q), s, moe_util.pack(q2), s2, 64))):
            assert torch.equal(was[keep], now[keep]) and not now[~keep].isfinite().all()


@pytest.mark.parametrize("tokens", [1, 40, 300])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("k,group", [(96, 32), (160, 64), (320, 128), (352, 32)])
def test_an_infinite_scale_meets_no_element_past_the_end(k, group, dtype, tokens):
    # ones times ones: the sum of the last group is positive, so its scale makes infinity of every product, and NaN would come from places behind K
    x, chosen = torch.ones((tokens, k), dtype=dtype, device="cuda"), torch.zeros((tokens, 1), dtype=torch.int32, device="cuda")
    scale = torch.ones((2, 40, -(-k // group)), device="cuda")
    scale[..., -1] = float("inf")
    packed = torch.full((2, 40, k // 2), 0x11, dtype=torch.uint8, device="cuda")
    y = moe.gemm_experts(x, chosen, packed, scale, group)
    assert bool((y == float("inf")).all())


@pytest.mark.parametrize("tokens", [1, 5, 70])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_gates_at_both_ends(tokens, dtype):
    """Gates of minus and plus thousands: zero times a finite value, and the value times the gate; no NaN on the way."""
    q_up = torch.zeros(2, 64, 32, dtype=torch.int8, device="cuda")
    q_up[0, :16, 0], q_up[0, 16:32, 0], q_up[:, 32:, 1], q_up[1, :32, 0] = -7, 7, 1, 1
    s_up = torch.full((2, 64, 1), 1.0, device="cuda")
    q_down = torch.randint(-8, 8, (2, 32, 32), dtype=torch.int8, generator=torch.Generator().manual_seed(1)).cuda()
    s_down = torch.full((2, 32, 1), 2.0 ** -10, device="cuda")
    x = torch.zeros(tokens, 32, dtype=dtype, device="cuda")
    x[:, 0], x[:, 1] = 2000.0, 0.5
    chosen, weights = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").expand(tokens, 2).contiguous(), torch.ones(tokens, 2, device="cuda")
    y = moe.mlp(x, chosen, weights, moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, 32)
    assert y.isfinite().all() and y.any()
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, 32, y)


@pytest.mark.parametrize("tokens", [1, 6, 70, 300])
def test_on_another_stream_and_in_a_graph(tokens):
    """The layer, from the hidden states to the sum, with other experts at every replay."""
    g = torch.Generator().manual_seed(12)
    layer = moe.SparseMLP(torch.randn(8, 256, generator=g).half().cuda(), moe.W4A16Experts.from_float(torch.randn(8, 128, 256, generator=g).half().cuda() * 0.06,
                          torch.randn(8, 256, 64, generator=g).half().cuda() * 0.12, 64), 2, renormalise=True)
    x = torch.randn(tokens, 256, generator=g).half().cuda()
    first = layer(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = layer(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    graphs = []
    for _ in range(2):  # two that share a workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            y = layer(x)
        graphs.append((graph, y))
    for seed in range(4):
        x.copy_(torch.randn(tokens, 256, generator=torch.Generator().manual_seed(seed)))
        for graph, y in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, layer(x))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 17, 200])
def test_the_layer_together(tokens, dtype):
    """Router, experts and sum as a module against the three from their definitions, quantised weights included."""
    g = torch.Generator().manual_seed(13)
    experts, hidden, inner, top_k = 12, 256, 96, 3
    up, down = (torch.randn(experts, 2 * inner, hidden, generator=g) / 16).to(dtype).cuda(), (torch.randn(experts, hidden, inner, generator=g) / 10).to(dtype).cuda()
    router, bias = (torch.randn(experts, hidden, generator=g) / 16).cuda(), torch.randn(experts, generator=g).cuda() * 0.05
    rule = dict(scores="sigmoid", groups=4, top_groups=2, renormalise=True, scale=1.25)
    layer = moe.SparseMLP(router, moe.W4A16Experts.from_float(up, down, 32), top_k, bias, **rule)
    x = torch.randn(tokens, hidden, generator=g).to(dtype).cuda()
    y = layer(x.reshape(1, tokens, hidden))
    assert y.shape == (1, tokens, hidden)
    e = layer.experts
    chosen, weights = moe_util.route((x.float() @ router.t()).double().cpu().numpy(), top_k, bias.cpu().numpy(), **rule)
    unpacked = [qm.unpack_int4(t.reshape(-1, t.shape[-1])).reshape(experts, t.shape[1], -1) for t in (e.up_packed, e.down_packed)]
    moe_util.check_mlp(x, torch.from_numpy(chosen).cuda(), torch.from_numpy(weights).cuda(), unpacked[0], e.up_scale, unpacked[1], e.down_scale, 32, y[0])


def test_refusals():
    x, chosen, q, s = moe_util.problem(4, 2, 3, 64, 128, 64, torch.float16, torch.float16, 14)
    w, bias, weights = moe_util.pack(q), torch.zeros(3, 64, dtype=torch.float16, device="cuda"), torch.ones(4, 2, device="cuda")
    w2, s2 = torch.zeros(3, 128, 16, dtype=torch.int8, device="cuda"), torch.ones(3, 128, 1, dtype=torch.float16, device="cuda")
    assert moe.gemm_experts(x, chosen, w, s, 64, bias).shape == (4, 2, 64) and moe.mlp(x, chosen, weights, w, s, w2, s2, 64).shape == (4, 128)
    for args in [(x.float(), chosen, w, s, 64), (x, chosen.long(), w, s, 64), (x, chosen[:3], w, s, 64), (x, chosen.t().contiguous().t(), w, s, 64), (x, chosen, w.float(), s, 64), (x, chosen, w, s, 32),
                 (x, chosen, w, s, 48), (x, chosen, w, s, 0), (x, chosen, w, s, -64), (x, chosen, w[:, :, :32], s, 64), (x, chosen, w, s.to(torch.bfloat16), 64), (x, chosen, w, s[:2], 64),
                 (x, chosen, w[0], s[0], 64), (x[0], chosen, w, s, 64), (x[:, None], chosen, w, s, 64), (x, chosen, w, s, 64, bias[:, :63]), (x, chosen, w, s, 64, bias.float()),
                 (x, chosen, w, s, 64, bias.flatten()), (x.cpu(), chosen.cpu(), w.cpu(), s.cpu(), 64), (x, chosen.cpu(), w, s, 64), (x, chosen, w.cpu(), s, 64), (x, chosen, w.transpose(1, 2), s, 64)]:
        with pytest.raises(qm.QuadmulError):
            moe.gemm_experts(*args)
    for args in [(x.float(), chosen, weights, w, s, w2, s2, 64), (x, chosen, weights.half(), w, s, w2, s2, 64), (x, chosen, weights[:, :1], w, s, w2, s2, 64), (x, chosen, weights.cpu(), w, s, w2, s2, 64),
                 (x, chosen, weights, w[:, :60], s[:, :60], w2, s2, 64), (x, chosen, weights, w, s, w2[:2], s2[:2], 64), (x, chosen, weights, w, s, w2[:, :64], s2[:, :64], 64),
                 (x, chosen, weights, w2, s2, w2, s2, 64), (x[:, None], chosen, weights, w, s, w2, s2, 64), (x, chosen, weights, w, s, w2, s2, 32), (x, chosen[:2], weights[:2], w, s, w2, s2, 64)]:
        with pytest.raises(qm.QuadmulError):
            moe.mlp(*args)
    with pytest.raises(qm.QuadmulError):
        moe.W4A16Experts(w, s, w2, s2, 32)
    with pytest.raises(qm.QuadmulError):
        moe.W4A16Experts(w[:, :60], s[:, :60], w2, s2, 64)
    with pytest.raises(qm.QuadmulError):
        moe.SparseMLP(torch.zeros(3, 64, device="cuda"), moe.W4A16Experts(w, s, w2, s2, 64), 2)


def test_nothing_to_do():
    x, chosen, q, s = moe_util.problem(4, 2, 3, 64, 128, 64, torch.float16, torch.float16, 15)
    w, weights = moe_util.pack(q), torch.ones(4, 2, device="cuda")
    w2, s2 = torch.zeros(3, 128, 16, dtype=torch.int8, device="cuda"), torch.ones(3, 128, 1, dtype=torch.float16, device="cuda")
    assert moe.gemm_experts(x[:0], chosen[:0], w, s, 64).shape == (0, 2, 64) and moe.gemm_experts(x, chosen[:, :0].contiguous(), w, s, 64).shape == (4, 0, 64)
    assert moe.gemm_experts(x, chosen, w[:, :0], s[:, :0], 64).shape == (4, 2, 0)
    assert not moe.gemm_experts(x, chosen, w[:0], s[:0], 64).any()  # no expert at all
    assert moe.mlp(x[:0], chosen[:0], weights[:0], w, s, w2, s2, 64).shape == (0, 128)
    assert not moe.mlp(x, chosen[:, :0].contiguous(), weights[:, :0].contiguous(), w, s, w2, s2, 64).any()
    assert not moe.mlp(x, chosen, weights, w[:, :0], s[:, :0], w2[:, :, :0], s2[:, :, :0], 64).any()  # no inner columns
    assert not moe.mlp(x, chosen, weights, w[:0], s[:0], w2[:0], s2[:0], 64).any()


def test_without_the_extension_the_same(monkeypatch):
    import types

    x, chosen, q, s = moe_util.problem(6, 2, 3, 64, 128, 64, torch.bfloat16, torch.float32, 16)
    _, _, q2, s2 = moe_util.problem(1, 1, 3, 128, 32, 64, torch.bfloat16, torch.float32, 17)
    w, w2, weights, bias = moe_util.pack(q), moe_util.pack(q2), torch.rand(6, 2, device="cuda"), torch.rand(3, 64, device="cuda").to(torch.bfloat16)
    calls = [lambda: moe.gemm_experts(x, chosen, w, s, 64, bias), lambda: moe.gemm_experts(x[:, None].expand(-1, 2, -1), chosen, w, s, 64), lambda: moe.mlp(x, chosen, weights, w, s, w2, s2, 64)]
    first = [call() for call in calls]
    monkeypatch.setattr(qm, "_ext", types.SimpleNamespace(**dict.fromkeys(qm._EXT_FUNCTIONS, lambda *a: None)))
    assert all(torch.equal(a, call()) for a, call in zip(first, calls))
    test_refusals()
    test_nothing_to_do()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens,top_k,experts", [(1, 70, 80), (2, 33, 40), (8, 8, 128), (16, 4, 129), (1, 130, 64), (9, 8, 128), (1, 2, 4200), (30, 3, 4097)])
def test_numbers_of_choices_and_of_experts(tokens, top_k, experts, dtype):
    """One token of more choices than a wave has lanes, 64 slots and one or two more, more experts than slots are sorted by."""
    product(tokens, top_k, experts, 34, 96, 32, dtype, dtype, experts, distinct=top_k <= experts, with_bias=True)
    gated(tokens, top_k, experts, 96, 32, 32, dtype, dtype, experts, distinct=top_k <= experts, absent=0.1)


@pytest.mark.parametrize("tokens", [2, 70, 300])
def test_two_streams_at_once(tokens):
    g = torch.Generator().manual_seed(16)
    layer = moe.SparseMLP(torch.randn(16, 512, generator=g).half().cuda(), moe.W4A16Experts.from_float(torch.randn(16, 512, 512, generator=g).half().cuda() * 0.04,
                          torch.randn(16, 512, 256, generator=g).half().cuda() * 0.06, 128), 4)
    xs = [torch.randn(tokens, 512, generator=g).half().cuda() for _ in range(2)]
    want, streams, got = [layer(x) for x in xs], [torch.cuda.Stream() for _ in xs], [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for x, s, y in zip(xs, streams, got):
            with torch.cuda.stream(s):
                y.append(layer(x))
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)


def test_weights_behind_four_gigabytes():
    """Ten experts of half a gigabyte; and all of it as one expert, whose offsets have more than 32 bits."""
    experts, n, k, group = 10, 65536, 16384, 128
    g = torch.Generator(device="cuda").manual_seed(17)
    flat = torch.empty(experts * n * (k // 2) + 16, dtype=torch.uint8, device="cuda").random_(0, 256, generator=g)
    scale = (torch.rand(experts, n, k // group, generator=g, device="cuda") * 0.02 + 0.001).half()
    x = torch.randn(200, k, generator=g, device="cuda").half()
    for tokens, off in ((2, 0), (200, 0), (2, 1)):
        packed = flat[off:off + experts * n * (k // 2)].view(experts, n, k // 2)
        chosen = (torch.arange(tokens, device="cuda") % 2 * -3 + 9).to(torch.int32)[:, None].contiguous()  # the last expert and one in the middle
        y = moe.gemm_experts(x[:tokens], chosen, packed, scale, group)
        for first in (0, n - 40):
            some = slice(first, first + 40)
            q = torch.stack([qm.unpack_int4(packed[e, some].contiguous()) for e in range(experts)])
            moe_util.check_product(x[:tokens], chosen, q, scale[:, some].contiguous(), group, None, y[:, :, some])
    one, zero = flat[:-16].view(1, experts * n, k // 2), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    y = moe.gemm_experts(x[:2], zero, one, scale.view(1, experts * n, -1), group)
    q = qm.unpack_int4(one[0, -40:].contiguous())[None]
    moe_util.check_product(x[:2], zero, q, scale.view(1, experts * n, -1)[:, -40:].contiguous(), group, None, y[:, :, -40:])


def test_rows_behind_four_gigabytes():
    """Activations a gigabyte apart; products and sums of more elements than 32 bits count."""
    _, chosen, q, s = moe_util.problem(3, 2, 4, 64, 256, 64, torch.float16, torch.float16, 18)
    far = torch.zeros((1 << 31) + 256, dtype=torch.float16, device="cuda").as_strided((3, 256), (1 << 30, 1))
    far.copy_(torch.randn(3, 256, generator=torch.Generator().manual_seed(18)))
    moe_util.check_product(far, chosen, q, s, 64, None, moe.gemm_experts(far, chosen, moe_util.pack(q), s, 64))
    del far
    tokens, hidden, inner = 70000, 65536, 32
    g = torch.Generator(device="cuda").manual_seed(19)
    x = torch.randn(tokens, hidden, generator=g, device="cuda", dtype=torch.bfloat16)
    _, _, q_up, s_up = moe_util.problem(1, 1, 2, 2 * inner, hidden, 128, torch.bfloat16, torch.bfloat16, 20)
    _, _, q_down, s_down = moe_util.problem(1, 1, 2, hidden, inner, 128, torch.bfloat16, torch.bfloat16, 21)
    chosen = (torch.arange(tokens, device="cuda") % 2).to(torch.int32)[:, None].contiguous()
    weights = torch.rand(tokens, 1, generator=g, device="cuda")
    y = moe.mlp(x, chosen, weights, moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, 128)
    for some in (slice(0, 2), slice(32767, 32770), slice(65535, 65538), slice(tokens - 3, tokens)):
        moe_util.check_mlp(x[some], chosen[some], weights[some], q_up, s_up, q_down, s_down, 128, y[some])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 5, 70, 300])
def test_a_row_that_is_not_finite_is_so_in_all_columns(tokens, dtype):
    x, chosen, q, s = moe_util.problem(tokens, 2, 3, 64, 256, 64, dtype, dtype, 22)
    first = moe.gemm_experts(x, chosen, moe_util.pack(q), s, 64)
    for bad in (float("inf"), -float("inf"), float("nan")):
        lost = x.clone()
        lost[tokens // 2, 100] = bad
        y, others = moe.gemm_experts(lost, chosen, moe_util.pack(q), s, 64), torch.arange(tokens, device="cuda") != tokens // 2
        assert not y[tokens // 2].isfinite().any() and torch.equal(y[others], first[others])


@pytest.mark.parametrize("tokens", [1, 5, 70, 300])
@pytest.mark.parametrize("power", [-126, -110, 100])
def test_rows_of_any_size(power, tokens):
    """bf16 rows far from float16's range, each of another size; elements from there down to nothing in one row."""
    x, chosen, q, s = moe_util.problem(tokens, 2, 3, 64, 256, 64, torch.bfloat16, torch.float32, 23)
    x = torch.ldexp(x.float(), torch.full((tokens, 1), power, device="cuda") + torch.arange(tokens, device="cuda")[:, None] % 7)
    x[tokens - 1] = torch.ldexp(x[tokens - 1], -(torch.arange(256, device="cuda") % 60))
    x = x.to(torch.bfloat16)
    moe_util.check_product(x, chosen, q, s, 64, None, moe.gemm_experts(x, chosen, moe_util.pack(q), s, 64))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens,top_k,experts,hidden,inner,group", [(70, 2, 4, 256, 2112, 64), (40, 1, 1, 384, 4096, 128), (150, 2, 3, 288, 3104, 32), (300, 1, 4, 640, 9600, 128), (500, 2, 2, 4096, 2048, 256)])
def test_second_products_cut_along_k(tokens, top_k, experts, hidden, inner, group, dtype):
    gated(tokens, top_k, experts, hidden, inner, group, dtype, dtype, inner)
    gated(tokens, top_k, experts, hidden, inner, group, dtype, torch.float32, inner + 1, absent=0.3)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens,top_k,experts,n,k,group", [(140, 2, 4, 259, 2112, 64), (200, 1, 5, 36, 9312, 32), (64, 2, 2, 260, 8192, 128), (33, 1, 1, 7, 2304, 256)])
def test_products_cut_along_k(tokens, top_k, experts, n, k, group, dtype):
    product(tokens, top_k, experts, n, k, group, dtype, dtype, k, with_bias=True)
    product(tokens, top_k, experts, n, k, group, dtype, torch.float32, k + 1, per_choice=True, with_bias=n % 2 == 0, absent=0.3)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_cast_module_chooses_the_same_experts(dtype):
    """The usual cast of a model to its activations' type: float32 router, bias and scales stay, and so do the choices and every bit of the result."""
    g = torch.Generator().manual_seed(24)
    experts, hidden, inner, top_k = 16, 256, 64, 4
    _, _, q_up, s_up = moe_util.problem(1, 1, experts, 2 * inner, hidden, 64, dtype, torch.float32, 25)
    _, _, q_down, s_down = moe_util.problem(1, 1, experts, hidden, inner, 64, dtype, torch.float32, 26)
    router, bias = (torch.randn(experts, hidden, generator=g) / 16).cuda(), torch.randn(experts, generator=g).cuda() * 0.05
    layer = moe.SparseMLP(router, moe.W4A16Experts(moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, 64), top_k, bias, scores="sigmoid")
    x = torch.randn(50, hidden, generator=g).to(dtype).cuda()
    first, chosen = layer(x), moe.route(x.float() @ router.t(), top_k, bias=bias, scores="sigmoid")[0]
    for cast in (layer.half, layer.bfloat16, lambda: layer.to("cuda", torch.float16)):
        assert cast() is layer
        assert torch.equal(layer(x), first)
        assert torch.equal(moe.route(x.to(layer.router.dtype) @ layer.router.t(), top_k, bias=layer.bias, scores="sigmoid")[0], chosen)

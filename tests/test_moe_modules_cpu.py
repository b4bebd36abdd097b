"""The modules of the mixture of experts without a GPU: what a cast does to their tensors, and what their constructors refuse."""
import pytest
import torch

from quadmul_amd import QuadmulError, moe


def experts(scales=torch.float32, count=6, hidden=64, inner=32):
    g = torch.Generator().manual_seed(count)
    packed = lambda *shape: torch.randint(-128, 128, shape, dtype=torch.int8, generator=g)  # noqa: E731
    return moe.W4A16Experts(packed(count, 2 * inner, hidden // 2), torch.rand(count, 2 * inner, hidden // 32, generator=g).to(scales), packed(count, hidden, inner // 2),
                            torch.rand(count, hidden, inner // 32, generator=g).to(scales), 32)


def layer(scales=torch.float32, **rule):
    g = torch.Generator().manual_seed(1)
    return moe.SparseMLP(torch.randn(6, 64, generator=g), experts(scales), 2, torch.randn(6, generator=g), **rule)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float16)],
                         ids=["half", "bfloat16", "double", "to", "to_device"])
def test_a_cast_leaves_float32_as_it_is(cast):
    m = layer()
    before = {name: t.clone() for name, t in m.state_dict().items()}
    assert cast(m) is m
    after = m.state_dict()
    assert set(after) == set(before) == {"router", "bias", "experts.up_packed", "experts.up_scale", "experts.down_packed", "experts.down_scale"}
    assert all(after[name].dtype == t.dtype and torch.equal(after[name], t) for name, t in before.items())


def test_a_cast_of_sixteen_bits_is_one():
    m = layer(torch.float16)
    assert m.bfloat16().experts.up_scale.dtype == torch.bfloat16 and m.router.dtype == m.bias.dtype == torch.float32
    assert m.float().experts.down_scale.dtype == torch.float32


def test_a_cast_with_a_move():
    m = layer().to("meta", torch.bfloat16)
    assert all(t.is_meta for t in m.state_dict().values()) and m.bias.dtype == m.router.dtype == m.experts.up_scale.dtype == torch.float32
    m = moe.SparseMLP(torch.randn(6, 64), experts(), 2).half()  # no bias
    assert m.bias is None and m.router.dtype == torch.float32


@pytest.mark.parametrize("rule", [{"score": "sigmoid"}, {"renormalize": True}, {"scores": "tanh"}, {"groups": 4}, {"groups": 0}, {"groups": 3, "top_groups": 4}, {"groups": 6, "top_groups": 1},
                                  {"group_best": 3}], ids=str)
def test_options_that_route_would_refuse(rule):
    with pytest.raises(QuadmulError):
        layer(**rule)


def test_what_the_layer_refuses():
    router, e = torch.randn(6, 64), experts()
    for args in [(router, e, 0), (router, e, 7), (router[:5], e, 2), (router.double(), e, 2), (router.int(), e, 2), (router, e, 2, torch.zeros(5)), (router, e, 2, torch.zeros(6, 1)),
                 (router, e, 2, torch.zeros(6, dtype=torch.int32))]:
        with pytest.raises(QuadmulError):
            moe.SparseMLP(*args)
    for x in (torch.randn(3, 32), torch.randn(2, 3, 128)):
        with pytest.raises(QuadmulError):
            moe.SparseMLP(router, e, 2)(x)
    m = moe.SparseMLP(router, e, 2, torch.ones(6, dtype=torch.bfloat16), scores="sigmoid", groups=3, top_groups=1, group_best=1, renormalise=True, scale=2.5)
    assert m.bias.dtype == torch.float32 and m.bias.tolist() == [1.0] * 6

"""Products with experts' weights and their gated MLP at sizes far from one: activations, scales and weights of the choices of which some step on the way could leave float32's range
though the result does not, for few rows to an expert and for many."""
import math

import pytest
import torch

import moe_util
from quadmul_amd import moe

pytestmark = pytest.mark.gpu

TOKENS = [1, 5, 70, 300]


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("k,group", [(96, 32), (256, 64), (416, 128), (2304, 128), (66, 64)])
@pytest.mark.parametrize("down,up", [(-100, 115), (-126, 120), (-60, 126), (100, -120)])
def test_small_rows_and_large_scales(down, up, k, group, tokens):
    """bf16 rows of about 2^down (every third one no larger than ordinary ones), float32 scales of about 2^(up - 4)."""
    x, chosen, q, s = moe_util.problem(tokens, 2, 3, 40, k, group, torch.bfloat16, torch.float32, 31)
    x = torch.ldexp(x.float(), torch.where(torch.arange(tokens, device="cuda") % 3 == 2, min(down, 0), down)[:, None]).to(torch.bfloat16)
    s = (s.double() * 2.0 ** (up - 4 + math.floor(math.log2(math.sqrt(k) * 4.0)))).float()
    y = moe.gemm_experts(x, chosen, moe_util.pack(q), s, group)
    assert bool(y.isfinite().all())
    moe_util.check_product(x, chosen, q, s, group, None, y, near=True)


@pytest.mark.parametrize("tokens", [70, 300])
def test_a_row_keeps_its_bits_beside_one_that_is_summed_again(tokens):
    """Rows of a tile in which another one's sums pass float32's range before the row's power of two comes off."""
    x, chosen, q, s = moe_util.problem(tokens, 1, 2, 300, 640, 64, torch.bfloat16, torch.float32, 32)
    s[:, :, 3] *= 2.0 ** 115
    q[:, :, 192:256] = torch.where(q[:, :, 192:256] == 0, 1, q[:, :, 192:256])
    x[:, 192:256] = 0.0
    first = moe.gemm_experts(x, chosen, moe_util.pack(q), s, 64)
    small = torch.arange(tokens, device="cuda") % 5 == 1
    other = x.clone()
    other[small, 192:256] = 2.0 ** -100
    other[small, :192] *= 2.0 ** -90
    other[small, 256:] *= 2.0 ** -90
    again = moe.gemm_experts(other, chosen, moe_util.pack(q), s, 64)
    assert torch.equal(first[~small], again[~small]) and bool(again.isfinite().all())
    moe_util.check_product(other, chosen, q, s, 64, None, again, near=True)


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("hidden,inner,group", [(256, 96, 32), (384, 128, 128), (384, 2176, 64), (34, 6, 32)])
@pytest.mark.parametrize("rows,up,down", [(-100, 100, 0), (0, -30, 115), (0, 0, -40)])
def test_an_mlp_of_small_values_and_large_scales(rows, up, down, hidden, inner, group, tokens):
    """bf16 rows of about 2^rows, float32 scales of the first matrix 2^up and of the second 2^down times the usual ones."""
    x, chosen, q_up, s_up = moe_util.problem(tokens, 2, 3, 2 * inner, hidden, group, torch.bfloat16, torch.float32, 33)
    _, _, q_down, s_down = moe_util.problem(1, 1, 3, hidden, inner, group, torch.bfloat16, torch.float32, 34)
    x, s_up, s_down = ((t.double() * 2.0 ** by).to(t.dtype) for t, by in ((x, rows), (s_up, up), (s_down, down)))
    weights = torch.rand(tokens, 2, generator=torch.Generator().manual_seed(35)).cuda()
    y = moe.mlp(x, chosen, weights, moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, group)
    assert bool(y.isfinite().all())
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, group, y, near=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("k,group", [(66, 32), (64, 32), (256, 128)])
def test_the_largest_scales(k, group, tokens, dtype):
    """Scales of which eight are no float32 any more, under small rows."""
    x, chosen, q, s = moe_util.problem(tokens, 2, 3, 40, k, group, dtype, torch.float32, 36)
    x, s = (x.double() * 2.0 ** (-60 if dtype == torch.bfloat16 else -14)).to(dtype), torch.full_like(s, 2.0 ** (127 if dtype == torch.bfloat16 else 10))
    y = moe.gemm_experts(x, chosen, moe_util.pack(q), s, group)
    assert bool(y.isfinite().all())
    moe_util.check_product(x, chosen, q, s, group, None, y, near=True)
    _, _, q_down, s_down = moe_util.problem(1, 1, 3, k, 20, group, dtype, torch.float32, 37)
    s.fill_(2.0 ** (127 if dtype == torch.bfloat16 else 10))
    x = (x.double() * (2.0 ** -70 if dtype == torch.bfloat16 else 1.0)).to(dtype)
    weights = torch.rand(tokens, 2, generator=torch.Generator().manual_seed(38)).cuda()
    y = moe.mlp(x, chosen, weights, moe_util.pack(q), s, moe_util.pack(q_down), s_down, group)
    assert bool(y.isfinite().all())
    moe_util.check_mlp(x, chosen, weights, q, s, q_down, s_down, group, y, near=True)


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("hidden,inner,group", [(256, 96, 32), (384, 320, 64), (384, 128, 128), (34, 6, 32)])
@pytest.mark.parametrize("rows,down,share", [(40, -100, -50), (-30, 100, 60)])
def test_weights_of_the_choices_beside_scales(rows, down, share, hidden, inner, group, tokens):
    """bf16 rows of about 2^rows; the weight of a choice times a scale of the second matrix alone is below float32's normal numbers, or above its largest."""
    x, chosen, q_up, s_up = moe_util.problem(tokens, 2, 3, 2 * inner, hidden, group, torch.bfloat16, torch.float32, 39)
    _, _, q_down, s_down = moe_util.problem(1, 1, 3, hidden, inner, group, torch.bfloat16, torch.float32, 40)
    x, s_down = (x.double() * 2.0 ** rows).to(x.dtype), (s_down.double() * 2.0 ** down).float()
    weights = ((torch.rand(tokens, 2, generator=torch.Generator().manual_seed(41)).double() + 0.5) * 2.0 ** share).float().cuda()
    y = moe.mlp(x, chosen, weights, moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, group)
    assert bool(y.isfinite().all())
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, group, y, near=True)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [70, 300, 1100])
def test_bits_of_the_rows_beside_sums_made_again(tokens, group):
    """Every fifth row's sums pass float32's range before its power of two comes off; the others meet the large scales with zeros, and keep their bits."""
    x, chosen, q, s = moe_util.problem(tokens, 1, 1, 300, 672, group, torch.bfloat16, torch.float32, 42)
    some = slice(group, 2 * group)  # the second group
    s[:, :, 1] = 2.0 ** 120
    x[:, some] = 0.0
    first = moe.gemm_experts(x, chosen, moe_util.pack(q), s, group)
    small = torch.arange(tokens, device="cuda") % 5 == 1
    other = x.clone()
    other[small] *= 2.0 ** -100
    other[small, some] = 2.0 ** -100
    again = moe.gemm_experts(other, chosen, moe_util.pack(q), s, group)
    assert torch.equal(first[~small], again[~small]) and bool(again.isfinite().all())
    moe_util.check_product(other, chosen, q, s, group, None, again, near=True)


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("hidden,inner,group", [(256, 96, 32), (384, 320, 64), (384, 128, 128), (34, 6, 32)])
def test_small_weights_of_the_choices_beside_small_scales(hidden, inner, group, tokens):
    """Gates of ordinary size and large values: the weight of a choice times a scale of the second matrix is nothing in float32, the result is not."""
    x, chosen, q_up, s_up = moe_util.problem(tokens, 2, 3, 2 * inner, hidden, group, torch.bfloat16, torch.float32, 43)
    _, _, q_down, s_down = moe_util.problem(1, 1, 3, hidden, inner, group, torch.bfloat16, torch.float32, 44)
    s_up[:, inner:] *= 2.0 ** 80
    s_down *= 2.0 ** -100
    weights = ((torch.rand(tokens, 2, generator=torch.Generator().manual_seed(45)) + 0.5) * 2.0 ** -50).cuda()
    y = moe.mlp(x, chosen, weights, moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, group)
    assert bool((y != 0.0).any())
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, group, y, near=True)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("tokens", [70, 300, 1100])
def test_rows_that_are_not_finite_beside_sums_made_again(tokens, bad):
    """Padding that is no number, in tiles with and without rows whose sums leave float32's range."""
    x, chosen, q, s = moe_util.problem(tokens, 1, 1, 300, 672, 64, torch.bfloat16, torch.float32, 46)
    s[:, :, 1] = 2.0 ** 120
    x[:, 64:128] = 0.0
    number = torch.arange(tokens, device="cuda")
    small, lost = number % 7 == 1, number % 5 == 2
    x[small & (number > 40)] *= 2.0 ** -100
    x[small & (number > 40), 64:128] = 2.0 ** -100
    first = moe.gemm_experts(x, chosen, moe_util.pack(q), s, 64)
    moe_util.check_product(x, chosen, q, s, 64, None, first, near=True)
    other = x.clone()
    other[lost, 100] = bad
    again = moe.gemm_experts(other, chosen, moe_util.pack(q), s, 64)
    assert torch.equal(first[~lost], again[~lost]) and not bool(again[lost].isfinite().any())


@pytest.mark.parametrize("tokens,k,group", [(1, 66, 32), (5, 66, 64), (300, 66, 32), (300, 96, 32), (300, 256, 128)])
@pytest.mark.parametrize("power,up", [(126, -30), (127, -126)])
def test_the_largest_elements(power, up, k, group, tokens):
    """bf16 elements of which eight are no float32 any more, under small scales, where the weights take part as they are."""
    x, chosen, q, s = moe_util.problem(tokens, 2, 3, 40, k, group, torch.bfloat16, torch.float32, 47)
    x, s = (torch.sign(x.double()) * 2.0 ** power).to(torch.bfloat16), torch.full_like(s, 2.0 ** up)
    y = moe.gemm_experts(x, chosen, moe_util.pack(q), s, group)
    assert bool(y.isfinite().all())
    moe_util.check_product(x, chosen, q, s, group, None, y, near=True)

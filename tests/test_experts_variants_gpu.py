"""Every kernel that the sizes of a call can lead to, products and gated MLPs, within bounds that would see one wrong scale among hundreds: heights of tiles of 2 to 64 rows, found
by the kernel or from lists, four, eight and sixteen waves, groups of 32 to 384, rows at any address."""
import ctypes

import pytest
import torch

import moe_util
import quadmul_amd as qm
from quadmul_amd import moe
from test_experts_gpu import MLPS, SIZES

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]
IDS = ["f16", "bf16"]


def product(tokens, top_k, experts, n, k, group, dtype, scales, seed, per_choice=False, with_bias=False, **how):
    x, chosen, q, s = moe_util.problem(tokens, top_k, experts, n, k, group, dtype, scales, seed, **how)
    g = torch.Generator().manual_seed(seed + 1)
    if per_choice:
        x = (torch.randn(tokens, top_k, k, generator=g) * 2.0).to(dtype).cuda()
    bias = torch.randn(experts, n, generator=g).to(dtype).cuda() if with_bias else None
    moe_util.check_product(x, chosen, q, s, group, bias, moe.gemm_experts(x, chosen, moe_util.pack(q), s, group, bias), near=True)


def gated(tokens, top_k, experts, hidden, inner, group, dtype, scales, seed, **how):
    x, chosen, q_up, s_up = moe_util.problem(tokens, top_k, experts, 2 * inner, hidden, group, dtype, scales, seed, **how)
    _, _, q_down, s_down = moe_util.problem(1, 1, experts, hidden, inner, group, dtype, scales, seed + 1)
    weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(seed + 2)).cuda()
    y = moe.mlp(x, chosen, weights, moe_util.pack(q_up), s_up, moe_util.pack(q_down), s_down, group)
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, group, y, near=True)


PRODUCTS = (
    [(24, 8, 64, 100, 384, g) for g in (32, 64, 128)]  # 8 rows, from a list
    + [(32, 8, 128, 100, 384, g) for g in (32, 64, 128)]  # 4 rows, from a list
    + [(48, 8, 64, 100, 384, g) for g in (32, 64, 128)]  # 16 rows, from a list
    + [(8, 4, 10, 100, 384, g) for g in (32, 64, 128)] + [(3, 4, 10, 100, 384, 64)]  # 8 and 4 rows, found by the kernel
    + [(12, 1, 1, 100, 4160, g) for g in (32, 64, 128)] + [(12, 2, 4, 100, 4160, 128)]  # eight waves, 16 rows
    + [(5, 2, 3, 100, 4160, g) for g in (32, 64, 128)]  # eight waves, 8 rows
    + [(3, 2, 3, 100, 4160, 64), (1, 2, 3, 100, 4160, 32)]  # eight waves, 4 and 2 rows
    + [(1100, 1, 1, 140, 160, g) for g in (32, 64, 128)] + [(1600, 1, 1, 516, 1024, 64)]  # tiles of 64 rows, K in one piece
    + [(t, k, e, n, 1152, g) for t, k, e, n in ((4, 2, 8, 70), (40, 2, 8, 70), (300, 2, 3, 130), (1100, 2, 2, 66)) for g in (96, 192, 384)]  # groups of some blocks
    + [(700, 1, 2, 520, 2176, 192), (90, 1, 2, 260, 8448, 384)]  # tiles of 32 and of 64 rows, K in parts
)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("wide", [False, True], ids=["scales16", "scales32"])
@pytest.mark.parametrize("tokens,top_k,experts,n,k,group", PRODUCTS + SIZES)
def test_products(tokens, top_k, experts, n, k, group, wide, dtype):
    scales = torch.float32 if wide else dtype
    product(tokens, top_k, experts, n, k, group, dtype, scales, 3 * tokens + n + k, with_bias=True)
    product(tokens, top_k, experts, n, k, group, dtype, scales, 5 * tokens + n + k, per_choice=True, absent=0.3)


GATED = (
    [(8, 8, 128, 1024, 128, g) for g in (32, 64, 128)] + [(4, 8, 64, 1056, 160, 32)]  # a token's choices added up on the way, 32 columns to an item
    + [(24, 8, 64, 256, 256, g) for g in (64, 128)] + [(24, 8, 64, 288, 160, 32)]  # 8 rows, from a list
    + [(32, 8, 128, 256, 128, g) for g in (64, 128)] + [(32, 8, 128, 288, 96, 32)]  # 4 rows, from a list
    + [(48, 8, 64, 256, 256, 128), (48, 8, 64, 256, 128, 64), (48, 8, 64, 256, 96, 32)]  # 16 rows, from a list
    + [(8, 4, 10, 384, 256, 128), (8, 4, 10, 384, 160, 32)]  # 8 rows, found by the kernel
    + [(12, 1, 1, 4160, 64, 128), (12, 1, 2, 64, 4160, 128), (5, 2, 3, 4160, 96, 32), (5, 2, 3, 96, 4160, 64)]  # eight waves, 16 and 8 rows
    + [(1, 2, 6, 1152, 384, 192), (1, 2, 6, 1152, 384, 384), (40, 2, 8, 1152, 384, 192), (40, 2, 8, 768, 384, 384), (300, 2, 3, 384, 576, 192), (300, 2, 3, 768, 384, 384)]
    + [(1100, 1, 1, 384, 160, 32), (1100, 2, 3, 256, 192, 64), (90, 1, 2, 320, 2176, 192), (150, 2, 3, 288, 3104, 32)]
)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("wide", [False, True], ids=["scales16", "scales32"])
@pytest.mark.parametrize("tokens,top_k,experts,hidden,inner,group", GATED + MLPS)
def test_mlps(tokens, top_k, experts, hidden, inner, group, wide, dtype):
    scales = torch.float32 if wide else dtype
    gated(tokens, top_k, experts, hidden, inner, group, dtype, scales, 3 * tokens + hidden)
    gated(tokens, top_k, experts, hidden, inner, group, dtype, scales, 5 * tokens + inner, absent=0.4)


@pytest.mark.parametrize("tokens", [1, 5, 40, 200])
@pytest.mark.parametrize("off", [1, 4])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_rows_of_the_c_entries_at_any_address(dtype, off, tokens):
    """The C entries take x as it is (the Python calls copy such rows first): tiles of few rows."""
    lib, code, stream = qm.library(), 1 if dtype == torch.float16 else 2, torch.cuda.current_stream().cuda_stream
    experts, hidden, inner, group, top_k = 6, 416, 96, 32, 2
    x, chosen, q_up, s_up = moe_util.problem(tokens, top_k, experts, 2 * inner, hidden, group, dtype, torch.float32, 51)
    _, _, q_down, s_down = moe_util.problem(1, 1, experts, hidden, inner, group, dtype, torch.float32, 52)
    weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(53)).cuda()
    apart = torch.zeros(tokens * (hidden + 2) + off, dtype=dtype, device="cuda")
    rows = apart[off:].view(tokens, hidden + 2)[:, :hidden]
    rows.copy_(x)
    w_up, w_down = moe_util.pack(q_up), moe_util.pack(q_down)
    up = qm.ExpertWeights(w_up.data_ptr(), s_up.data_ptr(), None, 3, experts, 2 * inner, hidden, group)
    down = qm.ExpertWeights(w_down.data_ptr(), s_down.data_ptr(), None, 3, experts, hidden, inner, group)
    need = max(lib.qm_gemm_experts_workspace_bytes(ctypes.byref(up), tokens, top_k), lib.qm_moe_mlp_workspace_bytes(ctypes.byref(up), ctypes.byref(down), tokens, top_k))
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    y, z = torch.empty(tokens, top_k, 2 * inner, dtype=dtype, device="cuda"), torch.empty(tokens, hidden, dtype=dtype, device="cuda")
    assert lib.qm_gemm_experts_i4(rows.data_ptr(), code, hidden + 2, 0, chosen.data_ptr(), ctypes.byref(up), y.data_ptr(), tokens, top_k, stream, scratch.data_ptr(), need) == 0
    moe_util.check_product(x, chosen, q_up, s_up, group, None, y, near=True)
    assert lib.qm_moe_mlp_i4(rows.data_ptr(), code, hidden + 2, chosen.data_ptr(), weights.data_ptr(), ctypes.byref(up), ctypes.byref(down), z.data_ptr(), tokens, top_k, stream,
                             scratch.data_ptr(), need) == 0
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, group, z, near=True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 6, 300])
def test_small_elements_beside_a_large_one_that_no_weight_meets(dtype, tokens):
    """What is left of a row when its largest elements meet zeros."""
    x, chosen, q, s = moe_util.problem(tokens, 2, 3, 70, 512, 64, dtype, dtype, 54)
    q[:, :, ::64] = 0
    x[:, ::64] = 2.0 ** 12 if dtype == torch.bfloat16 else 60000.0
    x[:, 1::2] *= 2.0 ** -8
    moe_util.check_product(x, chosen, q, s, 64, None, moe.gemm_experts(x, chosen, moe_util.pack(q), s, 64), near=True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 6, 40, 300])
def test_matrices_with_groups_and_scales_of_their_own(dtype, tokens):
    """The C entry takes groups of another size, and scales of another type, for each of the two matrices."""
    lib, code, stream = qm.library(), 1 if dtype == torch.float16 else 2, torch.cuda.current_stream().cuda_stream
    experts, hidden, inner, top_k = 5, 384, 192, 2
    for (g_up, s_up_type), (g_down, s_down_type) in [((128, dtype), (32, torch.float32)), ((32, torch.float32), (64, dtype)), ((384, torch.float32), (96, torch.float32))]:
        x, chosen, q_up, s_up = moe_util.problem(tokens, top_k, experts, 2 * inner, hidden, g_up, dtype, s_up_type, 55)
        _, _, q_down, s_down = moe_util.problem(1, 1, experts, hidden, inner, g_down, dtype, s_down_type, 56)
        weights = torch.rand(tokens, top_k, generator=torch.Generator().manual_seed(57)).cuda()
        w_up, w_down = moe_util.pack(q_up), moe_util.pack(q_down)
        up = qm.ExpertWeights(w_up.data_ptr(), s_up.data_ptr(), None, 3 if s_up_type == torch.float32 else code, experts, 2 * inner, hidden, g_up)
        down = qm.ExpertWeights(w_down.data_ptr(), s_down.data_ptr(), None, 3 if s_down_type == torch.float32 else code, experts, hidden, inner, g_down)
        need = lib.qm_moe_mlp_workspace_bytes(ctypes.byref(up), ctypes.byref(down), tokens, top_k)
        scratch, y = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(tokens, hidden, dtype=dtype, device="cuda")
        assert lib.qm_moe_mlp_i4(x.data_ptr(), code, hidden, chosen.data_ptr(), weights.data_ptr(), ctypes.byref(up), ctypes.byref(down), y.data_ptr(), tokens, top_k, stream,
                                 scratch.data_ptr(), need) == 0
        # (the bounds take one size of groups: scales repeated to that of the smallest common one)
        s_up, s_down = s_up.repeat_interleave(g_up // 32, dim=2)[..., :-(-hidden // 32)], s_down.repeat_interleave(g_down // 32, dim=2)[..., :-(-inner // 32)]
        moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, 32, y, near=True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 6, 40, 300])
def test_rows_in_another_order(dtype, tokens):
    """A row for each choice, the choices outside the tokens; and rows that all choices of all tokens share."""
    _, chosen, q, s = moe_util.problem(tokens, 3, 5, 90, 384, 64, dtype, dtype, 58)
    w, each = moe_util.pack(q), torch.randn(3, tokens, 384, generator=torch.Generator().manual_seed(59)).to(dtype).cuda()
    for x in (each.transpose(0, 1), each[:, :1].transpose(0, 1).expand(tokens, 3, 384), each[0, 0].expand(tokens, 3, 384)):
        moe_util.check_product(x, chosen, q, s, 64, None, moe.gemm_experts(x, chosen, w, s, 64), near=True)


@pytest.mark.parametrize("tokens", [1, 6, 300])
def test_weights_of_the_choices_that_are_not_finite(tokens):
    """They make their own token's row infinite or NaN and no other one's; those of choices without an expert count for nothing."""
    x, chosen, q, s = moe_util.problem(tokens, 3, 6, 64, 256, 64, torch.bfloat16, torch.bfloat16, 60)
    _, _, q2, s2 = moe_util.problem(1, 1, 6, 256, 32, 64, torch.bfloat16, torch.bfloat16, 61)
    weights = torch.rand(tokens, 3, generator=torch.Generator().manual_seed(62)).cuda()
    call = lambda c, w: moe.mlp(x, c, w, moe_util.pack(q), s, moe_util.pack(q2), s2, 64)  # noqa: E731
    first, row = call(chosen, weights), tokens // 2
    others = torch.arange(tokens, device="cuda") != row
    for bad in (float("inf"), -float("inf"), float("nan")):
        lost = weights.clone()
        lost[row, 1] = bad
        y = call(chosen, lost)
        assert not y[row].isfinite().any() and torch.equal(y[others], first[others])
        nobody = chosen.clone()
        nobody[row, 1] = -1
        assert call(nobody, lost).isfinite().all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tokens", [1, 3, 40, 300])
@pytest.mark.parametrize("top_k,experts", [(2, 3), (4, 40)])
@pytest.mark.parametrize("hidden,inner,group", [(34, 64, 32), (130, 96, 32), (96, 34, 32), (256, 34, 64), (258, 128, 128)])
def test_one_matrix_for_the_matrix_cores_and_one_not(hidden, inner, group, top_k, experts, tokens, dtype):
    """A hidden or an inner size that is no multiple of 32: the two products run on kernels of different kinds."""
    gated(tokens, top_k, experts, hidden, inner, group, dtype, dtype, tokens + hidden, absent=0.2)


@pytest.mark.parametrize("tokens", [1, 5, 60, 300])
@pytest.mark.parametrize("up_off,down_off", [(0, 8), (8, 0)])
def test_one_matrix_at_sixteen_bytes_and_one_not(up_off, down_off, tokens):
    x, chosen, q_up, s_up = moe_util.problem(tokens, 2, 5, 128, 256, 64, torch.float16, torch.float16, 63)
    _, _, q_down, s_down = moe_util.problem(1, 1, 5, 256, 64, 64, torch.float16, torch.float16, 64)
    at = lambda t, off: torch.zeros(t.numel() + off, dtype=t.dtype, device="cuda")[off:].view(t.shape).copy_(t)  # noqa: E731
    weights = torch.rand(tokens, 2, generator=torch.Generator().manual_seed(65)).cuda()
    y = moe.mlp(x, chosen, weights, at(moe_util.pack(q_up), up_off), s_up, at(moe_util.pack(q_down), down_off), s_down, 64)
    moe_util.check_mlp(x, chosen, weights, q_up, s_up, q_down, s_down, 64, y, near=True)

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

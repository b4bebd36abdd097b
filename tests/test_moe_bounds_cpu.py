"""The bounds that the products of the mixture of experts are held to: the exact result, rounded once, is within them, and one wrong scale, one wrong weight in sixty-four or a missing
run of K is not. On the host, against a mistake planted in what is expected."""
import pytest
import torch

import moe_util

SIZES = [(200, 1, 5, 36, 9312, 32), (64, 2, 2, 60, 8192, 128), (3, 2, 4, 7, 8192, 128), (2, 2, 4, 40, 14336, 128), (13, 4, 16, 60, 672, 96), (300, 4, 8, 60, 288, 32)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("tokens,top_k,experts,n,k,group", SIZES)
def test_one_wrong_scale_is_seen(tokens, top_k, experts, n, k, group, dtype):
    x, chosen, q, s = moe_util.problem(tokens, top_k, experts, n, k, group, dtype, torch.float32, 61, device="cpu")
    w = moe_util.values(q, s, group)
    y = torch.stack([torch.stack([w[e] @ x[t].double() for e in chosen[t].tolist()]) for t in range(tokens)]).to(dtype)
    moe_util.check_product(x, chosen, q, s, group, None, y, near=True)

    def seen(q, s):
        with pytest.raises(AssertionError):
            moe_util.check_product(x, chosen, q, s, group, None, y, near=True)

    groups = s.shape[2]
    for g in (0, groups // 2, groups - 1):
        wrong = s.clone()
        wrong[:, :, g] = s[:, :, (g + 1) % groups]
        seen(q, wrong)
    wrong = q.clone()
    wrong[:, :, ::64] = 0
    seen(wrong, s)
    wrong = q.clone()
    wrong[:, :, -32:] = 0
    seen(wrong, s)

"""The mixture of experts at the ends of its index ranges: columns and tokens that 31 bits just count."""
import ctypes

import pytest
import torch

import quadmul_amd as qm

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gives_memory_back")]


@pytest.mark.parametrize("top_k", [0, 1])
@pytest.mark.parametrize("hidden", [2 ** 30 + 2, 2 ** 31 - 4, 2 ** 31 - 2])
def test_sums_of_the_most_columns(hidden, top_k):
    """An MLP without inner columns: sums of nothing, zeros in every column, and what lies behind the last one is left alone."""
    lib = qm.library()
    up, down = qm.ExpertWeights(None, None, None, 1, 1, 0, hidden, 32), qm.ExpertWeights(None, None, None, 1, 1, hidden, 0, 32)
    y = torch.empty(hidden + 512, dtype=torch.float16, device="cuda").fill_(7.0)
    x = torch.empty(hidden, dtype=torch.float16, device="cuda")
    chosen, weights = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, 1, device="cuda")
    need = lib.qm_moe_mlp_workspace_bytes(ctypes.byref(up), ctypes.byref(down), 1, top_k)
    scratch = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    at = y[256:]  # as many elements in front of the result as behind it
    st = lib.qm_moe_mlp_i4(x.data_ptr(), 1, hidden, chosen.data_ptr(), weights.data_ptr(), ctypes.byref(up), ctypes.byref(down), at.data_ptr(), 1, top_k,
                           torch.cuda.current_stream().cuda_stream, scratch.data_ptr(), need)
    assert st == 0
    torch.cuda.synchronize()
    assert not at[:hidden].any() and bool((y[:256] == 7.0).all()) and bool((at[hidden:] == 7.0).all())


@pytest.mark.parametrize("tokens", [2 ** 31 - 1, 2 ** 31 - 15])
def test_choices_of_the_most_tokens(tokens):
    """One expert: it is chosen, with a weight of one, by every token up to the last."""
    logits = torch.zeros(tokens, 1, dtype=torch.float16, device="cuda")
    chosen = torch.full((tokens + 64,), 9, dtype=torch.int32, device="cuda")
    weights = torch.full((tokens + 64,), 9.0, device="cuda")
    st = qm.library().qm_moe_route(logits.data_ptr(), 1, 1, tokens, 1, 1, None, 0, 1, 1, 1, 0, 1.0, chosen.data_ptr(), weights.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert st == 0
    torch.cuda.synchronize()
    assert not chosen[:tokens].any() and bool((weights[:tokens] == 1.0).all())
    assert bool((chosen[tokens:] == 9).all()) and bool((weights[tokens:] == 9.0).all())

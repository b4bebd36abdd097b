"""Argument checks of the C entries of the mixture of experts, and the sizes of their workspaces: no kernel is launched."""
import ctypes

import pytest
import torch

import quadmul_amd as qm

ONE = 4096  # never dereferenced: the checks come first


def test_route_status_codes():
    lib = qm.library()

    def f(logits=ONE, dtype=3, stride=64, tokens=4, experts=64, top_k=4, bias=None, scores=0, groups=1, top_groups=1, best=2, chosen=ONE, weights=ONE):
        return lib.qm_moe_route(logits, dtype, stride, tokens, experts, top_k, bias, scores, groups, top_groups, best, 0, 1.0, chosen, weights, None)

    for bad, code in (({"dtype": 0}, -6), ({"dtype": 4}, -6), ({"tokens": -1}, -2), ({"experts": 0}, -2), ({"experts": 1025, "stride": 2000}, -2), ({"top_k": 0}, -2), ({"top_k": 65}, -2),
                      ({"groups": 0}, -2), ({"groups": 3}, -2), ({"groups": 65, "experts": 130, "stride": 130}, -2), ({"groups": 8, "top_groups": 9}, -2), ({"groups": 8, "top_groups": 0}, -2),
                      ({"groups": 8, "top_groups": 1, "top_k": 9}, -2), ({"best": 0}, -2), ({"best": 3}, -2), ({"scores": 2}, -2), ({"scores": -1}, -2), ({"stride": 63}, -2),
                      ({"logits": None}, -1), ({"chosen": None}, -1), ({"weights": None}, -1), ({"logits": ONE + 2}, -5), ({"logits": ONE + 1, "dtype": 1}, -5), ({"chosen": ONE + 2}, -5),
                      ({"bias": ONE + 1}, -5), ({"weights": ONE + 3}, -5)):
        assert f(**bad) == code, bad
    assert f(tokens=0, logits=None, chosen=None, weights=None) == 0


def matrices(**changes):
    w = qm.ExpertWeights(ONE, ONE, None, 1, 8, 256, 128, 64)
    for k, v in changes.items():
        setattr(w, k, v)
    return ctypes.byref(w)


BAD = [({"experts": -1}, -2), ({"n": -1}, -2), ({"k": -2}, -2), ({"k": 127}, -2), ({"group": 0}, -2), ({"group": 48}, -2), ({"weight": None}, -1), ({"scale": None}, -1), ({"scale_dtype": 2}, -6),
       ({"scale_dtype": 0}, -6), ({"scale": ONE + 1}, -5), ({"scale": ONE + 2, "scale_dtype": 3}, -5)]


def test_product_status_codes():
    lib = qm.library()

    def f(w=None, x=ONE, dtype=1, token=128, choice=0, chosen=ONE, y=ONE, tokens=3, top_k=2, ws=ONE, ws_bytes=1 << 30):
        return lib.qm_gemm_experts_i4(x, dtype, token, choice, chosen, w or matrices(), y, tokens, top_k, None, ws, ws_bytes)

    for bad, code in BAD + [({"bias": ONE + 1}, -5)]:
        assert f(matrices(**bad)) == code, bad
    for bad, code in (({"dtype": 3}, -6), ({"tokens": -1}, -2), ({"top_k": -1}, -2), ({"tokens": 1 << 20, "top_k": 1 << 12}, -2), ({"token": -1}, -2), ({"choice": -1}, -2), ({"x": None}, -1),
                      ({"chosen": None}, -1), ({"y": None}, -1), ({"x": ONE + 1}, -5), ({"y": ONE + 1}, -5), ({"chosen": ONE + 2}, -5), ({"ws": ONE + 8}, -5)):
        assert f(**bad) == code, bad
    assert f(tokens=0, x=None, y=None, chosen=None) == 0 and f(top_k=0, x=None, y=None, chosen=None) == 0 and f(matrices(n=0), y=None) == 0
    assert lib.qm_gemm_experts_i4(ONE, 1, 128, 0, ONE, None, ONE, 3, 2, None, None, 0) == -1
    need = lib.qm_gemm_experts_workspace_bytes(matrices(), 3, 2)
    if need:
        assert f(ws_bytes=need - 1) == -7 and f(ws=None) == -7
    assert lib.qm_gemm_experts_workspace_bytes(matrices(group=48), 3, 2) == 0 and lib.qm_gemm_experts_workspace_bytes(None, 3, 2) == 0 and lib.qm_gemm_experts_workspace_bytes(matrices(), -1, 2) == 0


def test_mlp_status_codes():
    lib = qm.library()

    def f(up=None, down=None, x=ONE, dtype=1, token=128, chosen=ONE, weights=ONE, y=ONE, tokens=3, top_k=2, ws=ONE, ws_bytes=1 << 30):
        return lib.qm_moe_mlp_i4(x, dtype, token, chosen, weights, up or matrices(), down or matrices(n=128, k=128), y, tokens, top_k, None, ws, ws_bytes)

    for bad, code in BAD:
        assert f(up=matrices(**bad)) == code, bad
        assert f(down=matrices(**({"n": 128, "k": 128} | bad))) == code, bad
    for bad, code in (({"up": matrices(n=250)}, -2), ({"up": matrices(k=256)}, -2), ({"up": matrices(experts=7)}, -2), ({"up": matrices(bias=ONE)}, -2), ({"down": matrices(n=128, k=128, bias=ONE)}, -2),
                      ({"dtype": 3}, -6), ({"tokens": -1}, -2), ({"top_k": -1}, -2), ({"tokens": 1 << 20, "top_k": 1 << 12}, -2), ({"token": -1}, -2), ({"x": None}, -1), ({"chosen": None}, -1),
                      ({"weights": None}, -1), ({"y": None}, -1), ({"x": ONE + 1}, -5), ({"y": ONE + 1}, -5), ({"chosen": ONE + 2}, -5), ({"weights": ONE + 2}, -5), ({"ws": ONE + 8}, -5)):
        assert f(**bad) == code, bad
    assert f(tokens=0, x=None, y=None, chosen=None, weights=None) == 0
    need = lib.qm_moe_mlp_workspace_bytes(matrices(), matrices(n=128, k=128), 3, 2)
    assert need >= 3 * 2 * (128 * 2) and f(ws_bytes=need - 1) == -7 and f(ws=None) == -7
    assert lib.qm_moe_mlp_workspace_bytes(matrices(), matrices(n=64, k=128), 3, 2) == 0 and lib.qm_moe_mlp_workspace_bytes(None, matrices(), 3, 2) == 0


def test_traceable_forms():
    import quadmul  # noqa: F401  (registers the operators)

    ops, meta = torch.ops.quadmul, lambda *s, dtype=torch.float16: torch.empty(s, dtype=dtype, device="meta")
    chosen, weights = ops.moe_route(meta(5, 64), 4, None, True, 8, 4, 2, True, 2.5)
    assert chosen.shape == weights.shape == (5, 4) and chosen.dtype == torch.int32 and weights.dtype == torch.float32
    w, s = meta(8, 256, 64, dtype=torch.int8), meta(8, 256, 2)
    for x in (meta(5, 128), meta(5, 4, 128)):
        y = ops.gemm_experts(x, chosen, w, s, 64, None)
        assert y.shape == (5, 4, 256) and y.dtype == torch.float16
    assert ops.moe_mlp(meta(5, 128), chosen, weights, w, s, meta(8, 128, 64, dtype=torch.int8), meta(8, 128, 2), 64).shape == (5, 128)
    for bad in (lambda: ops.moe_route(meta(5, 64), 65, None, True, 1, 1, 2, True, 1.0), lambda: ops.gemm_experts(meta(5, 130), chosen, w, s, 64, None),
                lambda: ops.moe_mlp(meta(5, 128), chosen, weights, w, s, meta(8, 64, 64, dtype=torch.int8), meta(8, 64, 2), 64)):
        with pytest.raises(RuntimeError):
            bad()


def test_workspaces_of_the_longest_rows():
    lib, longest = qm.library(), 2 ** 31 - 2
    # (one row: what lists there are, and no copy of a row that no tiles take)
    assert 0 < lib.qm_gemm_experts_workspace_bytes(matrices(experts=1, n=1, k=longest), 1, 1) < 4096
    # (a row of gated products in 16 bits, a row of sums in 32)
    need = lib.qm_moe_mlp_workspace_bytes(matrices(experts=1, n=4, k=longest), matrices(experts=1, n=longest, k=2), 1, 1)
    assert 0 <= need - 4 * longest < 4096
    need = lib.qm_moe_mlp_workspace_bytes(matrices(experts=1, n=2 ** 31 - 4, k=2), matrices(experts=1, n=2, k=2 ** 30 - 2), 1, 1)
    assert 0 <= need - 2 * (2 ** 30 - 2) < 4096


def test_the_most_choices():
    """The kernels step through a token's choices, and through the slots of an expert, by up to 64: so many below 2^31 are refused."""
    lib, w, down, most = qm.library(), matrices(), matrices(n=128, k=128), 2 ** 31 - 64
    for tokens, top_k, code in ((1, most, -7), (1, most + 1, -2), (1, 2 ** 31 - 1, -2), (most, 1, -7), (2 ** 31 - 1, 1, -2), (2, 2 ** 30 - 32, -7), (2, 2 ** 30 - 31, -2)):
        assert lib.qm_gemm_experts_i4(ONE, 1, 128, 0, ONE, w, ONE, tokens, top_k, None, None, 0) == code
        assert lib.qm_moe_mlp_i4(ONE, 1, 128, ONE, ONE, w, down, ONE, tokens, top_k, None, None, 0) == code
        assert (lib.qm_gemm_experts_workspace_bytes(w, tokens, top_k) > 0) == (lib.qm_moe_mlp_workspace_bytes(w, down, tokens, top_k) > 0) == (code == -7)


def test_workspaces_go_by_sizes_alone():
    """A program may ask for them before its weights are anywhere."""
    lib, nowhere = qm.library(), {"weight": None, "scale": None}
    for tokens, top_k in ((1, 2), (40, 2), (700, 4)):
        need = lib.qm_gemm_experts_workspace_bytes(matrices(), tokens, top_k)
        assert need > 0 and lib.qm_gemm_experts_workspace_bytes(matrices(**nowhere), tokens, top_k) == need
        need = lib.qm_moe_mlp_workspace_bytes(matrices(), matrices(n=128, k=128), tokens, top_k)
        assert need > 0 and lib.qm_moe_mlp_workspace_bytes(matrices(**nowhere), matrices(n=128, k=128, **nowhere), tokens, top_k) == need
    assert lib.qm_gemm_experts_workspace_bytes(matrices(k=127, **nowhere), 3, 2) == 0

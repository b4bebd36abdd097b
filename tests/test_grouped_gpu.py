"""16-bit activations times packed int4 weights with group scales (csrc/qm_grouped.hpp) against the sum in 64 bits: every kernel that the choice
leads to, both types, scales of both kinds, odd sizes, rows at a distance, groups that end early."""
import math

import pytest
import torch

import quadmul_amd as qm
from util import pack_cpu

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def problem(m, n, k, group, dtype, scales, bias, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k + pad, generator=g)
    x[:, ::97] *= 8.0
    x = x.to(dtype)[:, :k]
    q = torch.randint(-8, 8, (n, k), dtype=torch.int8, generator=g)
    s = ((torch.rand(n, -(-k // group), generator=g) + 0.1) * 0.05).to(scales)
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    return x, q, s, b


def check(x, q, s, group, b, y):
    """The sum of K products in float32, in any order: rounding errors of at most half a unit each, 6 standard deviations of their sum against the
    sum of the terms' sizes; one rounding to the result's type; half of float16's smallest step."""
    k = q.shape[1]
    w = q.double() * s.double().repeat_interleave(group, dim=1)[:, :k]
    want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    if b is not None:
        want, size = want + b.double(), size + b.double().abs()
    bound = UNIT[x.dtype] * want.abs() + 6.0 * math.sqrt(max(k, 1)) * 2.0 ** -24 * size + 2.0 ** -24
    off = (y.double().cpu() - want).abs()
    assert y.dtype == x.dtype and y.shape == want.shape
    assert bool((off <= bound).all()), float((off - bound).max())


SIZES = [  # m, n, k, group
    (1, 64, 32, 32), (1, 1, 128, 128), (1, 257, 4096, 128), (1, 1000, 4128, 32), (2, 96, 2048, 64), (3, 130, 1024, 256), (5, 77, 544, 32), (8, 512, 2048, 128),
    (9, 100, 1056, 96), (16, 640, 4096, 128), (17, 333, 992, 32), (31, 64, 256, 512), (33, 129, 2080, 64), (64, 1024, 1024, 128), (65, 70, 160, 64),
    (127, 257, 640, 128), (128, 128, 128, 128), (200, 300, 1504, 32), (257, 511, 768, 96), (513, 384, 2048, 128),
    (1, 300, 14336, 128), (13, 260, 28672, 128), (1, 4, 57344, 64), (40, 48, 28672, 64),
    (1, 50, 2, 32), (3, 65, 66, 32), (4, 100, 1002, 64), (70, 33, 130, 128), (1, 64, 0, 32), (5, 9, 34, 32),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("wide", [False, True], ids=["scales16", "scales32"])
@pytest.mark.parametrize("m,n,k,group", SIZES)
def test_against_64_bits(m, n, k, group, wide, dtype):
    x, q, s, b = problem(m, n, k, group, dtype, torch.float32 if wide else dtype, (m + n) % 2 == 0, m * 1000 + n + k)
    y = qm.gemm_grouped(x.cuda(), pack_cpu(q).cuda(), s.cuda(), group, None if b is None else b.cuda())
    check(x, q, s, group, b, y)


@pytest.mark.parametrize("m,n,k,group", [(1, 64, 256, 32), (7, 40, 512, 128), (40, 65, 320, 64), (150, 130, 256, 128)])
@pytest.mark.parametrize("pad", [1, 2, 8, 64])
def test_rows_at_a_distance(m, n, k, group, pad):
    x, q, s, b = problem(m, n, k, group, torch.float16, torch.float16, True, 5, pad)
    wide = torch.full((m, k + pad), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, :k] = x.cuda()
    check(x, q, s, group, b, qm.gemm_grouped(wide[:, :k], pack_cpu(q).cuda(), s.cuda(), group, b.cuda()))
    turned = x.cuda().t().contiguous().t()  # rows that are not contiguous
    check(x, q, s, group, b, qm.gemm_grouped(turned, pack_cpu(q).cuda(), s.cuda(), group, b.cuda()))


@pytest.mark.parametrize("m,n,k,group", [(1, 70, 512, 64), (6, 33, 1024, 128), (80, 48, 256, 32), (300, 140, 512, 128)])
@pytest.mark.parametrize("x_off,w_off", [(1, 0), (0, 1), (0, 4), (3, 2), (8, 16)])
def test_any_address(m, n, k, group, x_off, w_off):
    x, q, s, b = problem(m, n, k, group, torch.bfloat16, torch.bfloat16, False, 6)
    xs = torch.zeros(m * k + 16, dtype=torch.bfloat16, device="cuda")[x_off:x_off + m * k].view(m, k)
    ws = torch.zeros(n * (k // 2) + 32, dtype=torch.int8, device="cuda")[w_off:w_off + n * (k // 2)].view(n, k // 2)
    xs.copy_(x), ws.copy_(pack_cpu(q))
    check(x, q, s, group, b, qm.gemm_grouped(xs, ws, s.cuda(), group))


@pytest.mark.parametrize("m", [1, 4, 20, 100, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_large_and_tiny_values(m, dtype):
    """Activations over the type's range, scales that undo it: nothing overflows on the way."""
    x, q, s, _ = problem(m, 96, 512, 128, dtype, torch.float32, False, 7)
    x = (x.float() * torch.logspace(-4, 3, 512)).to(dtype)
    s[:, 0] *= 1e3
    check(x, q, s, 128, None, qm.gemm_grouped(x.cuda(), pack_cpu(q).cuda(), s.cuda(), 128))
    one = torch.zeros(m, 512, dtype=dtype)
    one[:, 77] = torch.finfo(dtype).smallest_normal / 4   # below the normal numbers
    s32 = torch.full((96, 4), 2.0 ** 14)
    check(one, q, s32, 128, None, qm.gemm_grouped(one.cuda(), pack_cpu(q).cuda(), s32.cuda(), 128))


@pytest.mark.parametrize("m", [1, 3, 20, 100, 300])
def test_infinities_and_nans_stay_in_their_rows(m):
    x, q, s, _ = problem(m, 80, 512, 64, torch.float16, torch.float16, False, 8)
    q[0] = 0
    x[m // 2, 100] = float("inf")
    y = qm.gemm_grouped(x.cuda(), pack_cpu(q).cuda(), s.cuda(), 64).cpu()
    assert not y[m // 2].isfinite().any() or bool((~y[m // 2].isfinite() | (q[:, 100] == 0)).all())
    keep = torch.arange(m) != m // 2
    if keep.any():
        check(x[keep], q, s, 64, None, y[keep])


def test_same_values_whatever_the_stream_and_in_a_graph():
    x, q, s, _ = problem(3, 512, 2048, 128, torch.float16, torch.float16, False, 9)
    x, w, s = x.cuda(), pack_cpu(q).cuda(), s.cuda()
    first = qm.gemm_grouped(x, w, s, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = qm.gemm_grouped(x, w, s, 128)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = qm.gemm_grouped(x, w, s, 128)
    for seed in range(4):
        x.copy_(torch.randn(3, 2048, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, qm.gemm_grouped(x, w, s, 128))


def test_quantize_groups_is_the_rule_of_rows_by_groups():
    w = torch.randn(40, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    packed, scales = qm.quantize_groups(w, 64)
    assert packed.shape == (40, 256) and scales.shape == (40, 8) and scales.dtype == torch.float32
    rows, row_scales = qm.quantize_pack(w.reshape(-1, 64))
    assert torch.equal(packed.reshape(-1), rows.reshape(-1)) and torch.equal(scales.reshape(-1), row_scales)
    x = torch.randn(5, 512, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    y = qm.gemm_grouped(x, packed, scales, 64)
    rough = x.float() @ w.float().T
    assert float((y.float() - rough).norm() / rough.norm()) < 0.2   # what 4 bits leave


def test_refusals():
    x = torch.zeros(4, 128, dtype=torch.float16, device="cuda")
    w = torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(8, 2, dtype=torch.float16, device="cuda")
    b = torch.zeros(8, dtype=torch.float16, device="cuda")
    assert qm.gemm_grouped(x, w, s, 64, b).shape == (4, 8)
    bad = [
        (x.float(), w, s, 64, None), (x, w.float(), s, 64, None), (x, w, s.to(torch.bfloat16), 64, None), (x, w, s, 128, None), (x, w, s, 48, None),
        (x, w, s, 0, None), (x, w, s, -64, None), (x, w[:, :32], s, 64, None), (x[0], w, s, 64, None), (x, w, s.t(), 64, None), (x, w, s, 64, b[:7]),
        (x, w, s, 64, b.float()), (x.cpu(), w.cpu(), s.cpu(), 64, None), (x, w.cpu(), s, 64, None), (x, w, s.cpu(), 64, None), (x[:, :126], w, s, 64, None),
    ]
    for args in bad:
        with pytest.raises(qm.QuadmulError):
            qm.gemm_grouped(*args)
    with pytest.raises(qm.QuadmulError):
        qm.quantize_groups(torch.zeros(4, 100, device="cuda"), 64)
    assert qm.gemm_grouped(x[:0], w, s, 64).shape == (0, 8)
    assert qm.gemm_grouped(x, w[:0], s[:0], 64).shape == (4, 0)


def test_without_the_extension_the_same(monkeypatch):
    import types

    x, q, s, b = problem(3, 70, 512, 64, torch.bfloat16, torch.bfloat16, True, 12)
    args = (x.cuda(), pack_cpu(q).cuda(), s.cuda(), 64, b.cuda())
    first = qm.gemm_grouped(*args)
    monkeypatch.setattr(qm, "_ext", types.SimpleNamespace(**dict.fromkeys(qm._EXT_FUNCTIONS, lambda *a: None)))
    assert torch.equal(first, qm.gemm_grouped(*args))


@pytest.mark.parametrize("m,n,k,x_off,w_off", [(13, 40, 16384, 1, 0), (13, 40, 16384, 0, 16), (16, 40, 16384, 3, 3), (20, 40, 16384, 1, 0), (100, 40, 16384, 5, 16), (100, 40, 16384, 1, 1)])
def test_any_address_with_k_in_runs(m, n, k, x_off, w_off):
    """K summed in several runs, with x and the weights at any address: whether there is a workspace goes by the weights' alignment alone."""
    test_any_address(m, n, k, 128, x_off, w_off)
    assert (qm.library().qm_gemm_grouped_workspace_bytes(m, n, k, 128, 16) > 0) and qm.library().qm_gemm_grouped_workspace_bytes(m, n, k, 128, 1) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("m,n,k,group,wide", [(1024, 8300, 160, 64, True), (1030, 8191, 288, 32, False), (1100, 8192, 416, 128, True), (1024, 8200, 224, 96, False), (500, 16500, 96, 128, False),
                                              (1024, 8192, 32, 256, True)])
def test_tiles_of_256_rows(m, n, k, group, wide, dtype):
    """Enough tiles for the largest ones: edges in rows and columns, a K that ends inside a step, every kind of group."""
    x, q, s, b = problem(m, n, k, group, dtype, torch.float32 if wide else dtype, m == 1024, m + n + k)
    y = qm.gemm_grouped(x.cuda(), pack_cpu(q).cuda(), s.cuda(), group, None if b is None else b.cuda())
    check(x, q, s, group, b, y)


@pytest.mark.usefixtures("gives_memory_back")
@pytest.mark.parametrize("m", [1, 6])
def test_more_columns_than_a_grid_has_threads(m):
    """2^26 columns and a few: a wave to each would be 2^32 threads and more. Every result is an integer of few bits."""
    n = 2 ** 26 + 5
    g = torch.Generator(device="cuda").manual_seed(13)
    w = torch.randint(-128, 128, (n, 1), dtype=torch.int8, device="cuda", generator=g)
    x = torch.tensor([[i + 1.0, -3.0] for i in range(m)], dtype=torch.float16, device="cuda")
    y = qm.gemm_grouped(x, w, torch.ones(n, 1, dtype=torch.float16, device="cuda"), 32)
    low, high = ((w[:, 0] << 4) >> 4).half(), (w[:, 0] >> 4).half()
    for i in range(m):
        assert torch.equal(y[i], low * (i + 1.0) - high * 3.0)


@pytest.mark.parametrize("m", [1, 3, 16, 20, 60, 64, 65, 300])
def test_bf16_activations_near_the_end_of_their_range(m):
    """Up to 64 rows the weights take part as 136 more than they are and 136 times the sum of x is taken off: 2^118 is held, above 2^119 or with an infinity the
    row is lost and no other. Above 64 rows they are integers, and a row is lost where its exact result is. The error of a term is half a unit of it in float32, with the 136
    and what is taken off counted to its size up to 64 rows."""
    x, q, s, _ = problem(m, 80, 512, 64, torch.bfloat16, torch.bfloat16, False, 14)
    w = q.double() * s.double().repeat_interleave(64, dim=1)
    extra = 272.0 * s.double().repeat_interleave(64, dim=1) if m <= 64 else torch.zeros_like(w)
    row, keep = m // 2, torch.arange(m) != m // 2
    for big in (2.0 ** 118, -2.0 ** 118, 2.0 ** 121, float("inf"), float("-inf"), float("nan")):
        x[row, 100] = big
        y = qm.gemm_grouped(x.cuda(), pack_cpu(q).cuda(), s.cuda(), 64).cpu()
        held = abs(big) <= (2.0 ** 118 if m <= 64 else 2.0 ** 121)
        if held:
            want, size = x.double() @ w.T, x.double().abs() @ (w.abs() + extra).T
            bound = UNIT[torch.bfloat16] * want.abs() + 6.0 * math.sqrt(512) * 2.0 ** -24 * size
            assert bool(((y.double() - want).abs() <= bound)[row].all())
        else:
            assert not y[row].isfinite().any()
        if keep.any():
            check(x[keep], q, s, 64, None, y[keep])


@pytest.mark.parametrize("m", [1, 7, 16, 33, 64, 100, 300])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
def test_scales_and_bias_at_any_address(m, group):
    x, q, s, b = problem(m, 70, 672, group, torch.bfloat16, torch.bfloat16, True, 15)
    at = torch.zeros(s.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(s.shape)
    bias = torch.zeros(71, dtype=torch.bfloat16, device="cuda")[1:]
    at.copy_(s), bias.copy_(b)
    check(x, q, s, group, b, qm.gemm_grouped(x.cuda(), pack_cpu(q).cuda(), at, group, bias))

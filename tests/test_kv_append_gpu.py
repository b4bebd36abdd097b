"""Storing into the paged 8-bit cache (csrc/qm_kv.hpp): codes, scales and rotated queries bit for bit as the definition's 32-bit operations give
them, the values within the definition's roundings of what 64 bits give."""
import pytest
import torch

import quadmul_amd as qm
from quadmul_amd import kv_cache
from kv_util import append_plain, make_cache, make_table, starts

pytestmark = pytest.mark.gpu


def tables(positions, pairs):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    return angle.cos().float(), angle.sin().float()


def case(lengths, counts, heads, kv_heads, dim, page, dtype, seed, pairs=None, positions=None):
    g = torch.Generator().manual_seed(seed)
    tokens, held = sum(counts), sum(-(-max(n, 0) // page) for n in lengths)
    cache = make_cache(held + 3, kv_heads, dim, page, seed, scale=0.01)
    table = make_table(lengths, page, held + 3, seed + 1)
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g)
    qkv[:, ::113] *= 7.0
    qkv = qkv.to(dtype)
    pairs = dim // 2 if pairs is None else pairs
    cos, sin = tables(positions or max(max(lengths), 1), pairs) if pairs else (None, None)
    return cache, table, qkv, cos, sin


def split(qkv, heads, kv_heads, dim):
    q, k, v = qkv.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1)
    return q.unflatten(1, (heads, dim)), k.unflatten(1, (kv_heads, dim)), v.unflatten(1, (kv_heads, dim))


def gpu(t):
    return None if t is None else t.cuda()


def run(cache, table, qkv, cos, sin, lengths, counts, heads, kv_heads, dim, interleaved=False, packed=True, **options):
    on = [t.clone().cuda() for t in cache]
    q, k, v = split(qkv.cuda(), heads, kv_heads, dim)
    out = kv_cache.append(k, v, *on, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), starts(counts).cuda() if packed else None,
                          q=q, cos=gpu(cos), sin=gpu(sin), interleaved=interleaved, **options)
    return [t.cpu() for t in on] + [out.cpu()]


CASES = [  # lengths, new tokens of each, heads, kv heads, dim, page
    ([1], [1], 4, 1, 64, 16), ([17], [1], 8, 2, 128, 16), ([16], [16], 2, 2, 128, 16), ([5, 40, 128], [5, 3, 128], 4, 2, 64, 32),
    ([100, 1, 33, 64], [37, 1, 33, 1], 6, 2, 96, 16), ([300], [299], 3, 1, 256, 128), ([130, 129, 128, 127], [2, 2, 2, 2], 12, 12, 64, 64),
    ([0, 50, 0, 7], [0, 50, 0, 7], 4, 4, 192, 32), ([3, 20], [8, 20], 2, 1, 128, 16), ([-5, 31], [2, 1], 2, 2, 128, 16), ([77] * 20, [1] * 20, 28, 4, 128, 16),
    ([1000, 513], [700, 513], 2, 1, 128, 64), ([90], [70], 2, 2, 128, 128),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("lengths,counts,heads,kv_heads,dim,page", CASES)
def test_bit_for_bit(lengths, counts, heads, kv_heads, dim, page, interleaved, dtype):
    cache, table, qkv, cos, sin = case(lengths, counts, heads, kv_heads, dim, page, dtype, 3)
    k, v, scales, q = run(cache, table, qkv, cos, sin, lengths, counts, heads, kv_heads, dim, interleaved)
    qs, ks, vs = split(qkv, heads, kv_heads, dim)
    wk, wv, ws, wq = append_plain(ks, vs, *cache, table, lengths, counts, cos, sin, interleaved, qs)
    assert torch.equal(scales, ws)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    assert torch.equal(q, wq.to(dtype))


@pytest.mark.parametrize("lengths,counts,heads,kv_heads,dim,page", CASES)
def test_against_64_bits(lengths, counts, heads, kv_heads, dim, page):
    """What is stored now is within half a step of its value, and the codes that were there within half a step more than before; half a
    hundredth of a step for the 32-bit operations."""
    cache, table, qkv, cos, sin = case(lengths, counts, heads, kv_heads, dim, page, torch.float16, 4)
    k, v, scales, q = run(cache, table, qkv, cos, sin, lengths, counts, heads, kv_heads, dim)
    qs, ks, vs = split(qkv, heads, kv_heads, dim)
    wk, wv, ws, wq = append_plain(ks, vs, *cache, table, lengths, counts, cos, sin, False, qs, wide=True)
    assert float(((scales.double() - ws) / ws.clamp(min=1e-30)).abs().max()) < 2.0 ** -21
    for got, want in ((k, wk), (v, wv)):
        assert float((got.double() - want).abs().max()) <= 1.0             # a tie may fall to either side,
        assert float((got.double() != want).double().mean()) < 1e-3        # and few do
    assert float((q.double() - wq).abs().max()) <= float(wq.abs().max()) * 2.0 ** -11 * 1.01


@pytest.mark.parametrize("pairs", [0, 1, 16, 20, 32])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
def test_part_of_a_head_rotated(pairs, interleaved):
    lengths, counts = [70, 9], [40, 9]
    cache, table, qkv, cos, sin = case(lengths, counts, 4, 2, 64, 32, torch.bfloat16, 5, pairs=pairs)
    k, v, scales, q = run(cache, table, qkv, cos, sin, lengths, counts, 4, 2, 64, interleaved)
    qs, ks, vs = split(qkv, 4, 2, 64)
    wk, wv, ws, wq = append_plain(ks, vs, *cache, table, lengths, counts, cos, sin, interleaved, qs)
    assert torch.equal(scales, ws) and torch.equal(k, wk) and torch.equal(v, wv) and torch.equal(q, wq.to(torch.bfloat16))


@pytest.mark.parametrize("packed,max_query", [(True, 0), (True, 1), (True, 1000), (False, 0)])
def test_the_hint_and_equal_counts_change_nothing(packed, max_query):
    lengths, counts = [130, 90, 33, 48], [33, 33, 33, 33]
    cache, table, qkv, cos, sin = case(lengths, counts, 4, 2, 128, 16, torch.float16, 6)
    got = run(cache, table, qkv, cos, sin, lengths, counts, 4, 2, 128, packed=packed, max_query=max_query)
    qs, ks, vs = split(qkv, 4, 2, 128)
    want = append_plain(ks, vs, *cache, table, lengths, counts, cos, sin, False, qs)
    assert all(torch.equal(a, b.to(a.dtype)) for a, b in zip(got, want))


def test_token_by_token_and_again():
    """Sixty tokens one at a time: the scales only grow inside a page, and what comes back is near what went in."""
    g = torch.Generator().manual_seed(7)
    cache = kv_cache.PagedKVCache(8, 2, 64, 16)
    table = torch.arange(8, dtype=torch.int32).flip(0)[None].cuda()
    k, v = (torch.randn(60, 2, 64, generator=g).to(torch.float16).cuda() for _ in range(2))
    for t in range(60):
        cache.append(k[t:t + 1], v[t:t + 1], table, torch.tensor([t + 1], dtype=torch.int32, device="cuda"))
        if t % 7 == 3:  # the last token once more: nothing may move
            before = [x.clone() for x in (cache.k, cache.v, cache.scales)]
            cache.append(k[t:t + 1], v[t:t + 1], table, torch.tensor([t + 1], dtype=torch.int32, device="cuda"))
            assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.scales)))
    got = [x.transpose(1, 2).reshape(64 + 64, 2, 64)[:60] for x in cache.read(table[0])]
    for side, (a, b) in enumerate(zip(got, (k, v))):
        step = cache.scales[table[0].long()][:4, :, side].repeat_interleave(16, dim=0)[:60, :, None]
        # half a step when stored, and up to half a step (a smaller one) each time that the scale grew: at most 15 times, far fewer on random data
        assert float(((a.float() - b.float()).abs() / step).max()) < 3.0
    assert bool((cache.scales[:4] == 0).all())  # pages that no token fell into


def test_pages_that_are_not_there():
    """Entries that are no page, and tokens past the table: dropped, and nothing else is touched."""
    lengths, counts = [100, 40], [100, 8]
    cache, table, qkv, cos, sin = case(lengths, counts, 2, 2, 64, 16, torch.float16, 8)
    table = table[:, :5].clone()   # room for 80 of the 100 tokens
    table[0, 1], table[0, 3], table[1, 2] = -1, cache[0].shape[0], -2 ** 31
    k, v, scales, q = run(cache, table, qkv, cos, sin, lengths, counts, 2, 2, 64)
    qs, ks, vs = split(qkv, 2, 2, 64)
    want = append_plain(ks, vs, *cache, table, lengths, counts, cos, sin, False, qs)
    assert all(torch.equal(a, b.to(a.dtype)) for a, b in zip((k, v, scales, q), want))


def test_lengths_and_starts_that_make_no_sense_stay_inside():
    cache, table, qkv, cos, sin = case([60, 60], [20, 20], 2, 2, 64, 16, torch.float16, 9)
    on = [t.clone().cuda() for t in cache]
    q, k, v = split(qkv.cuda(), 2, 2, 64)
    for lengths, start in (([2 ** 31 - 1, -2 ** 31], [0, 20, 40]), ([60, 60], [-7, 2 ** 31 - 1, 5]), ([60, 60], [40, 0, 40])):
        out = kv_cache.append(k, v, *on, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), torch.tensor(start, dtype=torch.int32, device="cuda"),
                              q=q, cos=cos.cuda(), sin=sin.cuda())
        torch.cuda.synchronize()
        assert out.shape == q.shape


def test_positions_past_the_tables_give_nan():
    lengths, counts = [40], [4]
    cache, table, qkv, cos, sin = case(lengths, counts, 2, 1, 64, 16, torch.float16, 10, positions=38)
    k, v, scales, q = run(cache, table, qkv, cos, sin, lengths, counts, 2, 1, 64)
    assert q[:2].isfinite().all() and q[2:].isnan().all()
    page = int(table[0, 2])
    assert scales[page, 0, 0].isnan() and scales[page, 0, 1].isfinite()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite_show(bad):
    lengths, counts = [20, 20], [3, 3]
    cache, table, qkv, cos, sin = case(lengths, counts, 2, 2, 64, 16, torch.bfloat16, 11, pairs=0)
    qkv[1, 2 * 64 + 5] = bad       # a key of the first sequence, head 0
    k, v, scales, q = run(cache, table, qkv, cos, sin, lengths, counts, 2, 2, 64)
    page = int(table[0, 1])
    assert not scales[page, 0, 0].isfinite()
    scales[page, 0, 0] = 1.0
    assert scales.isfinite().all()


def test_zeros_and_tiny_values():
    lengths, counts = [16, 16, 16], [16, 16, 16]
    cache, table, qkv, cos, sin = case(lengths, counts, 1, 1, 64, 16, torch.bfloat16, 12, pairs=0)
    qkv[:16] = 0
    qkv[16:32] = 1e-38
    k, v, scales, q = run(cache, table, qkv, cos, sin, lengths, counts, 1, 1, 64)
    for s in range(2):
        page = int(table[s, 0])
        assert bool((scales[page] == 0).all()) and not k[page].any() and not v[page].any()
    back = kv_cache.read(k.cuda(), v.cuda(), scales.cuda(), table[:2, 0].contiguous().cuda(), torch.bfloat16)
    assert not back[0].any() and not back[1].any()


@pytest.mark.parametrize("page,dim", [(16, 64), (32, 96), (64, 128), (128, 256), (16, 192)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_read(page, dim, dtype):
    cache = make_cache(9, 3, dim, page, 13)
    ids = torch.tensor([4, 0, 8, -1, 4, 9, 2], dtype=torch.int32)
    k, v = kv_cache.read(*[t.cuda() for t in cache], ids.cuda(), dtype)
    safe = ids.clamp(0, 8).long()
    there = (ids >= 0) & (ids < 9)
    wk = (cache[0][safe].float() * cache[2][safe][..., 0, None, None]).to(dtype)
    wv = (cache[1][safe].transpose(2, 3).float() * cache[2][safe][..., 1, None, None]).to(dtype)
    for got, want in ((k.cpu(), wk), (v.cpu(), wv)):
        assert torch.equal(got[there], want[there]) and got[~there].isnan().all()


def test_in_a_graph_and_on_another_stream():
    lengths, counts = [50, 17, 33], [1, 1, 1]
    cache, table, qkv, cos, sin = case(lengths, counts, 4, 2, 128, 16, torch.float16, 14)
    on = [t.clone().cuda() for t in cache]
    x, table, cos, sin = qkv.cuda(), table.cuda(), cos.cuda(), sin.cuda()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q, k, v = split(x, 4, 2, 128)
    kv_cache.append(k, v, *on, table, n, q=q, cos=cos, sin=sin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_cache.append(k, v, *on, table, n, q=q, cos=cos, sin=sin)
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        mine = [t.clone() for t in on]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = kv_cache.append(k, v, *mine, table, n, q=q, cos=cos, sin=sin)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and all(torch.equal(a, b) for a, b in zip(on, mine))


def test_refusals():
    cache = [t.cuda() for t in make_cache(4, 2, 64, 16, 15)]
    table, n = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    q, cos = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda"), torch.ones(10, 32, device="cuda")
    table[1] = 1
    assert kv_cache.append(k, k, *cache, table, n) is None
    assert kv_cache.append(k, k, *cache, table, n, q=q, cos=cos, sin=cos).shape == q.shape
    bad = [
        ((k.float(), k.float(), *cache, table, n), {}), ((k, k.to(torch.bfloat16), *cache, table, n), {}), ((k[:, :1], k[:, :1], *cache, table, n), {}),
        ((k[..., :32], k[..., :32], *cache, table, n), {}), ((k, k, cache[0], cache[0], cache[2], table, n), {}), ((k, k, cache[0].cpu(), cache[1], cache[2], table, n), {}),
        ((k, k, *cache, table.long(), n), {}), ((k, k, *cache, table, n.long()), {}), ((k, k, *cache, table[:1], n), {}), ((k, k, *cache, table.cpu(), n), {}),
        ((k, k, *cache, table, n, n), {}), ((torch.cat((k, k[:1])),) * 2 + (*cache, table, n), {}), ((k, k, *cache, table, n), {"q": q[:1]}), ((k, k, *cache, table, n), {"cos": cos}),
        ((k, k, *cache, table, n), {"cos": cos, "sin": cos[:5]}), ((k, k, *cache, table, n), {"cos": cos.half(), "sin": cos.half()}), ((k, k, cache[0], cache[1], cache[2][..., :1], table, n), {}),
        ((k, k, *cache, table, n), {"cos": torch.ones(10, 33, device="cuda"), "sin": torch.ones(10, 33, device="cuda")}), ((k, k, *cache, table, n), {"q": q.to(torch.bfloat16)}),
        ((k.transpose(0, 2).contiguous().transpose(0, 2),) * 2 + (*cache, table, n), {}),
    ]
    for args, options in bad:
        with pytest.raises(qm.QuadmulError):
            kv_cache.append(*args, **options)
    for pages in (table, torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(qm.QuadmulError):
            kv_cache.read(*cache, pages)
    with pytest.raises(qm.QuadmulError):
        kv_cache.read(*cache, n, torch.float32)
    for sizes in ((4, 2, 64, 17), (4, 2, 80, 16), (4, 0, 64, 16)):
        with pytest.raises(qm.QuadmulError):
            kv_cache.PagedKVCache(*sizes)
    assert kv_cache.append(k[:0], k[:0], *cache, table, n) is None
    assert kv_cache.read(*cache, n[:0])[0].shape == (0, 2, 16, 64)


def test_without_the_extension_the_same(monkeypatch):
    import types

    lengths, counts = [50, 17, 33], [3, 1, 20]
    inputs = case(lengths, counts, 4, 2, 128, 16, torch.float16, 16)
    first = run(*inputs, lengths, counts, 4, 2, 128)
    monkeypatch.setattr(qm, "_ext", types.SimpleNamespace(**dict.fromkeys(qm._EXT_FUNCTIONS, lambda *a: None)))
    assert all(torch.equal(a, b) for a, b in zip(first, run(*inputs, lengths, counts, 4, 2, 128)))
    ids = inputs[1][:, 0].contiguous().cuda()
    assert kv_cache.read(*[t.cuda() for t in inputs[0]], ids)[0].shape == (3, 2, 16, 128)


@pytest.mark.parametrize("new", [1, 20], ids=["few", "many"])
@pytest.mark.parametrize("side", ["key", "value"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_attention_to_a_page_that_is_not_finite_is_nan(bad, side, new):
    """Whatever the signs of the queries, and although the other tokens of the page have codes of 0; pages beside it are not touched by it, and a page
    that begins anew is as if nothing had been."""
    lengths, counts = [17, 33], [new if new < 17 else 17, new]
    cache, table, qkv, _, _ = case(lengths, counts, 4, 2, 64, 16, torch.float16, 17, pairs=0)
    on = [t.cuda() for t in cache]
    q, k, v = split(qkv.cuda(), 4, 2, 64)
    table, n, start = table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), starts(counts).cuda()
    (k if side == "key" else v)[counts[0] - 1, 0] = 0
    (k if side == "key" else v)[counts[0] - 1, 0, 5] = bad     # the only token of its page, head 0
    kv_cache.append(k, v, *on, table, n, start)
    ask = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    ask[:, 0::2, 5], ask[:, 1::2, 5] = 2.0, -2.0
    out = kv_cache.attend(ask, *on, table, n)
    assert out[0, :2].isnan().all() and out[0, 2:].isfinite().all() and out[1].isfinite().all()
    assert kv_cache.attend(ask, *on, table, n - 1)[0].isfinite().all()
    k[counts[0] - 1], v[counts[0] - 1] = 1.0, -1.0
    kv_cache.append(k, v, *on, table, n, start)
    assert kv_cache.attend(ask, *on, table, n).isfinite().all()


@pytest.mark.parametrize("counts", [[40, 0, 0, 0] + [0] * 40, [0, 20, 0, 23] + [0] * 40, [1] * 44])
def test_no_more_tokens_than_sequences(counts):
    """Without a hint these are taken for one each, which they need not be."""
    lengths = [50, 20, 3, 70] + [i + 1 for i in range(40)]
    cache, table, qkv, cos, sin = case(lengths, counts, 4, 2, 64, 16, torch.float16, 18)
    got = run(cache, table, qkv, cos, sin, lengths, counts, 4, 2, 64)
    qs, ks, vs = split(qkv, 4, 2, 64)
    want = append_plain(ks, vs, *cache, table, lengths, counts, cos, sin, False, qs)
    assert all(torch.equal(a, b.to(a.dtype)) for a, b in zip(got, want))

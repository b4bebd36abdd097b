"""Attention over the paged 8-bit cache (csrc/qm_attend.hpp) against 64 bits: every head layout and page size, one token and many, lengths from
none to several splits, windows, missing pages, rows that see nothing."""
import pytest
import torch

import quadmul_amd as qm
from quadmul_amd import kv_cache
from kv_util import attend_plain, check_attention, make_cache, make_table, starts

pytestmark = pytest.mark.gpu


def problem(lengths, counts, heads, kv_heads, dim, page, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    held = sum(-(-max(n, 0) // page) for n in lengths)
    cache = make_cache(held + 2, kv_heads, dim, page, seed)
    table = make_table(lengths, page, held + 2, seed + 1)
    q = (torch.randn(sum(counts), heads, dim, generator=g) * size).to(dtype)
    return q, cache, table


def attend(q, cache, table, lengths, counts, packed=True, **options):
    return kv_cache.attend(q.cuda(), *[t.cuda() for t in cache], table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                           starts(counts).cuda() if packed else None, **options)


def both(q, cache, table, lengths, counts, scale=None, causal=True, window=0, **options):
    got = attend(q, cache, table, lengths, counts, scale=scale, causal=causal, window=window, **options)
    check_attention(got, attend_plain(q, *cache, table, lengths, counts, scale, causal, window), q.dtype)
    return got


LAYOUTS = [(4, 4, 64, 16), (8, 2, 128, 16), (12, 12, 64, 32), (7, 1, 128, 64), (16, 1, 256, 32), (6, 2, 96, 16), (3, 3, 192, 128), (20, 1, 64, 16), (40, 2, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", LAYOUTS)
def test_one_token_each(heads, kv_heads, dim, page, dtype):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 100, 128, 129, 200, 300, 511]
    q, cache, table = problem(lengths, [1] * len(lengths), heads, kv_heads, dim, page, dtype, 1)
    both(q, cache, table, lengths, [1] * len(lengths), packed=heads % 2 == 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", LAYOUTS)
def test_several_tokens_each(heads, kv_heads, dim, page, dtype):
    lengths, counts = [5, 40, 130, 33, 1, 90], [5, 7, 19, 1, 1, 64]
    q, cache, table = problem(lengths, counts, heads, kv_heads, dim, page, dtype, 2)
    both(q, cache, table, lengths, counts, max_query=64, max_length=130)


@pytest.mark.parametrize("length", [1, 700, 1023, 1024, 1025, 2049, 5000, 9000])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (2, 2, 64, 64), (1, 1, 256, 128)])
def test_one_long_sequence(length, heads, kv_heads, dim, page):
    q, cache, table = problem([length], [1], heads, kv_heads, dim, page, torch.float16, 3)
    first = both(q, cache, table, [length], [1], max_length=length)
    # a hint that is too short, none, one that is too long: the same within the bounds
    for hint in (1, 0, 100000):
        check_attention(attend(q, cache, table, [length], [1], max_length=hint), attend_plain(q, *cache, table, [length], [1]), q.dtype)
    assert torch.equal(first, attend(q, cache, table, [length], [1], max_length=length))  # no order of atomics in the result


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("window", [0, 1, 7, 64, 100])
@pytest.mark.parametrize("page", [16, 64])
def test_windows(window, causal, page):
    lengths, counts = [300, 65, 1, 20, 150], [40, 1, 1, 20, 3]
    q, cache, table = problem(lengths, counts, 4, 2, 64, page, torch.float16, 4)
    both(q, cache, table, lengths, counts, causal=causal, window=window, max_query=40, max_length=300)


@pytest.mark.parametrize("counts", [[300, 257], [129, 1], [1, 600], [128, 128]])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (3, 3, 64), (8, 2, 96)])
def test_prompts(counts, heads, kv_heads, dim):
    lengths = [counts[0] + 37, counts[1]]
    q, cache, table = problem(lengths, counts, heads, kv_heads, dim, 32, torch.bfloat16, 5)
    both(q, cache, table, lengths, counts, max_query=max(counts), max_length=max(lengths))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window,causal", [(32, 16, 64, 16, 0, True), (12, 12, 96, 64, 50, True), (8, 8, 128, 32, 0, False), (28, 14, 192, 16, 100, False),
                                                                  (16, 16, 256, 128, 0, True)])
def test_many_rows(heads, kv_heads, dim, page, window, causal, dtype):
    """Enough rows for tiles of 64 of them: several tiles to a sequence, the last one not full, histories of all lengths, none among them, padding."""
    lengths, counts = [150, 400, 130, 70, 3, 0], [150, 131, 65, 1, 40, 2]
    q, cache, table = problem(lengths, counts, heads, kv_heads, dim, page, dtype, 17)
    table[1, 1] = -1
    both(q, cache, table, lengths, counts, causal=causal, window=window, max_query=150, max_length=400)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim,page,window,causal", [(64, 16, 0, True), (96, 64, 50, True), (128, 32, 0, False), (192, 16, 100, True), (256, 128, 0, True)])
def test_many_rows_of_many_sequences(dim, page, window, causal, dtype):
    """Enough tiles of 64 rows for workgroups that take the steps one by one."""
    lengths, counts = [150, 400] + [3 * i for i in range(30)], [150, 131] + [7] * 30
    q, cache, table = problem(lengths, counts, 16, 16, dim, page, dtype, 19)
    table[1, 1] = -1
    both(q, cache, table, lengths, counts, causal=causal, window=window, max_query=sum(counts), max_length=400)   # 8 tiles, 16 heads, 32 sequences


def test_rows_that_see_nothing_are_zero():
    lengths, counts = [0, 30, 3, -4, 64], [1, 1, 6, 2, 1]   # no tokens at all; three rows in front of position 0; no tokens; only missing pages
    q, cache, table = problem(lengths, counts, 4, 2, 64, 16, torch.float16, 6)
    table[4] = -1
    got = both(q, cache, table, lengths, counts)
    assert not got[0].any() and not got[2:5].any() and not got[8:10].any() and not got[10].any() and got[5].any()


def test_missing_pages_and_tokens_past_the_table():
    lengths, counts = [200, 90, 130], [1, 5, 1]
    q, cache, table = problem(lengths, counts, 4, 2, 64, 16, torch.bfloat16, 7)
    table = table[:, :6].clone()    # 96 of the 200 tokens
    table[0, 0], table[0, 4], table[1, 5], table[2, 3] = -1, cache[0].shape[0], -2 ** 31, 2 ** 31 - 1
    both(q, cache, table, lengths, counts)
    # pages that a window has left behind, as a server frees them
    table[2, :4] = -1
    both(q, cache, table, lengths, counts, window=40)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_lies_in_unused_places_does_not_matter(bad):
    """Scales of pages that are not read, and of tokens that a mask hides, may be anything."""
    lengths, counts = [100, 40], [1, 10]
    q, cache, table = problem(lengths, counts, 4, 2, 64, 16, torch.float16, 8)
    table = torch.cat((table, torch.full((2, 2), 0, dtype=torch.int32)), dim=1)
    unused = next(i for i in range(cache[0].shape[0]) if i not in table[:, :-2].tolist()[0] + table[:, :-2].tolist()[1])
    table[:, -3:] = unused
    want = attend_plain(q, *cache, table, lengths, counts)
    cache[2][unused] = bad
    check_attention(attend(q, cache, table, lengths, counts, max_length=4096), want, q.dtype)
    # hidden by the window: the first pages of sequence 0
    want = attend_plain(q, *cache, table, lengths, counts, window=20)
    cache[2][int(table[0, 0])] = bad
    cache[2][int(table[0, 3])] = bad
    check_attention(attend(q, cache, table, lengths, counts, window=20), want, q.dtype)
    # seen: it shows, in this sequence alone
    got = attend(q, cache, table, lengths, counts)
    assert not got[0].isfinite().all() and got[1:].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("size", [0.0, 1e-6, 100.0, 3000.0])
def test_sharp_and_flat_weights(size, dtype):
    """Scores of thousands (one token takes all) down to none at all; sizes of q up to where float16 ends."""
    lengths, counts = [150, 64, 10], [1, 1, 10]
    q, cache, table = problem(lengths, counts, 4, 2, 128, 16, dtype, 9, size)
    q[0, 0, 3] = 65504.0 if dtype == torch.float16 else 3e38 if size == 3000.0 else 1.0
    scale = 1e-38 if size == 3000.0 and dtype == torch.bfloat16 else 0.01
    both(q, cache, table, lengths, counts, scale=scale)


@pytest.mark.parametrize("spread", [1e3, 1e6])
def test_pages_of_very_different_scales(spread):
    """Values of one page a thousand or a million times those of another, the larger ones first, last, and with hardly any weight."""
    lengths, counts = [200, 200, 200, 200], [1, 1, 1, 1]
    q, cache, table = problem(lengths, counts, 4, 2, 64, 16, torch.bfloat16, 10)
    for s, number in ((0, 0), (1, 12), (2, 5)):
        cache[2][int(table[s, number]), :, 1] *= spread
    cache[2][int(table[3, 2]), :, 1] *= spread
    cache[2][int(table[3, 2]), :, 0] = 0.0
    for p in table[3].tolist():
        if p >= 0:
            cache[1][p].clamp_(min=1)
    both(q, cache, table, lengths, counts)
    for p in table[2].tolist():
        cache[2][p, :, 1] *= 1e-30 / spread
    both(q, cache, table, lengths, counts)


def test_scales_of_zero():
    lengths, counts = [64, 40], [1, 3]
    q, cache, table = problem(lengths, counts, 4, 2, 64, 16, torch.float16, 11)
    cache[2][int(table[0, 1])] = 0.0
    for p in table[1].tolist():
        cache[2][p] = 0.0
    got = both(q, cache, table, lengths, counts)
    assert not got[1:].any()


@pytest.mark.parametrize("layout", ["view", "heads_first", "odd"])
def test_queries_of_any_strides(layout):
    lengths, counts = [70, 33], [5, 9]
    q, cache, table = problem(lengths, counts, 4, 2, 64, 16, torch.float16, 12)
    want = attend_plain(q, *cache, table, lengths, counts)
    if layout == "view":
        wide = torch.full((14, 8 * 64), float("nan"), dtype=torch.float16, device="cuda")
        given = wide[:, :4 * 64].view(14, 4, 64)
    elif layout == "heads_first":
        given = torch.empty(4, 14, 64, dtype=torch.float16, device="cuda").transpose(0, 1)
    else:
        given = torch.empty(14 * 4 * 67 + 1, dtype=torch.float16, device="cuda")[1:].view(14, 4, 67)[..., :64]
    given.copy_(q)
    check_attention(attend(given, cache, table, lengths, counts), want, torch.float16)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: the pages at its far end."""
    pages, heads, dim, page = 33000, 8, 256, 64   # 4.3e9 codes on each side
    if torch.cuda.mem_get_info()[0] < 12e9:
        pytest.skip("needs 9 GB")
    k = torch.zeros(pages, heads, page, dim, dtype=torch.int8, device="cuda")
    v = torch.zeros(pages, heads, dim, page, dtype=torch.int8, device="cuda")
    scales = torch.full((pages, heads, 2), 0.02, device="cuda")
    ids = torch.tensor([pages - 1, 16500, pages - 2, 0], dtype=torch.int32)
    small = make_cache(4, heads, dim, page, 13)
    for i, p in enumerate(ids.tolist()):
        k[p], v[p], scales[p] = small[0][i].cuda(), small[1][i].cuda(), small[2][i].cuda()
    g = torch.Generator().manual_seed(13)
    q = torch.randn(1, heads, dim, generator=g).to(torch.float16)
    n = torch.tensor([250], dtype=torch.int32, device="cuda")
    got = kv_cache.attend(q.cuda(), k, v, scales, ids[None].cuda(), n)
    check_attention(got, attend_plain(q, *small, torch.arange(4, dtype=torch.int32)[None], [250], [1]), torch.float16)
    new = torch.randn(2, 1, heads, dim, generator=g).to(torch.float16).cuda()
    kv_cache.append(new[0], new[1], k, v, scales, ids[None].flip(1).contiguous().cuda(), n)   # into the page at the far end
    for side, codes in enumerate((k[pages - 1, :, 249 % 64], v[pages - 1, :, :, 249 % 64])):
        step = scales[pages - 1, :, side, None]
        assert float((codes.float() - new[side][0].float() / step).abs().max()) <= 0.51
    back = kv_cache.read(k, v, scales, ids[:1].cuda())
    assert torch.equal(back[0][0], (k[pages - 1].float() * scales[pages - 1, :, 0, None, None]).half())
    assert torch.equal(back[1][0], (v[pages - 1].transpose(1, 2).float() * scales[pages - 1, :, 1, None, None]).half())


def test_in_a_graph_and_on_another_stream():
    lengths, counts = [600, 17, 2000], [1, 1, 1]
    q, cache, table = problem(lengths, counts, 8, 2, 128, 16, torch.float16, 14)
    q, cache, table, n = q.cuda(), [t.cuda() for t in cache], table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kv_cache.attend(q, *cache, table, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_cache.attend(q, *cache, table, n)
    for lengths in ([600, 17, 2000], [1, 16, 1999], [0, 3, 40]):
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        q.mul_(1.01)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = kv_cache.attend(q, *cache, table, n)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals():
    cache = [t.cuda() for t in make_cache(4, 2, 64, 16, 15)]
    table, n = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    assert kv_cache.attend(q, *cache, table, n).shape == q.shape
    bad = [
        ((q.float(), *cache, table, n), {}), ((q[:, :3], *cache, table, n), {}), ((q[..., :32], *cache, table, n), {}), ((q[0], *cache, table, n), {}),
        ((q.cpu(), *cache, table, n), {}), ((q, cache[0], cache[0], cache[2], table, n), {}), ((q, *cache, table.long(), n), {}), ((q, *cache, table, n.long()), {}),
        ((q, *cache, table[:1], n), {}), ((q, *cache, table, n, n), {}), ((torch.cat((q, q[:1])), *cache, table, n), {}), ((q, *cache, table, n), {"window": -1}),
        ((q, *cache, table.t(), n), {}), ((q, *cache, table, n[:0]), {}), ((q, cache[0].to(torch.uint8), cache[1], cache[2], table, n), {}),
    ]
    for args, options in bad:
        with pytest.raises(qm.QuadmulError):
            kv_cache.attend(*args, **options)
    assert kv_cache.attend(q[:0], *cache, table, n).shape == (0, 4, 64)


def test_without_the_extension_the_same(monkeypatch):
    import types

    lengths, counts = [600, 17, 200], [1, 5, 20]
    q, cache, table = problem(lengths, counts, 8, 2, 128, 16, torch.float16, 16)
    first = attend(q, cache, table, lengths, counts, window=100, max_query=20)
    monkeypatch.setattr(qm, "_ext", types.SimpleNamespace(**dict.fromkeys(qm._EXT_FUNCTIONS, lambda *a: None)))
    assert torch.equal(first, attend(q, cache, table, lengths, counts, window=100, max_query=20))


@pytest.mark.usefixtures("gives_memory_back")
def test_more_workgroups_than_a_grid_has():
    """2^15 sequences and 256 heads in a workgroup each would be 2^32 threads. Of one token each: its values come back."""
    sequences, heads = 2 ** 15, 256
    cache = [t.cuda() for t in make_cache(2, heads, 64, 16, 20)]
    table = torch.arange(sequences, dtype=torch.int32, device="cuda")[:, None] % 2
    q = torch.ones(sequences, heads, 64, dtype=torch.float16, device="cuda")
    out = kv_cache.attend(q, *cache, table, torch.ones(sequences, dtype=torch.int32, device="cuda"))
    for page in range(2):
        want = cache[1][page, :, :, 0].double() * cache[2][page, :, 1, None].double()
        off = (out[page::2].double() - want).abs()
        assert bool((off <= want.abs() * (2.0 ** -11 + 1.25 * 2.0 ** -11) + 2.0 ** -24).all())


@pytest.mark.parametrize("most", [34, 64, 128, 130, 512, 528])
def test_prompts_beside_single_tokens(most):
    """Tiles of 64 rows, from 2 to 33 of them (even and odd, many and few powers of two), in sequences that have all of them, some and one; a hint that is
    too small."""
    lengths = [most + 9, most // 2 + 3, 1, 70, 33, 5, most, 2]
    counts = [most, most // 2, 1, 1, 33, 1, 1, 0]
    q, cache, table = problem(lengths, counts, 16, 4, 64, 16, torch.bfloat16, 21)
    want = attend_plain(q, *cache, table, lengths, counts)
    for hint in (most, 40):
        check_attention(attend(q, cache, table, lengths, counts, max_query=hint, max_length=max(lengths)), want, torch.bfloat16)


@pytest.mark.parametrize("sequences", [257, 700])
def test_one_long_sequence_among_many(sequences):
    lengths = [(7 * i) % 40 for i in range(sequences)]
    lengths[sequences // 2], lengths[-1] = 5000, 1500
    counts = [i % 3 if i % 50 == 0 else 1 for i in range(sequences)]
    q, cache, table = problem(lengths, counts, 4, 2, 64, 16, torch.float16, 22)
    got = both(q, cache, table, lengths, counts, max_query=2, max_length=5000)
    assert torch.equal(got, attend(q, cache, table, lengths, counts, max_query=2, max_length=5000))


@pytest.mark.parametrize("lengths,counts", [([40, 900, 3, 2500, 1, 70], [6, 0, 0, 0, 0, 0]), ([40, 900, 3, 2500, 1, 70], [0, 2, 0, 3, 0, 1]), ([5, 1200, 33, 17, 1100, 2], [1, 1, 1, 1, 1, 1])])
def test_no_more_tokens_than_sequences(lengths, counts):
    """Without a hint these are taken for one each, which they need not be."""
    q, cache, table = problem(lengths, counts, 16, 2, 64, 16, torch.float16, 23)
    both(q, cache, table, lengths, counts)


@pytest.mark.parametrize("at", [5, 290])
@pytest.mark.parametrize("sequences,count", [(1, 1), (3, 4), (16, 40)], ids=["one", "few", "many"])
def test_weights_far_below_the_largest(sequences, count, at):
    """Weights 2^-20 to 2^-30 of one token's, in channels where that token's value is 0, so that they are all there is. Beside the bound of the other tests, each
    of them may be off by 2^-31 of the largest."""
    length, heads, kv_heads, dim, page = 700, 16, 4, 64, 16
    lengths, counts = [length] * sequences, [count] * sequences
    q, (k, v, scales), table = problem(lengths, counts, heads, kv_heads, dim, page, torch.bfloat16, 24)
    g = torch.Generator().manual_seed(25)
    q[:], k[:] = 0, 0
    q[..., 0] = 1.0
    k[..., 0] = torch.randint(7, 48, k.shape[:3], generator=g).to(torch.int8)
    for s in range(sequences):
        p = int(table[s, at // page])
        k[p, :, at % page, 0] = 127
        v[p, :, :dim // 2, at % page] = 0
    scales[..., 0], scales[..., 1] = 1.0, 100.0
    scale = 0.25 * 0.6931471805599453   # a quarter of a bit for a step of a key
    got = attend(q, (k, v, scales), table, lengths, counts, scale=scale, max_query=count, max_length=length).double().cpu()
    out, spread, size = attend_plain(q, k, v, scales, table, lengths, counts, scale)
    low = 2.0 ** -31 * 100.0 * 127.0 * length
    bound = 2.0 ** -8 * out.abs() + (1.25 * 2.0 ** -11 + 2.0 * 2.0 ** -20 * size) * spread + low
    off = (got - out).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    # nothing is lost: those channels are sums of hundreds of such weights, many times what rounding may take from them
    assert float(spread[..., :dim // 2].min()) > 10 * low and bool((got[..., :dim // 2] != 0).any())


@pytest.mark.parametrize("extension", [True, False], ids=["extension", "without"])
def test_sizes_that_are_refused(extension, monkeypatch):
    """The same refusals with the extension module and without: no heads, tokens past 32 bits."""
    import types

    if not extension:
        monkeypatch.setattr(qm, "_ext", types.SimpleNamespace(**dict.fromkeys(qm._EXT_FUNCTIONS, lambda *a: None)))
    cache = [t.cuda() for t in make_cache(4, 2, 64, 16, 15)]
    table, n = torch.zeros(1, 3, dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    one = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    none, many = [t[:, :0].contiguous() for t in cache], one.expand(2 ** 31 + 1, 2, 64)
    for call in (lambda: kv_cache.attend(one, *none, table, n), lambda: kv_cache.append(one[:, :0], one[:, :0], *none, table, n), lambda: kv_cache.read(*none, n),
                 lambda: kv_cache.attend(many, *cache, table, n), lambda: kv_cache.append(many, many, *cache, table, n),
                 lambda: qm.gemm_grouped(one[0, :, :64].expand(2, 64)[:1].expand(2 ** 31 + 1, 64), torch.zeros(4, 32, dtype=torch.int8, device="cuda"),
                                         torch.ones(4, 2, dtype=torch.float16, device="cuda"), 32)):
        with pytest.raises(qm.QuadmulError):
            call()

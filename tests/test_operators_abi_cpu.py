"""Argument checks of the C entries for grouped weights and the 8-bit cache, and the sizes of their workspaces: no kernel is launched."""
import ctypes

import torch
import pytest

import quadmul_amd as qm

ONE = 4096  # never dereferenced: the checks come first


def grouped(lib, x=ONE, dtype=1, stride=256, b=ONE, scale=ONE, scale_dtype=1, group=128, bias=None, d=ONE, m=4, n=64, k=256, ws=None, ws_bytes=0):
    return lib.qm_gemm_grouped_i4(x, dtype, stride, b, scale, scale_dtype, group, bias, d, m, n, k, None, ws, ws_bytes)


def test_grouped_status_codes():
    lib = qm.library()
    assert grouped(lib, dtype=3) == -6 and grouped(lib, scale_dtype=2) == -6 and grouped(lib, dtype=9) == -6
    for bad in ({"k": 255}, {"m": -1}, {"n": -1}, {"k": -2}, {"group": 0}, {"group": 48}, {"group": -32}, {"stride": 255}):
        assert grouped(lib, **bad) == -2, bad
    for null in ("x", "b", "scale", "d"):
        assert grouped(lib, **{null: None}) == -1, null
    assert grouped(lib, x=ONE + 1) == -5 and grouped(lib, d=ONE + 1) == -5 and grouped(lib, scale=ONE + 1) == -5 and grouped(lib, bias=ONE + 1) == -5
    assert grouped(lib, scale_dtype=3, scale=ONE + 2) == -5 and grouped(lib, ws=ONE + 8, ws_bytes=64) == -5
    assert grouped(lib, m=0, x=None, d=None) == 0 and grouped(lib, n=0, b=None, d=None) == 0
    need = lib.qm_gemm_grouped_workspace_bytes(16, 4096, 28672, 128, 16)
    assert need > 0 and grouped(lib, m=16, n=4096, k=28672, stride=28672) == -7 and grouped(lib, m=16, n=4096, k=28672, stride=28672, ws=ONE, ws_bytes=need - 1) == -7


def test_grouped_workspace():
    size = qm.library().qm_gemm_grouped_workspace_bytes
    assert size(1, 4096, 4096, 128, 16) == 0 and size(2048, 11008, 4096, 128, 16) == 0
    assert size(16, 4096, 28672, 128, 16) % (16 * 4096 * 4) == 0
    assert size(16, 4096, 28672, 128, 4) == 0 and size(16, 4096, 28670, 128, 16) == 0    # the kernel for any address
    assert size(-1, 4096, 28672, 128, 16) == size(16, 4096, 28671, 128, 16) == size(16, 4096, 28672, 40, 16) == 0


def cache(**changes):
    c = qm.KvCache(ONE, ONE, ONE, 8, 2, 16, 64, ONE, ONE, None, 3, 4)
    for k, v in changes.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def fresh(**changes):
    n = qm.KvNew(ONE, ONE, None, None, 128, 64, 128, 64, 0, 0, None, None, 3, 0, 1, 0, 0, 0, 1)
    for k, v in changes.items():
        setattr(n, k, v)
    return ctypes.byref(n)


BAD_CACHES = [({"pages": -1}, -2), ({"kv_heads": 0}, -2), ({"kv_heads": 5000}, -2), ({"head_dim": 80}, -2), ({"page_size": 8}, -2), ({"page_size": 24}, -2), ({"k": None}, -1),
              ({"scales": None}, -1), ({"k": ONE + 8}, -5), ({"v": ONE + 4}, -5), ({"scales": ONE + 4}, -5)]
BAD_SEQUENCES = [({"sequences": -1}, -2), ({"table_width": -1}, -2), ({"lengths": None}, -1), ({"block_table": None}, -1), ({"lengths": ONE + 2}, -5)]


def test_append_status_codes():
    f = qm.library().qm_kv_append_i8
    for bad, code in BAD_CACHES + BAD_SEQUENCES:
        assert f(cache(**bad), fresh(), None) == code, bad
    assert f(None, fresh(), None) == -1 and f(cache(), None, None) == -1
    for bad, code in (({"dtype": 3}, -6), ({"tokens": -1}, -2), ({"tokens": 4}, -2), ({"rotary_pairs": 33}, -2), ({"rotary_pairs": -1}, -2), ({"k": None}, -1), ({"v": None}, -1),
                      ({"q": ONE, "heads": 0}, -2), ({"q": ONE, "heads": 4}, -1), ({"rotary_pairs": 8, "positions": 0, "cos": ONE, "sin": ONE}, -2),
                      ({"rotary_pairs": 8, "positions": 5}, -1), ({"k": ONE + 1}, -5), ({"positions": -1}, -2), ({"rotary_pairs": 8, "positions": 5, "cos": ONE + 2, "sin": ONE}, -5)):
        assert f(cache(), fresh(**bad), None) == code, bad
    assert f(cache(), fresh(tokens=0, k=None, v=None), None) == 0
    assert f(cache(sequences=0), fresh(tokens=3), None) == -2


def test_attend_status_codes_and_workspace():
    lib = qm.library()

    def f(c=None, q=ONE, dtype=1, out=ONE, tokens=3, heads=4, window=0, ws=None, ws_bytes=0, longest=0):
        return lib.qm_kv_attend_i8(c or cache(), q, dtype, 256, 64, out, tokens, heads, 1.0, 1, window, 1, longest, None, ws, ws_bytes)

    for bad, code in BAD_CACHES + BAD_SEQUENCES:
        assert f(cache(**bad)) == code, bad
    for bad, code in (({"dtype": 3}, -6), ({"tokens": -1}, -2), ({"tokens": 4}, -2), ({"heads": 3}, -2), ({"heads": 0}, -2), ({"window": -1}, -2), ({"q": None}, -1), ({"out": None}, -1),
                      ({"q": ONE + 1}, -5), ({"ws": ONE + 8, "ws_bytes": 1 << 20}, -5)):
        assert f(**bad) == code, bad
    assert f(tokens=0, q=None, out=None) == 0
    size = lib.qm_kv_attend_workspace_bytes
    wide = dict(table_width=4096, sequences=2, query_start=ONE)
    need = size(cache(**wide), 2, 4, 0, 1, 65536)
    assert need > 0 and size(cache(**wide), 2, 4, 0, 1, 512) == 0 and size(cache(**wide), 2, 4, 256, 1, 65536) == 0   # short, or short for the window
    assert f(cache(**wide), tokens=2, longest=65536) == -7 and f(cache(**wide), tokens=2, longest=65536, ws=ONE, ws_bytes=need - 1) == -7
    assert size(cache(page_size=8), 2, 4, 0, 1, 65536) == 0


def test_read_status_codes():
    f = qm.library().qm_kv_read_i8
    for bad, code in BAD_CACHES:
        assert f(cache(**bad), ONE, 2, 1, ONE, ONE, None) == code, bad
    assert f(cache(), ONE, 2, 3, ONE, ONE, None) == -6 and f(cache(), ONE, -1, 1, ONE, ONE, None) == -2 and f(cache(), None, 2, 1, ONE, ONE, None) == -1
    assert f(cache(), ONE, 2, 1, ONE + 8, ONE, None) == -5 and f(cache(), ONE + 2, 2, 1, ONE, ONE, None) == -5
    assert f(cache(), None, 0, 1, None, None, None) == 0 and f(cache(pages=0), ONE, 2, 1, ONE, ONE, None) == -2


def test_traceable_forms():
    import quadmul  # noqa: F401  (registers the operators)

    ops, meta = torch.ops.quadmul, lambda *s, dtype=torch.float16: torch.empty(s, dtype=dtype, device="meta")
    y = ops.gemm_grouped(meta(3, 256), meta(64, 128, dtype=torch.int8), meta(64, 2), 128, None)
    assert y.shape == (3, 64) and y.dtype == torch.float16
    with pytest.raises(RuntimeError):
        ops.gemm_grouped(meta(3, 256), meta(64, 128, dtype=torch.int8), meta(64, 2), 64, None)
    codes = meta(8, 2, 16, 64, dtype=torch.int8), meta(8, 2, 64, 16, dtype=torch.int8), meta(8, 2, 2, dtype=torch.float32)
    table, lengths = meta(3, 4, dtype=torch.int32), meta(3, dtype=torch.int32)
    q, k = meta(3, 4, 64), meta(3, 2, 64)
    assert ops.kv_append(k, k, *codes, table, lengths, None, None, None, False, 1) is None
    assert ops.kv_append_rotate(q, k, k, *codes, table, lengths, None, None, None, False, 1).shape == q.shape
    assert ops.kv_attend(q, *codes, table, lengths, None, None, True, 0, 1, 64).shape == q.shape
    written = [a.name for a in ops.kv_append.default._schema.arguments if a.alias_info is not None and a.alias_info.is_write]
    assert written == ["cache_k", "cache_v", "scales"]


def test_sequences_are_cut_however_many_there_are():
    size = qm.library().qm_kv_attend_workspace_bytes
    for sequences in (2, 256, 257, 1000, 4096):
        c = cache(table_width=8192, sequences=sequences)
        assert size(c, sequences, 4, 0, 0, 131072) > sequences * 8, sequences


def test_a_packed_token_each_needs_no_hint():
    """As many packed tokens as sequences, or fewer: the plan is that of max_query = 1."""
    size = qm.library().qm_kv_attend_workspace_bytes
    for sequences, tokens in ((32, 32), (64, 50), (300, 300), (1, 1)):
        c = cache(table_width=8192, sequences=sequences, query_start=ONE)
        assert size(c, tokens, 8, 0, 0, 8192) == size(c, tokens, 8, 0, 1, 8192) > 0
    c = cache(table_width=8192, sequences=32, query_start=ONE)
    assert size(c, 33, 8, 0, 0, 8192) == size(c, 33, 8, 0, 33, 8192) != size(c, 33, 8, 0, 1, 8192)

"""The attention block (quadmul_amd/attention.py): prompts, then tokens one by one, eagerly and as a replayed graph, against a plain float64 model
that keeps every key and value as it is."""
import math

import pytest
import torch

import quadmul_amd as qm
from quadmul_amd.attention import CachedAttention, rotation
from quadmul_amd.kv_cache import PagedKVCache
from quadmul_amd.linear import W4A16Linear
from kv_util import rotate, starts

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM = 512, 8, 2, 64


def layer(n, k, seed, dtype):
    w = (torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) / math.sqrt(k)).to(dtype)
    made = W4A16Linear.from_float(w.cuda(), 64)
    values = qm.unpack_int4(made.weight_packed).double().cpu() * made.weight_scale.double().cpu().repeat_interleave(64, dim=1)
    return made, values


class Plain:
    """One sequence at a time in float64: no quantised cache."""

    def __init__(self, w_in, w_out, cos, sin, dtype):
        self.w_in, self.w_out, self.cos, self.sin, self.dtype, self.held = w_in, w_out, cos, sin, dtype, {}

    def __call__(self, s, x):
        qkv = (x.double() @ self.w_in.T).to(self.dtype).double()
        q, k, v = qkv.split((HEADS * DIM, KV * DIM, KV * DIM), dim=1)
        q, k, v = q.reshape(-1, HEADS, DIM), k.reshape(-1, KV, DIM), v.reshape(-1, KV, DIM)
        old = self.held.get(s, (torch.zeros(0, KV, DIM, dtype=torch.float64),) * 2)
        pos = torch.arange(old[0].shape[0], old[0].shape[0] + x.shape[0])
        k, v = torch.cat((old[0], rotate(k, pos, self.cos, self.sin, False))), torch.cat((old[1], v))
        self.held[s] = (k, v)
        q = rotate(q, pos, self.cos, self.sin, False)
        scores = torch.matmul(q.transpose(0, 1), k.repeat_interleave(HEADS // KV, dim=1).permute(1, 2, 0).contiguous()) / math.sqrt(DIM)
        scores.masked_fill_(torch.arange(k.shape[0]) > pos[:, None], -math.inf)
        o = torch.matmul(torch.softmax(scores, dim=-1), v.repeat_interleave(HEADS // KV, dim=1).transpose(0, 1).contiguous()).transpose(0, 1)
        return o.reshape(-1, HEADS * DIM) @ self.w_out.T


def near(got, want):
    """What 8 bits a key and value leave, with the scale of a page of 16 tokens: steps of 1 / 127 of the largest of a thousand normal values (3.5 of their
    deviation) are errors of 3.5 / 127 / sqrt(12) = 0.8 % each, less in the mean over tokens; twice that for the keys' way through the softmax; 2.5 %."""
    assert float((got.double().cpu() - want).norm() / want.norm()) < 0.025


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_prompts_then_tokens(dtype):
    (qkv, w_in), (out, w_out) = layer((HEADS + 2 * KV) * DIM, HIDDEN, 1, dtype), layer(HIDDEN, HEADS * DIM, 2, dtype)
    cos, sin = rotation(128, DIM)
    block = CachedAttention(qkv, out, HEADS, KV, cos, sin).cuda()
    plain = Plain(w_in, w_out, cos.cpu(), sin.cpu(), dtype)
    cache = PagedKVCache(40, KV, DIM)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(3)).to(torch.int32)[:24].reshape(3, 8).cuda()
    g = torch.Generator().manual_seed(4)
    counts = [37, 1, 64]
    x = torch.randn(sum(counts), HIDDEN, generator=g).to(dtype)
    y = block(x.cuda(), cache, table, torch.tensor(counts, dtype=torch.int32, device="cuda"), starts(counts).cuda(), max_query=64)
    near(y, torch.cat([plain(s, p) for s, p in enumerate(x.split(counts))]))

    # a graph of one decode step, replayed with other tokens and lengths, and with eager work in between
    x_now, lengths = torch.zeros(3, HIDDEN, dtype=dtype, device="cuda"), torch.tensor([c + 1 for c in counts], dtype=torch.int32, device="cuda")
    first = torch.randn(3, HIDDEN, generator=g).to(dtype)
    x_now.copy_(first)
    y = block(x_now, cache, table, lengths)
    near(y, torch.cat([plain(s, first[s:s + 1]) for s in range(3)]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(x_now, cache, table, lengths)
    for step in range(20):
        new = torch.randn(3, HIDDEN, generator=g).to(dtype)
        x_now.copy_(new)
        lengths.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        near(y, torch.cat([plain(s, new[s:s + 1]) for s in range(3)]))
        if step % 7 == 0:
            again = block(x_now, cache, table, lengths)   # the same token once more: the same codes, the same result
            assert torch.equal(again, y)


def test_without_rotation_and_in_parts():
    """A prompt in two pieces gives what it gives in one, but for the rounding of a page that both pieces are in."""
    (qkv, w_in), (out, w_out) = layer((HEADS + 2 * KV) * DIM, HIDDEN, 5, torch.float16), layer(HIDDEN, HEADS * DIM, 6, torch.float16)
    block = CachedAttention(qkv, out, HEADS, KV).cuda()
    x = torch.randn(50, HIDDEN, generator=torch.Generator().manual_seed(7)).to(torch.float16).cuda()
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    n = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")
    whole, parts = PagedKVCache(4, KV, DIM), PagedKVCache(4, KV, DIM)
    a = block(x, whole, table, n(50))
    b = torch.cat((block(x[:32], parts, table, n(32)), block(x[32:], parts, table, n(50))))
    assert torch.equal(whole.k, parts.k) and torch.equal(whole.v, parts.v)
    assert float((a.float() - b.float()).norm() / a.float().norm()) < 2e-3
    plain = Plain(w_in, w_out, None, None, torch.float16)
    near(a, plain(0, x.cpu()))


def test_layers_refuse_and_take_any_leading_sizes():
    w = torch.randn(96, 256, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    made = W4A16Linear.from_float(w, 64, torch.zeros(96))
    x = torch.randn(2, 3, 256, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    made = made.cuda()
    assert made(x).shape == (2, 3, 96) and torch.equal(made(x).reshape(6, 96), made(x.reshape(6, 256)))
    assert "group_size=64" in repr(made)
    with pytest.raises(qm.QuadmulError):
        made(x[..., :128])
    with pytest.raises(qm.QuadmulError):
        W4A16Linear(made.weight_packed, made.weight_scale, 48)
    with pytest.raises(qm.QuadmulError):
        W4A16Linear(made.weight_packed, made.weight_scale[:, :2], 64)
    with pytest.raises(qm.QuadmulError):
        CachedAttention(made, made, 3, 2)
    with pytest.raises(qm.QuadmulError):
        CachedAttention(made, made, 1, 1, None, torch.ones(1, 1))

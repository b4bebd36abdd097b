"""A mixture of experts on packed int4 weights: the router's choice, products with the weights of each token's experts, their gated MLP (no
counterpart in the reference, which is one product).

    chosen, weights = moe.route(logits, top_k)                          # [tokens, top_k] int32 and float32
    y = moe.mlp(x, chosen, weights, up, up_scale, down, down_scale, group_size)
    z = moe.gemm_experts(x, chosen, weight, weight_scale, group_size)   # [tokens, top_k, n]: one matrix by itself

    layer = SparseMLP(router, W4A16Experts.from_float(w_up, w_down), top_k)   # the three as a module
    y = layer(x)

The weights of an expert are those of :func:`quadmul_amd.gemm_grouped`, all experts' in one tensor: ``weight`` [experts, n, k/2] int8 or uint8, ``weight_scale``
[experts, n, ceil(k / group_size)] float32 or of the activations' type. An expert number outside ``0 .. experts - 1`` (-1, say) is none: of another GPU, or of a
token of padding; it adds nothing. All calls are asynchronous, on the current stream, look at no number on the host and may be captured
into a HIP graph; none is differentiable. Exact definitions: ``include/qm_abi.h``.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import ExpertWeights, QuadmulError, _check, _has_extension, _is_byte, _native, _stream_ptr, library, quantize_groups

SCORES = ("softmax", "sigmoid")
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 64, 64

_KINDS = {torch.float16: 1, torch.bfloat16: 2, torch.float32: 3}
_INT_MAX = 2 ** 31 - 1
_RULE = {"scores": "softmax", "groups": 1, "top_groups": 1, "group_best": 2, "renormalise": False, "scale": 1.0}  # route's options and what they are without a word


def _check_rule(what: str, experts: int, top_k: int, scores: str, groups: int, top_groups: int, group_best: int) -> None:
    if scores not in SCORES:
        raise QuadmulError(f"{what}: scores must be one of {SCORES}")
    if not (1 <= groups <= MAX_GROUPS and experts % groups == 0 and 1 <= top_groups <= groups and group_best in (1, 2)):
        raise QuadmulError(f"{what}: groups must divide the experts and be at most {MAX_GROUPS}, top_groups at most as many, group_best 1 or 2")
    if not 1 <= top_k <= min(MAX_TOP_K, experts // groups * top_groups):
        raise QuadmulError(f"{what}: top_k must be 1 to {MAX_TOP_K}, and no more than the experts to choose from")


def route(logits: torch.Tensor, top_k: int, *, bias: Optional[torch.Tensor] = None, scores: str = "softmax", groups: int = 1, top_groups: int = 1, group_best: int = 2,
          renormalise: bool = False, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The experts of each token, best first, and their weights: ``logits`` [tokens, experts] float32, float16 or bfloat16 -> ``(chosen [tokens, top_k] int32,
    weights [tokens, top_k] float32)``.

    ``scores``: "softmax" over all experts or "sigmoid" of each; ``bias`` [experts] float32 is added for the choice, not for the weights. With ``groups`` > 1 the
    experts are as many equal runs and only those in the ``top_groups`` groups of the largest worth can be chosen: the sum of their ``group_best`` (1 or 2) best.
    ``renormalise``: the weights divided by their sum; ``scale``: times this. Scores, the choice and the weights are worked out in 64 bits; of equal experts the lower number
    is chosen. At most 1024 experts, 64 groups, a ``top_k`` of 64."""
    if scores not in SCORES:
        raise QuadmulError(f"route: scores must be one of {SCORES}")
    top_k, groups, top_groups, group_best, renormalise, scale = int(top_k), int(groups), int(top_groups), int(group_best), bool(renormalise), float(scale)
    if _has_extension():
        return _native("moe_route", logits, top_k, bias, scores == "sigmoid", groups, top_groups, group_best, renormalise, scale)
    if not (logits.is_cuda and logits.dim() == 2 and logits.dtype in _KINDS and logits.shape[0] <= _INT_MAX and 1 <= logits.shape[1] <= MAX_EXPERTS):
        raise QuadmulError(f"route: the logits must be a GPU tensor [tokens, 1 to {MAX_EXPERTS} experts], float32, float16 or bfloat16")
    tokens, experts = logits.shape
    _check_rule("route", experts, top_k, scores, groups, top_groups, group_best)
    if bias is not None and not (bias.device == logits.device and bias.dtype == torch.float32 and bias.is_contiguous() and bias.shape == (experts,)):
        raise QuadmulError(f"route: the bias must be a contiguous float32 vector of {experts} elements on the logits' device")
    if (experts > 1 and logits.stride(1) != 1) or (tokens > 1 and logits.stride(0) < experts):
        logits = logits.contiguous()
    chosen = torch.empty((tokens, top_k), dtype=torch.int32, device=logits.device)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=logits.device)
    with torch.cuda.device(logits.device):
        st = library().qm_moe_route(logits.data_ptr(), _KINDS[logits.dtype], logits.stride(0) if tokens > 1 else experts, tokens, experts, top_k,
                                    None if bias is None else bias.data_ptr(), SCORES.index(scores), groups, top_groups, group_best, int(renormalise), scale,
                                    chosen.data_ptr(), weights.data_ptr(), _stream_ptr(logits))
    _check(st, "qm_moe_route")
    return chosen, weights


def _weights(what, x, weight, scale, group, bias) -> ExpertWeights:
    if not (weight.dim() == 3 and _is_byte(weight) and weight.is_contiguous()):
        raise QuadmulError(f"{what}: the weights must be contiguous [experts, n, k / 2] int8 or uint8 tensors (packed int4)")
    if group < 32 or group % 32 or group > _INT_MAX:
        raise QuadmulError(f"{what}: the group size must be a multiple of 32")
    experts, n, k = weight.shape[0], weight.shape[1], weight.shape[2] * 2
    if max(experts, n, k) > _INT_MAX:
        raise QuadmulError(f"{what}: sizes must fit in int32")
    if not (scale.shape == (experts, n, -(-k // group)) and scale.is_contiguous() and scale.dtype in (torch.float32, x.dtype)):
        raise QuadmulError(f"{what}: the scales must be contiguous [experts, n, ceil(k / group)] tensors of float32 or of x's type")
    if not weight.device == scale.device == x.device:
        raise QuadmulError(f"{what}: all tensors must be on the same device")
    if bias is not None and not (bias.device == x.device and bias.dtype == x.dtype and bias.is_contiguous() and bias.shape == (experts, n)):
        raise QuadmulError(f"{what}: the bias must be a contiguous [experts, n] tensor of x's type on x's device")
    return ExpertWeights(weight.data_ptr(), scale.data_ptr(), None if bias is None else bias.data_ptr(), _KINDS[scale.dtype], experts, n, k, group)


def _activations(what, x, chosen, dims):
    if not (x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and x.dim() in dims and x.shape[-1] % 2 == 0):
        raise QuadmulError(f"{what}: x must be a float16 or bfloat16 GPU tensor [tokens, k]{' or [tokens, top_k, k]' if 3 in dims else ''}, k even")
    if not (chosen.device == x.device and chosen.dtype == torch.int32 and chosen.dim() == 2 and chosen.is_contiguous() and chosen.shape[0] == x.shape[0]):
        raise QuadmulError(f"{what}: the chosen experts must be a contiguous int32 tensor [tokens, top_k] on x's device")
    if max(*chosen.shape, chosen.numel()) > _INT_MAX:
        raise QuadmulError(f"{what}: tokens times top_k must fit in int32")


def _aligned(x):
    """Rows that the kernels for few rows to an expert can load, sixteen aligned bytes at a time; others are copied."""
    apart = x.data_ptr() % 16 != 0 or any(n > 1 and by % 8 for n, by in zip(x.shape[:-1], x.stride()[:-1]))
    if (x.shape[-1] > 1 and x.stride(-1) != 1) or (apart and x.shape[-1] % 32 == 0):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def gemm_experts(x: torch.Tensor, chosen: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, group_size: int, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t, j] = x[t] @ weight[e].T + bias[e]`` with ``e = chosen[t, j]``, as :func:`quadmul_amd.gemm_grouped` gives it, ``[tokens, top_k, n]``; zeros where ``e`` is
    no expert.

    ``x`` float16 or bfloat16: [tokens, k], a row for all of a token's choices, or [tokens, top_k, k], one for each; ``chosen`` [tokens, top_k] int32;
    ``bias`` [experts, n] of ``x``'s type. Sums are in float32 and rounded once; what is lost of bf16 on the way to the matrix cores stands at ``qm_gemm_experts_i4``."""
    group_size = int(group_size)
    if _has_extension():
        return _native("gemm_experts", x, chosen, weight, weight_scale, group_size, bias)
    _activations("gemm_experts", x, chosen, (2, 3))
    if x.dim() == 3 and x.shape[1] != chosen.shape[1]:
        raise QuadmulError("gemm_experts: x must have a row for each choice, or one for each token")
    w = _weights("gemm_experts", x, weight, weight_scale, group_size, bias)
    if w.k != x.shape[-1]:
        raise QuadmulError("gemm_experts: the weights must be [experts, n, k / 2], k x's last dimension")
    x = _aligned(x)
    tokens, top_k = chosen.shape
    y = torch.empty((tokens, top_k, w.n), dtype=x.dtype, device=x.device)
    need = library().qm_gemm_experts_workspace_bytes(ctypes.byref(w), tokens, top_k)
    scratch = torch.empty((need,), dtype=torch.uint8, device=x.device) if need else None
    with torch.cuda.device(x.device):
        st = library().qm_gemm_experts_i4(x.data_ptr(), _KINDS[x.dtype], x.stride(0), x.stride(1) if x.dim() == 3 else 0, chosen.data_ptr(), ctypes.byref(w), y.data_ptr(),
                                          tokens, top_k, _stream_ptr(x), scratch.data_ptr() if need else None, need)
    _check(st, "qm_gemm_experts_i4")
    return y


def mlp(x: torch.Tensor, chosen: torch.Tensor, weights: torch.Tensor, up: torch.Tensor, up_scale: torch.Tensor, down: torch.Tensor, down_scale: torch.Tensor,
        group_size: int) -> torch.Tensor:
    """``y[t] = sum_j weights[t, j] * (silu(a[:inner]) * a[inner:]) @ down[e].T`` with ``a = x[t] @ up[e].T`` and ``e = chosen[t, j]``: [tokens, hidden] of ``x``'s type.

    ``up`` [experts, 2 * inner, hidden/2], its first ``inner`` rows the gates; ``down`` [experts, hidden, inner/2]; ``weights`` [tokens, top_k] float32. The gated
    products are rounded to ``x``'s type, whatever else is summed stays in float32 until ``y`` is rounded."""
    group_size = int(group_size)
    if _has_extension():
        return _native("moe_mlp", x, chosen, weights, up, up_scale, down, down_scale, group_size)
    _activations("mlp", x, chosen, (2,))
    if not (weights.device == x.device and weights.dtype == torch.float32 and weights.is_contiguous() and weights.shape == chosen.shape):
        raise QuadmulError("mlp: the weights of the chosen must be a contiguous float32 tensor [tokens, top_k] on x's device")
    u, d = _weights("mlp", x, up, up_scale, group_size, None), _weights("mlp", x, down, down_scale, group_size, None)
    tokens, hidden = x.shape
    if not (u.k == d.n == hidden and u.n == 2 * d.k and u.experts == d.experts):
        raise QuadmulError("mlp: up must be [experts, 2 inner, hidden / 2], down [experts, hidden, inner / 2]")
    x = _aligned(x)
    y = torch.empty((tokens, hidden), dtype=x.dtype, device=x.device)
    need = library().qm_moe_mlp_workspace_bytes(ctypes.byref(u), ctypes.byref(d), tokens, chosen.shape[1])
    scratch = torch.empty((need,), dtype=torch.uint8, device=x.device) if need else None
    with torch.cuda.device(x.device):
        st = library().qm_moe_mlp_i4(x.data_ptr(), _KINDS[x.dtype], x.stride(0), chosen.data_ptr(), weights.data_ptr(), ctypes.byref(u), ctypes.byref(d), y.data_ptr(), tokens,
                                     chosen.shape[1], _stream_ptr(x), scratch.data_ptr() if need else None, need)
    _check(st, "qm_moe_mlp_i4")
    return y


class _Float32Kept(torch.nn.Module):
    """A module whose float32 buffers stay float32 where it is cast (``to(dtype)``, ``half``, ``bfloat16``, ``double``): a router that is rounded chooses other experts,
    :func:`route` takes its bias in float32 only, and the products take float32 scales beside activations of either type. Buffers of 16 bits follow the cast."""

    def _apply(self, fn, recurse=True):
        kept = {name: t for name, t in self._buffers.items() if t is not None and t.dtype == torch.float32}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            now = self._buffers[name]
            if now.dtype != torch.float32:
                self._buffers[name] = t.to(now.device)
        return self


class W4A16Experts(_Float32Kept):
    """The gated MLPs of a layer's experts: ``forward(x, chosen, weights)`` is :func:`mlp`, for ``x`` [..., hidden] with as many rows as ``chosen`` has. A cast of the
    module leaves float32 scales as they are."""

    def __init__(self, up_packed: torch.Tensor, up_scale: torch.Tensor, down_packed: torch.Tensor, down_scale: torch.Tensor, group_size: int):
        super().__init__()
        for t, s in ((up_packed, up_scale), (down_packed, down_scale)):
            if t.dim() != 3 or t.dtype not in (torch.int8, torch.uint8):
                raise QuadmulError("W4A16Experts: packed weights must be [experts, n, k / 2] int8 or uint8")
            if group_size < 32 or group_size % 32 or s.shape != (*t.shape[:2], -(-t.shape[2] * 2 // group_size)) or s.dtype not in _KINDS:
                raise QuadmulError("W4A16Experts: scales must be [experts, n, ceil(k / group_size)], the group size a multiple of 32")
        self.experts, self.hidden, self.inner, self.group_size = down_packed.shape[0], down_packed.shape[1], down_packed.shape[2] * 2, group_size
        if up_packed.shape != (self.experts, 2 * self.inner, self.hidden // 2) or self.hidden % 2:
            raise QuadmulError("W4A16Experts: up must be [experts, 2 inner, hidden / 2], down [experts, hidden, inner / 2]")
        for name, t in (("up_packed", up_packed), ("up_scale", up_scale), ("down_packed", down_packed), ("down_scale", down_scale)):
            self.register_buffer(name, t.contiguous())

    @classmethod
    def from_float(cls, up: torch.Tensor, down: torch.Tensor, group_size: int = 128, scale_dtype: Optional[torch.dtype] = None):
        """Quantise float weights (on the GPU) ``up`` [experts, 2 * inner, hidden] and ``down`` [experts, hidden, inner] group by group, one expert at a time;
        ``scale_dtype`` None: the scales in the weights' type, if that is one of 16 bits, else float32."""
        parts = []
        for w in (up, down):
            if w.dim() != 3 or w.shape[0] == 0:
                raise QuadmulError("W4A16Experts: expects up [experts, 2 inner, hidden] and down [experts, hidden, inner], an expert or more")
            kind = scale_dtype if scale_dtype is not None else w.dtype if w.dtype in (torch.float16, torch.bfloat16) else None
            each = [quantize_groups(e.contiguous(), group_size, kind) for e in w]
            parts += [torch.stack([p for p, _ in each]), torch.stack([s for _, s in each])]
        return cls(*parts, group_size)

    def forward(self, x: torch.Tensor, chosen: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.hidden:
            raise QuadmulError(f"W4A16Experts: last dimension of x must be {self.hidden}")
        flat = x if x.dim() == 2 else x.reshape(-1, self.hidden)
        y = mlp(flat, chosen, weights, self.up_packed, self.up_scale, self.down_packed, self.down_scale, self.group_size)
        return y if x.dim() == 2 else y.reshape(x.shape)

    def extra_repr(self) -> str:
        return f"experts={self.experts}, hidden={self.hidden}, inner={self.inner}, group_size={self.group_size}"


class SparseMLP(_Float32Kept):
    """``forward(x)``, ``x`` [..., hidden]: the router's logits (``router`` [experts, hidden], in its own type), :func:`route` with ``rule``'s options, the experts' MLPs. A cast
    of the module leaves a float32 router, the bias and float32 scales as they are."""

    def __init__(self, router: torch.Tensor, experts: W4A16Experts, top_k: int, bias: Optional[torch.Tensor] = None, **rule):
        super().__init__()
        if router.shape != (experts.experts, experts.hidden):
            raise QuadmulError(f"SparseMLP: the router must be [{experts.experts}, {experts.hidden}]")
        if router.dtype not in _KINDS:
            raise QuadmulError("SparseMLP: the router must be float32, float16 or bfloat16")
        if bias is not None and (bias.shape != (experts.experts,) or bias.dtype not in _KINDS):
            raise QuadmulError(f"SparseMLP: the bias must be float32 [{experts.experts}]")
        wrong = set(rule) - set(_RULE)
        if wrong:
            raise QuadmulError(f"SparseMLP: route has no option {', '.join(sorted(wrong))}")
        if not 1 <= experts.experts <= MAX_EXPERTS:
            raise QuadmulError(f"SparseMLP: 1 to {MAX_EXPERTS} experts")
        full = _RULE | rule
        _check_rule("SparseMLP", experts.experts, int(top_k), full["scores"], int(full["groups"]), int(full["top_groups"]), int(full["group_best"]))
        self.experts, self.top_k, self.rule = experts, top_k, rule
        self.register_buffer("router", router)
        self.register_buffer("bias", None if bias is None else bias.float().contiguous())

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.experts.hidden:
            raise QuadmulError(f"SparseMLP: last dimension of x must be {self.experts.hidden}")
        flat = x.reshape(-1, x.shape[-1])
        chosen, weights = route(flat.to(self.router.dtype) @ self.router.t(), self.top_k, bias=self.bias, **self.rule)
        return self.experts(flat, chosen, weights).reshape(x.shape)

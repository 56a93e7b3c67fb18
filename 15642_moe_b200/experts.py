"""Expert router in its general form with its gradient, and products with 4-bit weights.

The functions here take any expert count, layer width and routing rule, next to the fixed
DeepSeek-V3 layer of ``layer.py`` (256 experts, 7168 x 2048, FP8 weights; reference/moe_ref.py:26-42).
Like there, every call goes to ``libmoe_b200.so`` on the tensors' CUDA device and the current stream,
bad arguments raise ``RuntimeError``, and CPU tensors are rejected.

4-bit weights of a matrix [N, K]: ``codes`` uint8 [N, ceil(K / 2)], two codes per byte with the even
column in the low nibble; ``scale`` [N, ceil(K / group)] in the activations' type; ``zero`` uint8 of the
same shape with values 0 to 15, or None for 8. The weight is ``scale * (code - zero)``. The matrices of
several experts are stacked in a leading dimension.
"""
from __future__ import annotations

import functools
import operator
import struct

import torch

from . import _native

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SCORE = {"sigmoid": 0, "softmax": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}
_SCORES, _GROUP_SCORES = tuple(_SCORE), tuple(_GROUP_SCORE)
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS, MAX_ROWS = 1024, 32, 32, 65535
W4_GROUPS = (32, 64, 128)


# The handle of a device's current stream. torch.cuda.current_stream() builds a Stream object around it, which takes
# longer than the smallest kernels here.
_current_stream = torch._C._cuda_getCurrentRawStream
_lib = None


def _native_lib():
    global _lib
    if _lib is None:
        _lib = _native.cuda_lib()
    return _lib


# The argument structs of include/moe_b200.h, up to their last member, and the padding that may follow it.
_TAIL = bytes(4)
_ROUTE = struct.Struct("@5Pq9if").pack
_ROUTE_BACKWARD = struct.Struct("@5Pq6if").pack
_LINEAR = struct.Struct("@7P2q5i").pack
_EXPERTS = struct.Struct("@12P2q8i").pack


def _call(fn, index: int, args: bytes) -> None:
    """One C call with device `index` current."""
    args += _TAIL
    if index == torch.cuda.current_device():
        rc = fn(args)
    else:
        with torch.cuda.device(index):
            rc = fn(args)
    if rc:
        _native.check(rc)


def _fail(message: str) -> None:
    raise RuntimeError(message)


def _whole(name: str, value) -> int:
    try:
        return operator.index(value)
    except TypeError:
        _fail(f"{name} must be a whole number")


def _scale(value) -> float:
    if not hasattr(value, "__float__"):
        _fail("scale must be a number")
    return float(value)


# ------------------------------------------------------------------------------------ router
# The messages are built only where a check fails: a call is a few microseconds in all.
def _check_logits(logits) -> None:
    if logits.dim() != 2:
        _fail("logits must be [T, E]")
    if logits.dtype not in _DTYPE:
        _fail("logits must be float32, bfloat16 or float16")
    if not logits.is_cuda:
        _fail("logits must be a CUDA tensor")
    T, E = logits.shape
    if not 1 <= E <= MAX_EXPERTS:
        _fail(f"logits must have 1 to {MAX_EXPERTS} experts")
    if E > 1 and T > 0 and logits.stride(1) != 1:
        _fail("logits must have neighbouring experts in memory (stride 1)")


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
                  n_group: int = 1, topk_group: int = 1, group_score: str = "max", renormalize: bool = True,
                  scale: float = 1.0):
    """The ``top_k`` experts of each token and their weights: (idx int32 [T, top_k], weights fp32 [T, top_k]).

    ``logits`` [T, E] in float32, bfloat16 or float16, rows any distance apart; E up to 1024, top_k up to 32.
    Scores are the row's softmax or each logit's sigmoid. Experts are chosen by score + ``bias`` (fp32 [E]) and
    weighed by the score alone. With ``n_group`` > 1 the experts form n_group equal groups, scored by their best
    expert ("max") or the sum of their two best ("top2"), and only the ``topk_group`` best groups take part.
    ``idx`` is in descending order of the choice, ties to the lower expert. Experts with a logit (or bias) of -inf
    are never chosen; where a row has fewer than top_k experts left, idx is -1 and the weight 0. The weights are
    divided by their sum (plus 1e-20) if ``renormalize``, then multiplied by ``scale``. A NaN logit comes out as
    NaN weights. Scores, weights and their sums are in 32 bits; without a bias experts are compared by their logits, so those
    whose scores round together keep their order. Differentiable in ``logits`` (route_experts_backward); the choice, and with
    it the bias, has no gradient.

    The fixed router of moe_forward (reference/moe_ref.py:82-107) is score="sigmoid", n_group=8, topk_group=4,
    group_score="top2", top_k=8 over 256 experts.
    """
    if logits.requires_grad and torch.is_grad_enabled():
        return _RouteExperts.apply(logits, top_k, score, bias, n_group, topk_group, group_score, renormalize, scale)
    _check_logits(logits)
    T, E = logits.shape
    if score not in _SCORES:
        _fail("score must be 'softmax' or 'sigmoid'")
    if group_score not in _GROUP_SCORES:
        _fail("group_score must be 'max' or 'top2'")
    if not type(top_k) is type(n_group) is type(topk_group) is int:
        top_k, n_group, topk_group = _whole("top_k", top_k), _whole("n_group", n_group), _whole("topk_group", topk_group)
    if not (1 <= n_group <= MAX_GROUPS and E % n_group == 0):
        _fail(f"n_group must divide the experts and be 1 to {MAX_GROUPS}")
    if not 1 <= topk_group <= n_group:
        _fail("topk_group must be 1 to n_group")
    if not 1 <= top_k <= min(MAX_TOP_K, E // n_group * topk_group):
        _fail(f"top_k must be 1 to {MAX_TOP_K} and at most the experts of topk_group groups")
    if n_group > 1 and group_score == "top2" and E // n_group < 2:
        _fail("group_score 'top2' needs two experts per group")
    index, bias_ptr = logits.get_device(), 0
    if bias is not None:
        if not (bias.dtype == torch.float32 and bias.dim() == 1 and bias.shape[0] == E and bias.is_contiguous()
                and bias.is_cuda and bias.get_device() == index):
            _fail("bias must be a contiguous float32 [E] tensor on the logits' device")
        bias_ptr = bias.data_ptr()
    w = logits.new_empty((T, top_k), dtype=torch.float32)
    idx = torch.empty_like(w, dtype=torch.int32)
    if T:
        _call(_native_lib().moe_route_experts, index,
              _ROUTE(logits.data_ptr(), bias_ptr, idx.data_ptr(), w.data_ptr(), _current_stream(index), logits.stride(0),
                     _DTYPE[logits.dtype], T, E, top_k, _SCORE[score], n_group, topk_group, _GROUP_SCORE[group_score],
                     bool(renormalize), scale if type(scale) is float else _scale(scale)))
    return idx, w


def route_experts_backward(grad_weights: torch.Tensor, logits: torch.Tensor, idx: torch.Tensor, *,
                           score: str = "softmax", renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of route_experts' weights with respect to the logits: [T, E] in the logits' type.

    ``grad_weights`` fp32 [T, top_k], ``idx`` int32 [T, top_k] as route_experts returned it (distinct experts per
    row; -1 takes no part, and a row of -1 alone has a zero gradient), and the forward call's ``score``, ``renormalize`` and
    ``scale``. The choice of the experts has no gradient. The result itself is not differentiable."""
    _check_logits(logits)
    T, E = logits.shape
    if score not in _SCORES:
        _fail("score must be 'softmax' or 'sigmoid'")
    index = logits.get_device()
    if not (idx.dim() == 2 and idx.shape[0] == T and 1 <= idx.shape[1] <= MAX_TOP_K and idx.dtype == torch.int32
            and idx.is_contiguous() and idx.is_cuda and idx.get_device() == index):
        _fail(f"idx must be a contiguous int32 [T, top_k] tensor on the logits' device, top_k 1 to {MAX_TOP_K}")
    if not (grad_weights.shape == idx.shape and grad_weights.dtype == torch.float32 and grad_weights.is_contiguous()
            and grad_weights.is_cuda and grad_weights.get_device() == index):
        _fail("grad_weights must be a contiguous float32 [T, top_k] tensor on the logits' device")
    grad = logits.new_empty((T, E))
    if T:
        _call(_native_lib().moe_route_experts_backward, index,
              _ROUTE_BACKWARD(grad_weights.data_ptr(), logits.data_ptr(), idx.data_ptr(), grad.data_ptr(),
                              _current_stream(index), logits.stride(0), _DTYPE[logits.dtype], T, E, idx.shape[1],
                              _SCORE[score], bool(renormalize), scale if type(scale) is float else _scale(scale)))
    return grad


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, score, bias, n_group, topk_group, group_score, renormalize, scale):
        idx, w = route_experts(logits.detach(), top_k, score=score, bias=bias, n_group=n_group, topk_group=topk_group,
                               group_score=group_score, renormalize=renormalize, scale=scale)
        ctx.save_for_backward(logits, idx)
        ctx.rule = dict(score=score, renormalize=renormalize, scale=scale)
        ctx.mark_non_differentiable(idx)
        return idx, w

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, grad_weights):
        logits, idx = ctx.saved_tensors
        grad = route_experts_backward(grad_weights.contiguous(), logits, idx, **ctx.rule)
        return (grad,) + (None,) * 8


# ----------------------------------------------------------------------------- 4-bit products
class _NoGradient(torch.autograd.Function):
    """A product whose backward pass fails, as for torch's own operators without a derivative: a result without a graph
    would cut the gradient in silence."""

    @staticmethod
    def forward(ctx, name, product, *inputs):
        ctx.name = name
        return product()

    @staticmethod
    def backward(ctx, *_):
        _fail(f"{ctx.name} has no gradient: give it detached tensors, or call it under torch.no_grad()")


def _without_gradient(name, out, product, *inputs):
    if out is not None:
        _fail(f"{name} has no gradient: out= takes no inputs that require one")
    return _NoGradient.apply(name, product, *inputs)


def _w4(codes, scale, zero, group, shape, K, dtype, index, name) -> None:
    """Checks one 4-bit matrix (or a stack of them): `shape` without the columns, K columns."""
    if not (codes.dtype == torch.uint8 and codes.shape == (*shape, (K + 1) // 2) and codes.is_contiguous()):
        _fail(f"{name} must be a contiguous uint8 tensor of shape {[*shape, (K + 1) // 2]}")
    groups = (*shape, -(-K // group))
    if not (scale.dtype == dtype and scale.shape == groups and scale.is_contiguous()):
        _fail(f"{name}'s scale must be a contiguous {dtype} tensor of shape {list(groups)}")
    if not (codes.is_cuda and codes.get_device() == index and scale.is_cuda and scale.get_device() == index):
        _fail("all tensors must be on one device")
    if zero is not None and not (zero.dtype == torch.uint8 and zero.shape == groups and zero.is_contiguous()
                                 and zero.is_cuda and zero.get_device() == index):
        _fail(f"{name}'s zero must be a contiguous uint8 tensor of shape {list(groups)} on the same device")


def _check_x(x, group, what) -> None:
    if x.dim() != 2:
        _fail(f"x must be {what}")
    if x.dtype != torch.bfloat16 and x.dtype != torch.float16:
        _fail("x must be bfloat16 or float16")
    if not x.is_cuda:
        _fail("x must be a CUDA tensor")
    if group not in W4_GROUPS or type(group) is float:
        _fail("group must be 32, 64 or 128")
    if x.shape[0] > 0 and x.shape[1] > 1 and x.stride(1) != 1:
        _fail("x must have neighbouring columns in memory (stride 1)")


@functools.lru_cache(maxsize=4096)
def _linear_w4_workspace_bytes(M: int, N: int, K: int) -> int:
    return int(_native_lib().moe_linear_w4_workspace_bytes(M, N, K))


def linear_w4(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None, *,
              group: int = 128, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [M, K] (bfloat16 or float16, rows any distance apart) times the 4-bit W [N, K]: [M, N] in x's type.

    ``codes``, ``scale``, ``zero`` as in this module's description, ``group`` 32, 64 or 128. M up to 65535, any N and
    K from 1 on. ``out`` may not overlap an input. Sums are held in 32 bits and rounded once. There is no gradient: where
    ``x`` or ``scale`` requires one, the call works and a backward pass through its result raises ``RuntimeError``."""
    if (x.requires_grad or scale.requires_grad) and torch.is_grad_enabled():
        return _without_gradient("linear_w4", out, lambda: linear_w4(x, codes, scale, zero, group=group), x, scale)
    _check_x(x, group, "[M, K]")
    if codes.dim() != 2:
        _fail("codes must be [N, ceil(K / 2)]")
    (M, K), N, index = x.shape, codes.shape[0], x.get_device()
    if not (K >= 1 and N >= 1):
        _fail("x and codes must have at least one column and one row")
    if M > MAX_ROWS:
        _fail(f"x must have at most {MAX_ROWS} rows")
    _w4(codes, scale, zero, group, (N,), K, x.dtype, index, "codes")
    if out is None:
        out = x.new_empty((M, N))
    elif not (out.dtype == x.dtype and out.shape == (M, N) and out.is_contiguous() and out.is_cuda
              and out.get_device() == index):
        _fail("out must be a contiguous [M, N] tensor of x's type on its device")
    if M:
        need = _linear_w4_workspace_bytes(M, N, K)
        workspace = x.new_empty(need, dtype=torch.uint8) if need else None
        _call(_native_lib().moe_linear_w4, index,
              _LINEAR(x.data_ptr(), codes.data_ptr(), scale.data_ptr(), 0 if zero is None else zero.data_ptr(),
                      out.data_ptr(), 0 if workspace is None else workspace.data_ptr(), _current_stream(index),
                      x.stride(0), need, _DTYPE[x.dtype], group, M, N, K))
    return out


@functools.lru_cache(maxsize=4096)
def experts_w4_workspace_bytes(T: int, top_k: int, E: int, H: int, I: int) -> int:
    """Bytes of experts_w4's workspace; 0 for sizes that it refuses."""
    if max(T, top_k, E, H, I) >= 2 ** 31 or min(T, top_k, E, H, I) < 0:
        return 0
    return int(_native_lib().moe_experts_w4_workspace_bytes(T, top_k, E, H, I))


def experts_w4(x: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor,
               w2: torch.Tensor, w2_scale: torch.Tensor, *, w13_zero: torch.Tensor | None = None,
               w2_zero: torch.Tensor | None = None, group: int = 128, local_offset: int = 0,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The routed experts of a layer with 4-bit weights: [T, H] in x's type.

    For token t and each pick j with expert e = idx[t, j] - local_offset in [0, E):
    out[t] += weights[t, j] * W2[e] (X1 * silu(X2)), [X1 | X2] = W13[e] x[t] (the reference's order of the
    halves, reference/moe_ref.py:129-130). Other picks (-1, experts of other GPUs) add nothing.

    ``x`` [T, H] bfloat16 or float16, rows any distance apart; ``idx`` int32 and ``weights`` fp32 [T, top_k], as
    route_experts returns them; ``w13`` codes uint8 [E, 2 I, ceil(H / 2)], ``w2`` codes uint8 [E, H, ceil(I / 2)]
    (16-byte aligned), scales and zero points as in this module's description. T up to 65535. ``out`` may not overlap an
    input. Each product's sums and the weighted sum are held in 32 bits and the result is rounded once; between the products
    the SwiGLU's result carries 16 bits (two bfloat16 terms: an error of at most 2^-17 of each value, where a bfloat16 output
    is rounded by up to 2^-8). There is no gradient: where ``x``, ``weights`` or a scale requires
    one, the call works and a backward pass through its result raises ``RuntimeError``."""
    if (x.requires_grad or weights.requires_grad or w13_scale.requires_grad or w2_scale.requires_grad) and torch.is_grad_enabled():
        return _without_gradient("experts_w4", out, lambda: experts_w4(
            x, idx, weights, w13, w13_scale, w2, w2_scale, w13_zero=w13_zero, w2_zero=w2_zero, group=group,
            local_offset=local_offset, workspace=workspace), x, weights, w13_scale, w2_scale)
    _check_x(x, group, "[T, H]")
    if not (w13.dim() == 3 and w13.shape[1] % 2 == 0):
        _fail("w13 must be [E, 2 I, ceil(H / 2)]")
    (T, H), index = x.shape, x.get_device()
    E, I = w13.shape[0], w13.shape[1] // 2
    if not (1 <= E <= MAX_EXPERTS and H >= 1 and I >= 1):
        _fail(f"w13 must hold 1 to {MAX_EXPERTS} experts")
    if T > MAX_ROWS:
        _fail(f"x must have at most {MAX_ROWS} tokens")
    if not 0 <= _whole("local_offset", local_offset) < 2 ** 31:
        _fail("local_offset must be 0 to 2^31 - 1")
    if not (idx.dim() == 2 and idx.shape[0] == T and 1 <= idx.shape[1] <= MAX_TOP_K and idx.dtype == torch.int32
            and idx.is_contiguous() and idx.is_cuda and idx.get_device() == index):
        _fail(f"idx must be a contiguous int32 [T, top_k] tensor on x's device, top_k 1 to {MAX_TOP_K}")
    if not (weights.shape == idx.shape and weights.dtype == torch.float32 and weights.is_contiguous()
            and weights.is_cuda and weights.get_device() == index):
        _fail("weights must be a contiguous float32 [T, top_k] tensor on x's device")
    _w4(w13, w13_scale, w13_zero, group, (E, 2 * I), H, x.dtype, index, "w13")
    _w4(w2, w2_scale, w2_zero, group, (E, H), I, x.dtype, index, "w2")
    if out is None:
        out = x.new_empty((T, H))
    elif not (out.dtype == x.dtype and out.shape == (T, H) and out.is_contiguous() and out.is_cuda
              and out.get_device() == index):
        _fail("out must be a contiguous [T, H] tensor of x's type on its device")
    if T == 0:
        return out
    top_k = idx.shape[1]
    need = experts_w4_workspace_bytes(T, top_k, E, H, I)
    if workspace is None:
        workspace = x.new_empty(need, dtype=torch.uint8)
    elif not (workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need
              and workspace.is_cuda and workspace.get_device() == index):
        _fail(f"workspace must be a contiguous uint8 tensor of at least {need} bytes on x's device")
    _call(_native_lib().moe_experts_w4, index,
          _EXPERTS(x.data_ptr(), idx.data_ptr(), weights.data_ptr(), w13.data_ptr(), w13_scale.data_ptr(),
                   0 if w13_zero is None else w13_zero.data_ptr(), w2.data_ptr(), w2_scale.data_ptr(),
                   0 if w2_zero is None else w2_zero.data_ptr(), out.data_ptr(), workspace.data_ptr(),
                   _current_stream(index), x.stride(0), workspace.numel(), _DTYPE[x.dtype], group, T, top_k, E,
                   local_offset, H, I))
    return out

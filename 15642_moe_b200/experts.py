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

import torch

from . import _native
from .layer import _check

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SCORE = {"sigmoid": 0, "softmax": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS, MAX_TOKENS = 1024, 32, 32, 65536
W4_GROUPS = (32, 64, 128)


def _call(fn, device: torch.device, *args) -> None:
    """One C call on `device` and its current stream."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _native.check(rc)


# ------------------------------------------------------------------------------------ router
def _logits(logits) -> tuple[int, int]:
    _check(logits.dim() == 2, "logits must be [T, E]")
    _check(logits.dtype in _DTYPE, "logits must be float32, bfloat16 or float16")
    _check(logits.is_cuda, "logits must be a CUDA tensor")
    T, E = logits.shape
    _check(1 <= E <= MAX_EXPERTS, f"logits must have 1 to {MAX_EXPERTS} experts")
    _check(T == 0 or logits.stride(1) == 1 or E == 1, "logits must have neighbouring experts in memory (stride 1)")
    return T, E


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
    NaN weights. Differentiable in ``logits`` (route_experts_backward).

    The fixed router of moe_forward (reference/moe_ref.py:82-107) is score="sigmoid", n_group=8, topk_group=4,
    group_score="top2", top_k=8 over 256 experts.
    """
    if logits.requires_grad and torch.is_grad_enabled():
        return _RouteExperts.apply(logits, top_k, score, bias, n_group, topk_group, group_score, renormalize, scale)
    T, E = _logits(logits)
    _check(score in _SCORE, "score must be 'softmax' or 'sigmoid'")
    _check(group_score in _GROUP_SCORE, "group_score must be 'max' or 'top2'")
    _check(1 <= n_group <= MAX_GROUPS and E % n_group == 0, f"n_group must divide the experts and be 1 to {MAX_GROUPS}")
    _check(1 <= topk_group <= n_group, "topk_group must be 1 to n_group")
    _check(1 <= top_k <= min(MAX_TOP_K, E // n_group * topk_group),
           f"top_k must be 1 to {MAX_TOP_K} and at most the experts of topk_group groups")
    _check(n_group == 1 or group_score == "max" or E // n_group >= 2, "group_score 'top2' needs two experts per group")
    if bias is not None:
        _check(bias.dtype == torch.float32 and bias.dim() == 1 and bias.shape[0] == E and bias.is_contiguous()
               and bias.device == logits.device, "bias must be a contiguous float32 [E] tensor on the logits' device")
    dev = logits.device
    idx = torch.empty((T, top_k), dtype=torch.int32, device=dev)
    w = torch.empty((T, top_k), dtype=torch.float32, device=dev)
    if T:
        _call(_native.cuda_lib().moe_route_experts, dev, logits.data_ptr(), _DTYPE[logits.dtype], logits.stride(0),
              None if bias is None else bias.data_ptr(), T, E, top_k, _SCORE[score], n_group, topk_group,
              _GROUP_SCORE[group_score], 1 if renormalize else 0, scale, idx.data_ptr(), w.data_ptr())
    return idx, w


def route_experts_backward(grad_weights: torch.Tensor, logits: torch.Tensor, idx: torch.Tensor, *,
                           score: str = "softmax", renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of route_experts' weights with respect to the logits: [T, E] in the logits' type.

    ``grad_weights`` fp32 [T, top_k], ``idx`` int32 [T, top_k] as route_experts returned it (distinct experts per
    row; -1 takes no part), and the forward call's ``score``, ``renormalize`` and ``scale``. The choice of the
    experts has no gradient."""
    T, E = _logits(logits)
    _check(score in _SCORE, "score must be 'softmax' or 'sigmoid'")
    _check(idx.dim() == 2 and idx.shape[0] == T and 1 <= idx.shape[1] <= MAX_TOP_K and idx.dtype == torch.int32
           and idx.is_contiguous() and idx.device == logits.device,
           f"idx must be a contiguous int32 [T, top_k] tensor on the logits' device, top_k 1 to {MAX_TOP_K}")
    _check(grad_weights.shape == idx.shape and grad_weights.dtype == torch.float32 and grad_weights.is_contiguous()
           and grad_weights.device == logits.device,
           "grad_weights must be a contiguous float32 [T, top_k] tensor on the logits' device")
    dev = logits.device
    grad = torch.empty((T, E), dtype=logits.dtype, device=dev)
    if T:
        _call(_native.cuda_lib().moe_route_experts_backward, dev, grad_weights.data_ptr(), logits.data_ptr(),
              _DTYPE[logits.dtype], logits.stride(0), idx.data_ptr(), T, E, idx.shape[1], _SCORE[score],
              1 if renormalize else 0, scale, grad.data_ptr())
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
    def backward(ctx, _, grad_weights):
        logits, idx = ctx.saved_tensors
        grad = route_experts_backward(grad_weights.contiguous(), logits, idx, **ctx.rule)
        return (grad,) + (None,) * 8


# ----------------------------------------------------------------------------- 4-bit products
def _w4(codes, scale, zero, group, lead, N, K, dtype, dev, name) -> None:
    """Checks one 4-bit matrix (or a stack of them) of N rows and K columns."""
    _check(codes.dtype == torch.uint8 and codes.shape == (*lead, N, (K + 1) // 2) and codes.is_contiguous(),
           f"{name} must be a contiguous uint8 tensor of shape {[*lead, N, (K + 1) // 2]}")
    shape = (*lead, N, -(-K // group))
    _check(scale.dtype == dtype and scale.shape == shape and scale.is_contiguous(),
           f"{name}'s scale must be a contiguous {dtype} tensor of shape {list(shape)}")
    _check(codes.device == dev and scale.device == dev, "all tensors must be on one device")
    if zero is not None:
        _check(zero.dtype == torch.uint8 and zero.shape == shape and zero.is_contiguous() and zero.device == dev,
               f"{name}'s zero must be a contiguous uint8 tensor of shape {list(shape)} on the same device")


def linear_w4(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None, *,
              group: int = 128, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [M, K] (bfloat16 or float16, rows any distance apart) times the 4-bit W [N, K]: [M, N] in x's type.

    ``codes``, ``scale``, ``zero`` as in this module's description, ``group`` 32, 64 or 128. Any M, N and K from 1
    on. Sums are held in 32 bits and rounded once."""
    _check(x.dim() == 2, "x must be [M, K]")
    _check(x.dtype == torch.bfloat16 or x.dtype == torch.float16, "x must be bfloat16 or float16")
    _check(x.is_cuda, "x must be a CUDA tensor")
    _check(group in W4_GROUPS, "group must be 32, 64 or 128")
    _check(codes.dim() == 2, "codes must be [N, ceil(K / 2)]")
    (M, K), N, dev = x.shape, codes.shape[0], x.device
    _check(K >= 1 and N >= 1, "x and codes must have at least one column and one row")
    _check(M == 0 or K == 1 or x.stride(1) == 1, "x must have neighbouring columns in memory (stride 1)")
    _w4(codes, scale, zero, group, (), N, K, x.dtype, dev, "codes")
    if out is None:
        out = torch.empty((M, N), dtype=x.dtype, device=dev)
    else:
        _check(out.dtype == x.dtype and out.shape == (M, N) and out.is_contiguous() and out.device == dev,
               "out must be a contiguous [M, N] tensor of x's type on its device")
    if M:
        lib, ws, need = _native.cuda_lib(), None, 0
        if M > 8:
            need = int(lib.moe_linear_w4_workspace_bytes(M, N, K))
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _call(lib.moe_linear_w4, dev, x.data_ptr(), _DTYPE[x.dtype], x.stride(0), codes.data_ptr(), scale.data_ptr(),
              None if zero is None else zero.data_ptr(), group, M, N, K, out.data_ptr(),
              None if ws is None else ws.data_ptr(), need)
    return out


def experts_w4_workspace_bytes(T: int, top_k: int, E: int, H: int, I: int) -> int:
    return int(_native.cuda_lib().moe_experts_w4_workspace_bytes(T, top_k, E, H, I))


def experts_w4(x: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor,
               w2: torch.Tensor, w2_scale: torch.Tensor, *, w13_zero: torch.Tensor | None = None,
               w2_zero: torch.Tensor | None = None, group: int = 128, local_offset: int = 0,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The routed experts of a layer with 4-bit weights: [T, H] in x's type.

    For token t and each pick j with expert e = idx[t, j] - local_offset in [0, E):
    out[t] += weights[t, j] * W2[e] (X1 * silu(X2)), [X1 | X2] = W13[e] x[t] (the reference's order of the
    halves, reference/moe_ref.py:129-130). Other picks (-1, experts of other GPUs) add nothing.

    ``x`` [T, H] bfloat16 or float16, rows any distance apart; ``idx`` int32 and ``weights`` fp32 [T, top_k], as
    route_experts returns them; ``w13`` codes uint8 [E, 2 I, ceil(H / 2)], ``w2`` codes uint8 [E, H, ceil(I / 2)],
    scales and zero points as in this module's description. Sums are held in 32 bits and rounded once."""
    _check(x.dim() == 2, "x must be [T, H]")
    _check(x.dtype == torch.bfloat16 or x.dtype == torch.float16, "x must be bfloat16 or float16")
    _check(x.is_cuda, "x must be a CUDA tensor")
    _check(group in W4_GROUPS, "group must be 32, 64 or 128")
    _check(w13.dim() == 3 and w13.shape[1] % 2 == 0, "w13 must be [E, 2 I, ceil(H / 2)]")
    (T, H), dev = x.shape, x.device
    E, I = w13.shape[0], w13.shape[1] // 2
    _check(1 <= E <= MAX_EXPERTS and H >= 1 and I >= 1, f"w13 must hold 1 to {MAX_EXPERTS} experts")
    _check(T <= MAX_TOKENS, f"x must have at most {MAX_TOKENS} tokens")
    _check(T == 0 or H == 1 or x.stride(1) == 1, "x must have neighbouring columns in memory (stride 1)")
    _check(idx.dim() == 2 and idx.shape[0] == T and 1 <= idx.shape[1] <= MAX_TOP_K and idx.dtype == torch.int32
           and idx.is_contiguous() and idx.device == dev,
           f"idx must be a contiguous int32 [T, top_k] tensor on x's device, top_k 1 to {MAX_TOP_K}")
    _check(weights.shape == idx.shape and weights.dtype == torch.float32 and weights.is_contiguous()
           and weights.device == dev, "weights must be a contiguous float32 [T, top_k] tensor on x's device")
    _w4(w13, w13_scale, w13_zero, group, (E,), 2 * I, H, x.dtype, dev, "w13")
    _w4(w2, w2_scale, w2_zero, group, (E,), H, I, x.dtype, dev, "w2")
    if out is None:
        out = torch.empty((T, H), dtype=x.dtype, device=dev)
    else:
        _check(out.dtype == x.dtype and out.shape == (T, H) and out.is_contiguous() and out.device == dev,
               "out must be a contiguous [T, H] tensor of x's type on its device")
    if T == 0:
        return out
    lib, top_k = _native.cuda_lib(), idx.shape[1]
    need = int(lib.moe_experts_w4_workspace_bytes(T, top_k, E, H, I))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    else:
        _check(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == dev
               and workspace.numel() >= need, f"workspace must be a contiguous uint8 tensor of at least {need} bytes on x's device")
    _call(lib.moe_experts_w4, dev, x.data_ptr(), _DTYPE[x.dtype], x.stride(0), idx.data_ptr(), weights.data_ptr(),
          w13.data_ptr(), w13_scale.data_ptr(), None if w13_zero is None else w13_zero.data_ptr(), w2.data_ptr(),
          w2_scale.data_ptr(), None if w2_zero is None else w2_zero.data_ptr(), group, T, top_k, E, local_offset, H, I,
          out.data_ptr(), workspace.data_ptr(), workspace.numel())
    return out

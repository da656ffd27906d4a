"""
Experts in the head that reads the scattering coefficients: every row (node) goes through the k of E small MLPs that a
router picks for it.

    weights, experts = route_experts(logits, k)                      # (rows, E) -> (rows, k) fp32, (rows, k) int32
    y = expert_mlp(x, weights, experts, w1, b1, w2, b2)              # sum_j w_j (W2_e silu(W1_e x + b1_e) + b2_e)
    load = expert_counts(experts, E)                                 # rows per expert, for a balance bias

All three run on the current stream, read nothing back to the host, and give the same bits for the same inputs (no
floating-point atomics); they can be captured into a graph.  There is no CPU path.
"""
import math
from typing import Optional, Tuple
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .optim import DTYPE_CODES, _on

MAX_EXPERTS, MAX_K, MAX_GROUPS = 1024, 16, 64          # ESCAT_ROUTE_MAX_EXPERTS, ESCAT_ROUTE_MAX_K, groups a row's lanes hold
_SCORES = {"softmax": 0, "sigmoid": 1}


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _need_gpu(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise RuntimeError(f"escat: {name} must live on a GPU; the MI355X path has no CPU fallback")


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, k, score, groups, keep, group_top, renorm, scale):
        rows, E = logits.shape
        logits = logits.contiguous()
        weights = torch.empty(rows, k, dtype=torch.float32, device=logits.device)
        experts = torch.empty(rows, k, dtype=torch.int32, device=logits.device)
        with _on(logits.device) as stream:
            rc = _lib.load().escat_route(logits.data_ptr(), DTYPE_CODES[logits.dtype], rows, E, k, score, _ptr(bias), groups, keep,
                                         group_top, renorm, scale, weights.data_ptr(), experts.data_ptr(), stream)
        _lib.check(rc, "escat_route")
        ctx.mark_non_differentiable(experts)
        ctx.save_for_backward(logits, weights, experts)
        ctx.meta = (k, score, renorm, scale)
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        logits, weights, experts = ctx.saved_tensors
        k, score, renorm, scale = ctx.meta
        rows, E = logits.shape
        dweights = dweights.to(torch.float32).contiguous()
        dlogits = torch.empty_like(logits)
        with _on(logits.device) as stream:
            rc = _lib.load().escat_route_bwd(logits.data_ptr(), DTYPE_CODES[logits.dtype], rows, E, k, score, renorm, scale, weights.data_ptr(),
                                             experts.data_ptr(), dweights.data_ptr(), dlogits.data_ptr(), stream)
        _lib.check(rc, "escat_route_bwd")
        return dlogits, None, None, None, None, None, None, None, None


def route_experts(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
                  keep_groups: Optional[int] = None, group_top: int = 2, renormalize: bool = True,
                  scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    The k experts of every row and their weights.

    logits (rows, E), fp32 / bf16 / fp16; scores s = softmax or sigmoid of a row.  Experts are chosen by s + bias (bias: (E,)
    fp32, for balance; it takes no part in the weights and gets no gradient), without a bias in the order of the logits.
    With groups > 1 (E divided into that many equal runs) only experts of the keep_groups best groups can be chosen; a group
    counts by the sum of its group_top (1 or 2) largest keys.  Ties go to the lowest index; the order is decided in 64 bits.
    weights (rows, k) fp32 = scale * s_j / sum over the chosen (renormalize), or scale * s_j; experts (rows, k) int32.

    A logit or a bias of -inf masks an expert; where fewer than k can be chosen the rest is expert -1 with weight 0.  A NaN
    counts as the largest and shows in the row's weights.  At most 1024 experts, k <= 16, 64 groups.
    """
    if logits.dim() != 2 or logits.dtype not in DTYPE_CODES:
        raise ValueError(f"escat: logits must be (rows, E) in fp32, bf16 or fp16: {tuple(logits.shape)} {logits.dtype}")
    E = logits.shape[1]
    if score not in _SCORES:
        raise ValueError(f"escat: score must be 'softmax' or 'sigmoid': {score!r}")
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= min(E, MAX_K):
        raise ValueError(f"escat: E = {E} (1..{MAX_EXPERTS}), k = {k} (1..min(E, {MAX_K}))")
    if not 1 <= groups <= MAX_GROUPS or E % groups:
        raise ValueError(f"escat: groups = {groups} must divide E = {E} and be at most {MAX_GROUPS}")
    keep = groups if keep_groups is None else keep_groups
    if not 1 <= keep <= groups or group_top not in (1, 2):
        raise ValueError(f"escat: keep_groups = {keep} (1..{groups}), group_top = {group_top} (1 or 2)")
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"escat: scale must be positive: {scale}")
    if bias is not None and (bias.shape != (E,) or bias.dtype is not torch.float32 or bias.device != logits.device):
        raise ValueError(f"escat: bias must be ({E},) fp32 on {logits.device}: {tuple(bias.shape)} {bias.dtype} {bias.device}")
    _need_gpu(logits, "logits")
    return _Route.apply(logits, None if bias is None else bias.detach().contiguous(), k, _SCORES[score], groups, keep, group_top,
                        int(bool(renormalize)), float(scale))

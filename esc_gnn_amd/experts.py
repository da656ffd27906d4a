"""
Experts in the head that reads the scattering coefficients: every row (node) goes through the k of E small MLPs that a
router picks for it.

    weights, experts = route_experts(logits, k)                      # (rows, E) -> (rows, k) fp32, (rows, k) int32
    y = expert_mlp(x, weights, experts, w1, b1, w2, b2)              # sum_j w_j (W2_e silu(W1_e x + b1_e) + b2_e)
    load = expert_counts(experts, E)                                 # rows per expert, for a balance bias

All three run on the current stream, read nothing back to the host, and give the same bits for the same inputs (no
floating-point atomics); they can be captured into a graph.  There is no CPU path, and no forward-mode differentiation (an error).
"""
import ctypes
import functools
import math
from typing import Optional, Tuple
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.nn.functional import pad

from . import _lib
from .optim import DTYPE_CODES, _on

MAX_EXPERTS, MAX_K, MAX_GROUPS = 1024, 16, 64          # ESCAT_ROUTE_MAX_EXPERTS, ESCAT_ROUTE_MAX_K, groups a row's lanes hold
_SCORES = {"softmax": 0, "sigmoid": 1}


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _need_gpu(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise RuntimeError(f"escat: {name} must live on a GPU; the MI355X path has no CPU fallback")


def _wants_grad(ts) -> bool:
    """whether a call goes by its autograd function: for a gradient, or to be refused where a tensor has a forward-mode tangent"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


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
        ctx.set_materialize_grads(False)                  # (no zeros in the place of the experts' gradient)
        ctx.save_for_backward(logits, weights, experts)
        ctx.meta = (k, score, renorm, scale)
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        if dweights is None:
            return (None,) * 9
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
    if not 0.0 < ctypes.c_float(float(scale)).value < math.inf:                  # (the kernels' type)
        raise ValueError(f"escat: scale must be a positive fp32 number: {scale}")
    if bias is not None and (bias.shape != (E,) or bias.dtype is not torch.float32 or bias.device != logits.device):
        raise ValueError(f"escat: bias must be ({E},) fp32 on {logits.device}: {tuple(bias.shape)} {bias.dtype} {bias.device}")
    _need_gpu(logits, "logits")
    return _Route.apply(logits, None if bias is None else bias.detach().contiguous(), k, _SCORES[score], groups, keep, group_top,
                        int(bool(renormalize)), float(scale))


def _plan(experts: torch.Tensor, rows: int, k: int, E: int, counts: Optional[torch.Tensor], stream) -> torch.Tensor:
    lib = _lib.load()
    size = lib.escat_experts_plan_bytes(rows, k, E)
    plan = torch.empty(size, dtype=torch.uint8, device=experts.device)
    _lib.check(lib.escat_experts_plan(experts.data_ptr(), rows, k, E, plan.data_ptr(), size, _ptr(counts), stream), "escat_experts_plan")
    return plan


def _check_experts(experts: torch.Tensor, E: int):
    if experts.dtype is not torch.int32:
        raise ValueError(f"escat: experts must be int32: {experts.dtype}")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"escat: E = {E} (1..{MAX_EXPERTS})")
    if experts.numel() >= 1 << 30:
        raise ValueError(f"escat: {experts.numel()} (row, slot) pairs: fewer than 2^30 are supported")


def expert_counts(experts: torch.Tensor, n_experts: int) -> torch.Tensor:
    """(n_experts,) int32: how many (row, slot) pairs go to each expert; entries outside [0, n_experts) are left out"""
    _check_experts(experts, n_experts)
    _need_gpu(experts, "experts")
    counts = torch.empty(n_experts, dtype=torch.int32, device=experts.device)
    with _on(experts.device) as stream:
        _plan(experts.contiguous(), experts.numel(), 1, n_experts, counts, stream)
    return counts


@functools.lru_cache(maxsize=256)
def _sizes(*dims):
    """what the library says of a call's sizes: the dims structure, whether the forward sorts, the forward's workspace"""
    lib = _lib.load()
    d = _lib.EscatExpertsDims(*dims)
    at = ctypes.addressof(d)
    return d, at, bool(lib.escat_experts_fwd_needs_plan(at)), lib.escat_experts_workspace_bytes(at, 0, 0)


def _mlp_forward(x, weights, experts, w1, b1, w2, b2, keep=False):
    """y; the plan and (keep) the hidden rows where the forward made them (few rows do without)"""
    lib = _lib.load()
    (rows, d), k, (E, h, _), o = x.shape, experts.shape[1], w1.shape, w2.shape[1]
    dims, at, sorts, size = _sizes(rows, DTYPE_CODES[x.dtype], d, h, o, E, k)
    y, hidden = x.new_empty((rows, o)), None
    with _on(x.device) as stream:
        plan = _plan(experts, rows, k, E, None, stream) if sorts else None
        if keep and sorts:
            hidden = torch.empty(lib.escat_experts_hidden_bytes(at), dtype=torch.uint8, device=x.device)
            size = lib.escat_experts_workspace_bytes(at, 0, 1)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        rc = lib.escat_experts_fwd(at, x.data_ptr(), weights.data_ptr(), experts.data_ptr(), w1.data_ptr(), _ptr(b1), w2.data_ptr(), _ptr(b2),
                                   _ptr(plan), y.data_ptr(), _ptr(hidden), ws.data_ptr(), size, stream)
    _lib.check(rc, "escat_experts_fwd")
    return y, plan, hidden, dims


class _ExpertMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, experts, w1, b1, w2, b2):
        y, plan, hidden, ctx.dims = _mlp_forward(x, weights, experts, w1, b1, w2, b2, keep=True)
        ctx.save_for_backward(x, weights, experts, w1, b1, w2, b2, plan, hidden)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        lib = _lib.load()
        x, weights, experts, w1, b1, w2, b2, plan, hidden = ctx.saved_tensors
        dims = ctx.dims
        at = ctypes.addressof(dims)
        dy = dy.contiguous()
        need = ctx.needs_input_grad
        new = lambda t, n: torch.empty_like(t) if t is not None and n else None                  # noqa: E731
        dx, dweights = new(x, need[0]), new(weights, need[1])
        db1, db2 = new(b1, need[4]), new(b2, need[6])
        dw1, dw2 = new(w1, need[3] or need[4]), new(w2, need[5] or need[6])
        size = lib.escat_experts_workspace_bytes(at, 1, int(hidden is not None))
        with _on(x.device) as stream:
            if plan is None:
                plan = _plan(experts, dims.rows, dims.k, dims.experts, None, stream)
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
            rc = lib.escat_experts_bwd(at, x.data_ptr(), weights.data_ptr(), w1.data_ptr(), _ptr(b1), w2.data_ptr(), _ptr(b2), plan.data_ptr(),
                                       _ptr(hidden), dy.data_ptr(), _ptr(dx), _ptr(dweights), _ptr(dw1), _ptr(db1), _ptr(dw2), _ptr(db2), ws.data_ptr(), size,
                                       stream)
        _lib.check(rc, "escat_experts_bwd")
        return dx, dweights, None, dw1 if need[3] else None, db1, dw2 if need[5] else None, db2


def expert_mlp(x: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor, w1: torch.Tensor, b1: Optional[torch.Tensor],
               w2: torch.Tensor, b2: Optional[torch.Tensor]) -> torch.Tensor:
    """
    y_t = sum_j weights[t, j] (W2_e silu(W1_e x_t + b1_e) + b2_e) with e = experts[t, j]; gradients for all but `experts`.

    x (rows, d), w1 (E, h, d), b1 (E, h) or None, w2 (E, o, h), b2 (E, o) or None: one type, fp32, bf16 or fp16 (under autocast
    they are cast to its type); weights (rows, k) fp32, experts (rows, k) int32 as route_experts gives them.  A pair whose
    expert lies outside [0, E) counts for nothing and gets no gradient; the same expert may come twice in a row.  Sums are
    fp32; with 16-bit types the weighted hidden rows and their gradients are rounded to the type in between.  The backward
    sees the hidden rows unrounded.  A forward that gradients are wanted of keeps rows * k * h elements of its type, and with d > 64 (16-bit types: d > 640)
    as many in fp32, next to its arguments and the sorted pairs.  For a few rows the forward
    is a pair of matrix-vector kernels that read the weights in use once a pair, without sorting.  Weights must be
    contiguous; d, h, o are free (any alignment), k <= 64, E <= 1024, rows * k < 2^30, and a product has fewer than 2^24 tiles of 128 x 128
    (EscatError otherwise).
    """
    if torch.is_autocast_enabled("cuda") and x.is_cuda:
        t = torch.get_autocast_dtype("cuda")
        x, w1, w2 = x.to(t), w1.to(t), w2.to(t)
        b1, b2 = None if b1 is None else b1.to(t), None if b2 is None else b2.to(t)
    if x.dim() != 2 or w1.dim() != 3 or w2.dim() != 3 or x.dtype not in DTYPE_CODES:
        raise ValueError(f"escat: x (rows, d), w1 (E, h, d), w2 (E, o, h) in fp32, bf16 or fp16: {tuple(x.shape)} {x.dtype}, {tuple(w1.shape)}, {tuple(w2.shape)}")
    (rows, d), (E, h, d1), (E2, o, h2) = x.shape, w1.shape, w2.shape
    if d != d1 or h != h2 or E != E2 or min(d, h, o) < 1 or max(d, h, o) > 65536:
        raise ValueError(f"escat: x {tuple(x.shape)}, w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)} do not fit each other")
    if weights.dim() != 2 or weights.shape[0] != rows or experts.shape != weights.shape or not 1 <= weights.shape[1] <= 64 or weights.dtype is not torch.float32:
        raise ValueError(f"escat: weights and experts must be ({rows}, k), k <= 64, weights fp32: {tuple(weights.shape)} {weights.dtype}, {tuple(experts.shape)}")
    _check_experts(experts, E)
    dtype, at = x.dtype, x.get_device()
    for name, t, shape in (("w1", w1, None), ("w2", w2, None), ("b1", b1, (E, h)), ("b2", b2, (E, o))):
        if t is None:
            continue
        if (shape is not None and t.shape != shape) or t.dtype is not dtype:
            raise ValueError(f"escat: {name} must be {shape or tuple(t.shape)} {dtype}: {tuple(t.shape)} {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"escat: {name} must be contiguous (strides {t.stride()})")
        if t.get_device() != at:
            raise RuntimeError(f"escat: {name} lives on {t.device}, x on {x.device}")
    if weights.get_device() != at or experts.get_device() != at:
        raise RuntimeError(f"escat: weights and experts live on {weights.device} and {experts.device}, x on {x.device}")
    _need_gpu(x, "x")
    least = 4 if x.dtype is torch.float32 else 8            # the kernels move 16 bytes of a row at once: narrower ones get zeros
    if min(d, h, o) < least:
        more = lambda n: max(0, least - n)                                                       # noqa: E731
        x = pad(x, (0, more(d)))
        w1, w2 = pad(w1, (0, more(d), 0, more(h))), pad(w2, (0, more(h), 0, more(o)))
        b1, b2 = None if b1 is None else pad(b1, (0, more(h))), None if b2 is None else pad(b2, (0, more(o)))
    args = (x.contiguous(), weights.contiguous(), experts.contiguous(), w1, b1, w2, b2)
    y = _ExpertMLP.apply(*args) if _wants_grad(args) else _mlp_forward(*args)[0]
    return y if o >= least else y[:, :o].contiguous()

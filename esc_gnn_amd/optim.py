"""
AdamW over many tensors at once, states in 32 or in 8 bits, with the clip by the global gradient norm in the same call
(the reference: torch's AdamW, training/prep_optimizer.py:9, after clip_grad_norm_, training/train.py:411-415).

    opt = AdamW(model.parameters(), lr=1e-3, state_bits=8, max_grad_norm=1.0)      # a torch.optim.Optimizer
    adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=...)                 # the same on plain tensors

A step of up to 56 tensors of one type is three launches with clipping and two without (csrc/escat_adamw.hip): the squares, the
count with the scalars, the update.  Squares and update are one each per 56 tensors and type (the update: per group of settings
too), and parameters that count their steps apart (some paused) make a call each.  The step count lives on the GPU: a captured step
counts on when it is replayed (lr and the other hyperparameters are constants of the captured graph).  The same inputs give the same bits.

8-bit states hold one byte per element and moment and one fp32 scale per 256 elements: 2.03 bytes a parameter instead of
8.  They are rounded stochastically, by bits that depend on (seed, step, tensor, element) only, so ranks that average
their gradients keep identical parameters.  An element whose state is not finite is held as NaN.
"""
import array
import ctypes
from itertools import chain
from operator import attrgetter
from typing import Optional, Sequence
import torch

from . import _lib
from .pyg_utilities import _ptr

STATE_BLOCK = 256
MAX_GROUPS = 16                                            # ESCAT_ADAMW_MAX_GROUPS
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


_DTYPE, _LAYOUT, _SHAPE = map(attrgetter, ("dtype", "layout", "shape"))
_NUMEL, _DEVICE, _CONTIGUOUS, _PTR = torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous, torch.Tensor.data_ptr


class _Group(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay")]


class _on:
    """`with _on(device) as stream`: the device is current and `stream` its current stream's handle.  (torch.cuda.device and
    torch.cuda.current_stream cost some 5 us a call: as much as a small launch.)"""
    __slots__ = ("index", "before")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch._C._cuda_exchangeDevice(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *_):
        if self.before != self.index:
            torch._C._cuda_maybeExchangeDevice(self.before)


def new_state8(n: int, device) -> tuple:
    """(codes, scales) of a zero 8-bit state for a tensor of n elements"""
    return (torch.zeros(n, dtype=torch.uint8, device=device),
            torch.zeros(-(-n // STATE_BLOCK), dtype=torch.float32, device=device))


def dequantize_state(codes: torch.Tensor, scales: torch.Tensor, signed: bool) -> torch.Tensor:
    """the fp32 values of an 8-bit state, in the shape of the codes; signed: a first moment (exp_avg), else a second moment (exp_avg_sq)"""
    if codes.dtype != torch.uint8 or scales.dtype != torch.float32 or not codes.is_contiguous() or not scales.is_contiguous() \
            or scales.numel() != -(-codes.numel() // STATE_BLOCK):
        raise ValueError("escat: an 8-bit state is contiguous uint8 codes with one fp32 scale per 256 elements")
    if not codes.is_cuda or scales.device != codes.device:
        raise RuntimeError("escat: the state must live on one GPU; the MI355X path has no CPU fallback")
    out = torch.empty_like(codes, dtype=torch.float32)
    with _on(codes.device) as stream:
        rc = _lib.load().escat_state8_values(codes.data_ptr(), scales.data_ptr(), codes.numel(), int(bool(signed)), out.data_ptr(), stream)
    _lib.check(rc, "escat_state8_values")
    return out


def _check_hyper(lr, betas, eps, weight_decay):
    for name, v in (("lr", lr), ("eps", eps), ("weight_decay", weight_decay), ("beta1", betas[0]), ("beta2", betas[1])):
        if isinstance(v, torch.Tensor):
            raise TypeError(f"escat: {name} must be a number, not a tensor")
    if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
        raise ValueError(f"escat: lr, eps and weight_decay must not be negative: {lr}, {eps}, {weight_decay}")
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"escat: betas must lie in [0, 1): {betas}")


class _Tables:
    """tensors of one call sorted by (parameter type, gradient type, state bits), as the library's host table"""

    def __init__(self):
        self.by_type = {}
        self.keep = []                                     # contiguous copies of gradients: alive until the launches are queued

    def add(self, p, g, m, v, ordinal, dev):
        n = p.numel()
        if p.dtype not in DTYPE_CODES or (g.dtype is not p.dtype and g.dtype is not torch.float32):
            raise TypeError(f"escat: parameters are fp32, bf16 or fp16 and gradients of the same type or fp32; tensor {ordinal} has {p.dtype} and {g.dtype}")
        if p.device != dev or g.device != dev:
            raise RuntimeError(f"escat: tensor {ordinal} lives on {p.device} / {g.device}, the step runs on {dev} (one GPU; there is no CPU fallback)")
        if g.layout is not torch.strided or g.numel() != n or g.shape != p.shape:
            raise ValueError(f"escat: the gradient of tensor {ordinal} must be dense and of shape {tuple(p.shape)}")
        if not p.is_contiguous():
            raise ValueError(f"escat: parameter {ordinal} must be contiguous (shape {tuple(p.shape)}, strides {p.stride()})")
        if not g.is_contiguous():
            g = g.contiguous()
            self.keep.append(g)
        if type(m) is tuple or type(v) is tuple:
            if type(m) is not tuple or type(v) is not tuple or len(m) != 2 or len(v) != 2:
                raise ValueError(f"escat: the states of tensor {ordinal} must both be tensors or both (codes, scales) pairs")
            nb = -(-n // STATE_BLOCK)
            for c, s in (m, v):
                if c.dtype is not torch.uint8 or s.dtype is not torch.float32 or c.numel() != n or s.numel() != nb \
                        or not c.is_contiguous() or not s.is_contiguous() or c.device != dev or s.device != dev:
                    raise ValueError(f"escat: an 8-bit state of tensor {ordinal} is {n} contiguous uint8 codes and {nb} fp32 scales on {dev}")
            bits, row = 8, (p.data_ptr(), g.data_ptr(), m[0].data_ptr(), v[0].data_ptr(), m[1].data_ptr(), v[1].data_ptr(), n, ordinal)
        else:
            for s in (m, v):
                if s.dtype is not torch.float32 or s.numel() != n or not s.is_contiguous() or s.device != dev:
                    raise ValueError(f"escat: the states of tensor {ordinal} must be contiguous fp32 tensors of {n} elements on {dev}")
            bits, row = 32, (p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), 0, 0, n, ordinal)
        if n:
            key = (DTYPE_CODES[p.dtype], DTYPE_CODES[g.dtype], bits)
            t = self.by_type.get(key)
            if t is None:
                t = self.by_type[key] = array.array("Q")
            t.extend(row)

    def add_all(self, ps, gs, ms, vs, dev):
        """add() for whole lists that are all alike (one parameter type, one gradient type, contiguous, no empty tensor), checked
        a property at a time: a third of the time per tensor.  False: they are not, nothing was added."""
        n = len(ps)
        if n == 0 or len(set(map(_DTYPE, ps))) != 1 or len(set(map(_DTYPE, gs))) != 1:
            return False
        pt, gt = ps[0].dtype, gs[0].dtype
        if pt not in DTYPE_CODES or (gt is not pt and gt is not torch.float32):
            return False
        bits = 8 if type(ms[0]) is tuple else 32
        if bits == 8:
            if set(map(type, ms)) != {tuple} or set(map(type, vs)) != {tuple} or set(map(len, ms)) != {2} or set(map(len, vs)) != {2}:
                return False
            (ms, mz), (vs, vz) = zip(*ms), zip(*vs)
            scales = mz + vz
        elif tuple in map(type, ms) or tuple in map(type, vs):
            return False
        else:
            scales = ()
        states = [*ms, *vs]
        ns = list(map(_NUMEL, ps))
        if set(map(_LAYOUT, gs)) != {torch.strided} or set(map(_DEVICE, [*ps, *gs, *states, *scales])) != {dev.index} \
                or set(map(_DTYPE, states)) != {torch.uint8 if bits == 8 else torch.float32} or (scales and set(map(_DTYPE, scales)) != {torch.float32}) \
                or not all(map(_CONTIGUOUS, [*ps, *gs, *states, *scales])) or 0 in ns or list(map(_SHAPE, ps)) != list(map(_SHAPE, gs)) \
                or list(map(_NUMEL, states)) != ns * 2 or (scales and list(map(_NUMEL, scales)) != [-(-k // STATE_BLOCK) for k in ns] * 2):
            return False
        z = list(map(_PTR, scales)) or [0] * (2 * n)
        q = list(map(_PTR, states))
        rows = zip(map(_PTR, ps), map(_PTR, gs), q, q[n:], z, z[n:], ns, range(n))
        self.by_type[(DTYPE_CODES[pt], DTYPE_CODES[gt], bits)] = array.array("Q", chain.from_iterable(rows))
        return True

    def clashes(self, count):
        """whether the step would write a tensor twice (`count`: its address is the step count's) or one that it reads as a gradient"""
        written, read = [count], set()
        for (_, _, bits), t in self.by_type.items():
            for at in (0, 2, 3, 4, 5) if bits == 8 else (0, 2, 3):
                written += t[at::8]
            read.update(t[1::8])
        once = set(written)
        return len(once) != len(written) or not read.isdisjoint(once)


def _begin(lib, tables, max_norm, groups, step, ws, norm, stream):
    """one call per gradient type (the squares), the last of them counts the step; `tables`: all that share the norm"""
    by_grad = {}
    if max_norm:
        for t in tables:
            for (_, gt, _), rows in t.by_type.items():
                by_grad.setdefault(gt, array.array("Q")).extend(rows)
    arr = (_Group * len(groups))(*groups)
    work = list(by_grad.items()) or [(0, array.array("Q"))]
    slot = 0
    for i, (gt, rows) in enumerate(work):
        slot = lib.escat_adamw_begin(rows.buffer_info()[0], len(rows) // 8, gt, max_norm, slot, int(i == len(work) - 1), arr, len(groups),
                                     _ptr(step), _ptr(norm), _ptr(ws), ws.numel(), stream)
        _lib.check(min(slot, 0), "escat_adamw_begin")


def _update(lib, table, group, index, seed, step, ws, stream):
    for (pt, gt, bits), rows in table.by_type.items():
        rc = lib.escat_adamw_update(rows.buffer_info()[0], len(rows) // 8, pt, gt, bits, ctypes.byref(group), index, seed, _ptr(step), _ptr(ws), stream)
        _lib.check(rc, "escat_adamw_update")


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence, exp_avg_sqs: Sequence,
               step: torch.Tensor, *, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               max_grad_norm: Optional[float] = None, seed: int = 0) -> Optional[torch.Tensor]:
    """
    One AdamW step in place.  params: fp32 / bf16 / fp16, contiguous; grads: the same type or fp32; exp_avgs / exp_avg_sqs:
    fp32 tensors, or (codes, scales) pairs (new_state8); step: int32 tensor of one element on the same GPU, the number of
    steps done, counted here.  With max_grad_norm the gradients count as scaled by min(1, max_grad_norm / (norm + 1e-6)),
    norm over all of them (they are left as they are), and the norm is returned (fp32, on the GPU).
    """
    n = len(params)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n):
        raise ValueError("escat: params, grads, exp_avgs and exp_avg_sqs must have one entry per tensor")
    _check_hyper(lr, betas, eps, weight_decay)
    if max_grad_norm is not None and not max_grad_norm > 0.0:
        raise ValueError(f"escat: max_grad_norm must be positive: {max_grad_norm}")
    if step.dtype is not torch.int32 or step.numel() != 1:
        raise ValueError("escat: step is an int32 tensor of one element")
    dev = step.device
    table = _Tables()
    if dev.type != "cuda" or not table.add_all(params, grads, exp_avgs, exp_avg_sqs, dev):
        for i in range(n):
            table.add(params[i], grads[i], exp_avgs[i], exp_avg_sqs[i], i, dev)
    if table.clashes(step.data_ptr()):
        raise ValueError("escat: a parameter, state or count is listed twice, or as a gradient")
    if dev.type != "cuda":
        raise RuntimeError("escat: tensors must live on a GPU; the MI355X path has no CPU fallback")
    lib = _lib.load()
    norm = None if max_grad_norm is None else torch.empty((), dtype=torch.float32, device=dev)
    group = _Group(lr, betas[0], betas[1], eps, weight_decay)
    with _on(dev) as stream:
        ws = torch.empty(lib.escat_adamw_workspace_bytes(n), dtype=torch.uint8, device=dev)
        _begin(lib, [table], float(max_grad_norm or 0.0), [group], step, ws, norm, stream)
        _update(lib, table, group, 0, int(seed) & 0xFFFFFFFF, step, ws, stream)
    torch._C._increment_version(params)                    # a backward that saved one of them shall say so, as after torch's own step
    return norm


class AdamW(torch.optim.Optimizer):
    """
    torch.optim.AdamW's step on the kernels above.  state_bits: 32 or 8 (states); max_grad_norm: clip by the global norm of
    all gradients, `grad_norm` then holds the last step's (on the GPU); seed: of the 8-bit states' rounding.  These three are
    the constructor's: a copy or pickle has them, a state dict (states and groups, as torch's) does not.  Parameter
    groups may differ in lr, betas, eps and weight_decay.  A parameter without a gradient is left alone and does not count
    the step; parameters live on one GPU.  A step that is captured finds its states there: take one with the same gradients
    present before the capture (RuntimeError otherwise).
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, max_grad_norm: Optional[float] = None, seed: int = 0):
        _check_hyper(lr, betas, eps, weight_decay)
        if state_bits not in (32, 8):
            raise ValueError(f"escat: state_bits must be 32 or 8: {state_bits}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"escat: max_grad_norm must be positive: {max_grad_norm}")
        self.state_bits, self.max_grad_norm, self.seed, self.grad_norm = state_bits, max_grad_norm, int(seed), None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        """what a copy or a pickle takes along: the base class names its own attributes alone"""
        return {**super().__getstate__(), **{n: getattr(self, n) for n in ("state_bits", "max_grad_norm", "seed", "grad_norm")}}

    def _state_of(self, p, fresh):
        """a parameter's state; `fresh`: the step count that the parameters which begin in this step share"""
        st = self.state[p]
        if not st:
            st["step"] = fresh()
            for name in ("exp_avg", "exp_avg_sq"):
                if self.state_bits == 8:
                    st[name + "_codes"], st[name + "_scales"] = new_state8(p.numel(), p.device)
                else:
                    st[name] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
        return st

    @staticmethod
    def _not_in_a_capture(dev):
        with torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("escat: this step makes states or step counts, which a capture would make anew at every replay: take one such step before it")

    def _moments(self, st):
        if self.state_bits == 8:
            return ((st["exp_avg_codes"], st["exp_avg_scales"]), (st["exp_avg_sq_codes"], st["exp_avg_sq_scales"]))
        return st["exp_avg"], st["exp_avg_sq"]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        made = []

        def fresh():
            if not made:
                self._not_in_a_capture(dev)
                made.append(torch.zeros(1, dtype=torch.int32, device=dev))
            return made[0]

        dev, ordinal, calls, seen = None, 0, {}, {}
        for gi, group in enumerate(self.param_groups):
            _check_hyper(group["lr"], group["betas"], group["eps"], group["weight_decay"])
            for p in group["params"]:
                ordinal += 1
                if p.grad is None:
                    if p in self.state and self.state[p]:
                        seen.setdefault(id(self.state[p]["step"]), [None, []])[0] = True          # stays behind
                    continue
                if dev is None:
                    dev = p.device
                    if dev.type != "cuda":
                        raise RuntimeError("escat: parameters must live on a GPU; the MI355X path has no CPU fallback")
                st = self._state_of(p, fresh)
                seen.setdefault(id(st["step"]), [None, []])[1].append(p)
                calls.setdefault((id(st["step"]), gi), []).append((p, st, ordinal - 1))
        if dev is None:
            return loss
        # a step count is shared by the parameters that took every step together; where some stay behind, the others get their own
        moved = {}
        for key, (behind, ps) in seen.items():
            if ps:
                count = self.state[ps[0]]["step"]
                if count.dtype is not torch.int32 or count.numel() != 1 or count.device != dev:
                    raise ValueError(f"escat: step must be an int32 tensor of one element on {dev}: {count.dtype}, {tuple(count.shape)} on {count.device}")
            if behind and ps:
                self._not_in_a_capture(dev)
                own = self.state[ps[0]]["step"].clone()
                for p in ps:
                    self.state[p]["step"] = own
            if ps:
                moved[key] = self.state[ps[0]]["step"]
        lib = _lib.load()
        tables, groups, steps = {}, {}, {}
        for (key, gi), items in calls.items():
            t = tables[(key, gi)] = _Tables()
            moments = [self._moments(st) for _, st, _ in items]
            if [at for _, _, at in items] != list(range(len(items))) or not t.add_all(
                    [p for p, _, _ in items], [p.grad for p, _, _ in items], [m for m, _ in moments], [v for _, v in moments], dev):
                for (p, st, at), (m, v) in zip(items, moments):
                    t.add(p, p.grad, m, v, at, dev)
            g = self.param_groups[gi]
            groups.setdefault(key, []).append((gi, _Group(g["lr"], g["betas"][0], g["betas"][1], g["eps"], g["weight_decay"])))
            steps[key] = moved[key]
        n = sum(len(x) for x in calls.values())
        max_norm = float(self.max_grad_norm or 0.0)
        seed = self.seed & 0xFFFFFFFF
        with _on(dev) as stream:
            norm = torch.empty((), dtype=torch.float32, device=dev) if max_norm else None
            for key, gs in groups.items():
                for at in range(0, len(gs), MAX_GROUPS):
                    part = gs[at:at + MAX_GROUPS]
                    ws = torch.empty(lib.escat_adamw_workspace_bytes(n), dtype=torch.uint8, device=dev)
                    # more than MAX_GROUPS groups: the first part counts the step, the others read a copy that lags by it
                    step = steps[key] if at == 0 else steps[key] - 1
                    _begin(lib, list(tables.values()), max_norm, [g for _, g in part], step, ws, norm, stream)
                    for i, (gi, g) in enumerate(part):
                        _update(lib, tables[(key, gi)], g, i, seed, step, ws, stream)
        torch._C._increment_version([p for items in calls.values() for p, _, _ in items])
        self.grad_norm = norm
        return loss

    def state_dict(self):
        """As torch's: the moments themselves, and for each parameter a count of its own as torch keeps it, an fp32 number on the CPU (beyond
        2^24 steps fp64).  In the optimizer those that took every step together share one, on the GPU: this call waits for it."""
        out = super().state_dict()
        seen = {}

        def count(t):
            if id(t) not in seen:
                seen[id(t)] = int(t)
            k = seen[id(t)]
            return torch.tensor(float(k), dtype=torch.float32 if k <= 1 << 24 else torch.float64)
        out["state"] = {i: {n: count(t) if n == "step" else t for n, t in st.items()} for i, st in out["state"].items()}
        return out

    def load_state_dict(self, state_dict):
        """A state dict of this class, or of torch.optim.AdamW: the count becomes int32, moments that torch held in a 16-bit type fp32,
        both with the values they had.  States of another step (amsgrad, maximize, decay inside the gradient) are refused."""
        saved, groups = state_dict["state"], state_dict["param_groups"]
        for g in groups:
            if g.get("amsgrad") or g.get("maximize") or (g.get("weight_decay") and not g.get("decoupled_weight_decay", True)):
                raise ValueError("escat: the loaded states are of another step: amsgrad, maximize and coupled weight decay are not served")
        names = {"step"} | ({n + e for n in ("exp_avg", "exp_avg_sq") for e in ("_codes", "_scales")} if self.state_bits == 8 else {"exp_avg", "exp_avg_sq"})
        ids = [i for g in groups for i in g["params"]]
        counts = {}
        for i, p in zip(ids, [p for g in self.param_groups for p in g["params"]]):
            st = saved.get(i)
            if not st:
                continue
            if set(st) != names:
                raise ValueError(f"escat: a state with {self.state_bits} bits holds {sorted(names)}, the loaded one {sorted(st)}")
            step = torch.as_tensor(st["step"])
            t = float(step) if step.numel() == 1 else -1.0
            if not (0 <= t < 2 ** 31 and t == int(t)):
                raise ValueError(f"escat: step must be a whole number of steps: {st['step']}")
            counts[i] = int(t)
            for name in names - {"step"}:
                n = -(-p.numel() // STATE_BLOCK) if name.endswith("_scales") else p.numel()
                if st[name].numel() != n or not (st[name].dtype is torch.uint8 if name.endswith("_codes") else st[name].is_floating_point()):
                    raise ValueError(f"escat: {name} of a parameter of shape {tuple(p.shape)} has {st[name].numel()} elements of {st[name].dtype}")
        super().load_state_dict(state_dict)
        # the base class casts states to the parameter's type: take them as they were saved instead
        shared = {}
        for i, p in zip(ids, [p for g in self.param_groups for p in g["params"]]):
            if i in counts:
                st = self.state[p] = {}
                for name in saved[i]:
                    if name == "step":
                        if counts[i] not in shared:
                            shared[counts[i]] = torch.full((1,), counts[i], dtype=torch.int32, device=p.device)
                        st[name] = shared[counts[i]]
                    else:
                        dtype = torch.uint8 if name.endswith("_codes") else torch.float32
                        st[name] = saved[i][name].detach().to(device=p.device, dtype=dtype, copy=True).contiguous()

"""
GPU tests of AdamW where eps does not hide the root of the second moment (esc_gnn_amd/optim.py, csrc/escat_adamw.hip), against the formulas
in 64 bits.  u = 2^-24: an update errs by 18 u of itself as counted in test_gpu_optim.py.  v below 2^-126 has steps of 2^-149: each of its
<= 3 roundings errs by half of one, and the root by half of their share of v.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("eps", [0.0, 1e-25, 1e-19, 1e-17, 1e-13, 1e-11, 1e-8])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.5, 0.0), (0.0, 0.999999)])
def test_first_step_of_small_gradients(bits, dtype, eps, betas):
    """8-bit states do not enter the first step's update"""
    from esc_gnn_amd import adamw_step, new_state8
    size = [1.0, 1e-9, 1e-12, 1e-15, 2e-17, 5e-18, 1e-18, 3e-19]
    g = torch.tensor(size, device=DEV).repeat_interleave(70)
    g[::2] = -g[::2]
    if dtype is torch.bfloat16:
        g = g.to(dtype)
    n = g.numel()
    p = torch.zeros(n, dtype=dtype, device=DEV)
    m, v = (new_state8(n, DEV), new_state8(n, DEV)) if bits == 8 else (torch.zeros(n, device=DEV), torch.zeros(n, device=DEV))
    adamw_step([p], [g], [m], [v], torch.zeros(1, dtype=torch.int32, device=DEV), lr=1e-2, betas=betas, eps=eps, weight_decay=0.0)
    g64 = g.double()
    v64 = (1 - betas[1]) * g64 * g64
    keep = v64 > 2.0 ** -140                                                        # (further below, v's steps are too coarse to ask anything)
    root = v64.sqrt() / (1 - betas[1]) ** 0.5
    want = -1e-2 * g64 / (root + eps)
    # (1 - b as an fp32 constant is what the kernel has: its rounding is among the 18)
    tol = (18 * U + 1.5 * 2.0 ** -149 / v64) * want.abs()
    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)
    assert int(keep.sum()) >= 70 * 4
    assert bool(((p.double() - want).abs() <= tol)[keep].all())


def test_several_steps_without_eps():
    """32-bit states, five steps of one small gradient: every update is lr (to 1e-4: v's steps of 2^-149 at 1e-39)"""
    from esc_gnn_amd import AdamW
    p = torch.nn.Parameter(torch.zeros(300, device=DEV))
    p.grad = torch.full_like(p, 1e-18)
    opt = AdamW([p], lr=1e-2, eps=0.0, weight_decay=0.0, max_grad_norm=1.0)
    for t in range(1, 6):
        opt.step()
        assert float((p.detach().double() + 1e-2 * t).abs().max()) <= 1e-6 * t

"""
GPU tests of what may never be chosen (esc_gnn_amd/experts.py, csrc/escat_route.hip): an expert whose bias is -inf stays out also where
scores are not numbers.  The choice has to be equal; weights within 64 u of the weight (u = 2^-24), counted in test_gpu_route.py.
"""
import math
import numpy as np
import pytest
import torch

from .test_gpu_route import plain

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"
SIZES = [(8, 2, 1, 1), (8, 3, 4, 2), (24, 5, 3, 2), (64, 8, 8, 3), (160, 6, 1, 1), (256, 8, 8, 4), (320, 7, 64, 5), (1000, 4, 1, 1)]       # E, k, groups, kept


def _case(E, dtype, seed):
    """rows with NaN and +inf at masked and at other experts; a third of the experts masked by the bias"""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(40, E, generator=gen)
    bias = 0.1 * torch.randn(E, generator=gen)
    masked = torch.rand(E, generator=gen) < 0.3
    masked[0], masked[1], masked[E // 2] = True, False, False
    bias[masked] = -math.inf
    off, on = torch.nonzero(masked)[:, 0], torch.nonzero(~masked)[:, 0]
    x[0, off] = math.nan                                                            # every masked one
    x[1, 0] = math.nan                                                              # one masked one, the lowest index
    x[2, 0] = math.inf
    x[3, off[-1]] = -math.nan
    x[4, on[0]] = math.nan                                                          # one that may be chosen
    x[5, on[-1]], x[5, off] = math.inf, math.nan
    x[6, on[-1]] = math.inf
    x[7, on] = math.nan
    x[8] = math.nan
    x[9] = math.inf
    x[10, on], x[10, off] = -math.inf, math.nan                                     # nothing can be chosen
    x[11, 0], x[11, on[0]] = math.nan, -math.inf
    return x.to(dtype), bias, masked


@pytest.mark.parametrize("E,k,groups,keep", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renorm", [True, False])
def test_sigmoid(E, k, groups, keep, dtype, renorm):
    from esc_gnn_amd import route_experts
    x, bias, masked = _case(E, dtype, E)
    w, at = route_experts(x.to(DEV), k, score="sigmoid", bias=bias.to(DEV), groups=groups, keep_groups=keep, renormalize=renorm)
    want_at, want_w = plain(x.double().numpy(), k, "sigmoid", bias.double().numpy(), groups, keep, 2, renorm, 1.0)
    at, w = at.cpu().numpy(), w.double().cpu().numpy()
    assert np.array_equal(at, want_at)
    assert np.array_equal(np.isnan(w), np.isnan(want_w))
    ok = ~np.isnan(w)
    assert (np.abs(w - want_w)[ok] <= 64 * U * want_w[ok] + 1e-37).all()
    assert not np.isnan(w[[0, 1, 2, 3]]).any() and (at[10] == -1).all() and (w[10] == 0).all()


@pytest.mark.parametrize("E,k,groups,keep", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_softmax(E, k, groups, keep, dtype):
    """a NaN or +inf anywhere in a row makes all its scores NaN: those that may be chosen follow each other by their index, behind the
    one that is the cause"""
    from esc_gnn_amd import route_experts
    x, bias, masked = _case(E, dtype, E + 1)
    w, at = (t.cpu() for t in route_experts(x.to(DEV), k, bias=bias.to(DEV), groups=groups, keep_groups=keep))
    can = ~masked & (x != -math.inf)
    cause = torch.isnan(x) | (x == math.inf)
    for r in range(12):
        chosen = [e for e in at[r].tolist() if e >= 0]
        assert all(bool(can[r, e]) for e in chosen) and len(set(chosen)) == len(chosen), r
        assert at[r].tolist() == chosen + [-1] * (k - len(chosen)) and bool((w[r, len(chosen):] == 0).all()), r
        assert chosen or not bool(can[r].any()), r
        if groups == 1:
            assert chosen == sorted(torch.nonzero(can[r])[:, 0].tolist(), key=lambda e: (not bool(cause[r, e]), e))[:k], r
        elif bool((cause & can)[r].any()):
            assert bool(cause[r, chosen[0]]), r
    assert bool(torch.isfinite(w[[0, 1, 2, 3]]).all())                               # the weights are a softmax over the chosen logits alone
    assert bool(torch.isfinite(w[12:]).all()) and not bool((masked[at[12:].clamp(min=0).long()] & (at[12:] >= 0)).any())


@pytest.mark.parametrize("size", [30.0, 1e3, 1e4, 1e6])
@pytest.mark.parametrize("E,groups,keep,dtype", [(8, 4, 2, torch.float32), (24, 4, 2, torch.float32), (64, 8, 3, torch.float32), (256, 16, 7, torch.bfloat16), (512, 64, 20, torch.float32)])
def test_groups_whose_large_biases_cancel(E, groups, keep, dtype, size):
    """two biases of opposite sign in each group: their sum, near that of the next group, has less than the rounding of its terms.  Which
    groups stay is decided by the 64-bit sums"""
    from esc_gnn_amd import route_experts
    gen = torch.Generator().manual_seed(int(size) + E)
    gs = E // groups
    rows = 3000
    x = torch.randn(rows, E, generator=gen).to(dtype)
    bias = torch.full((E,), -4 * size)
    a = size * (1 + torch.rand(groups, generator=gen))
    for g in range(groups):
        at = g * gs + torch.randperm(gs, generator=gen)[:2]
        bias[at[0]], bias[at[1]] = a[g], -a[g]
    k = min(2 * keep, 8)
    _, at = route_experts(x.to(DEV), k, score="sigmoid", bias=bias.to(DEV), groups=groups, keep_groups=keep)
    want, _ = plain(x.double().numpy(), k, "sigmoid", bias.double().numpy(), groups, keep, 2, True, 1.0)
    assert np.array_equal(at.cpu().numpy(), want)

"""
GPU tests of expert routing (esc_gnn_amd/experts.py, csrc/escat_route.hip) against a plain loop in 64 bits.  Which experts
are chosen has to be equal.  Weights: exp (<= 2 units in the last place, argument rounded: |l - m| <= 30 here adds 30 u), k-term
sums, division, scale: <= 64 u of the weight, u = 2^-24.  Gradients: the same per term, plus k roundings of the dot product of its
terms' sizes, plus one rounding to the logits' type.
"""
import math
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"


def plain(x, k, score, bias, groups, keep, top, renorm, scale):
    """x (rows, E) float64 numpy: experts, weights in 64 bits"""
    rows, E = x.shape
    at = np.full((rows, k), -1, np.int64)
    w = np.zeros((rows, k))
    for r in range(rows):
        l = x[r]
        ok = ~np.isneginf(l) & (np.ones(E, bool) if bias is None else ~np.isneginf(bias))
        with np.errstate(all="ignore"):
            if score == "softmax":
                m = np.nanmax(np.where(np.isneginf(l), -np.inf, l)) if not np.isneginf(l).all() and not np.isnan(l).all() else 0.0
                s = np.exp(l - m); s = s / s.sum()
            else:
                s = 1 / (1 + np.exp(-l))
            key = s + (0.0 if bias is None else bias)
        key = np.where(np.isnan(key), np.inf, key)
        key = np.where(ok, key, -np.inf)
        if groups > 1:
            gs = E // groups
            gsc = []
            for g in range(groups):
                b = np.sort(key[g * gs:(g + 1) * gs])[::-1][:top]
                gsc.append(-np.inf if np.isneginf(b[0]) else b[b > -np.inf].sum())
            kept = [g for g in np.argsort(-np.array(gsc), kind="stable")[:keep] if gsc[g] > -np.inf]
            mask = np.zeros(E, bool)
            for g in kept:
                mask[g * gs:(g + 1) * gs] = True
            key = np.where(mask, key, -np.inf)
        if bias is None:                                   # the order of the logits
            key = np.where(np.isneginf(key), -np.inf, np.where(np.isnan(l), np.inf, l))
        order = np.argsort(-key, kind="stable")[:k]
        order = [e for e in order if key[e] > -np.inf]
        at[r, :len(order)] = order
        if order:
            with np.errstate(all="ignore"):
                if score == "softmax" and renorm:
                    q = np.exp(l[order] - np.nanmax(l[order]) if not np.isnan(l[order]).all() else l[order]); q = q / q.sum()
                elif renorm:
                    q = s[order] / (s[order].sum() + 1e-20)
                else:
                    q = s[order]
            w[r, :len(order)] = scale * q
    return at, w


CASES = [  # E, k, score, bias, groups, keep, group_top, renorm, scale
    (1, 1, "softmax", False, 1, 1, 2, True, 1.0),
    (2, 1, "softmax", False, 1, 1, 2, False, 1.0),
    (7, 3, "softmax", True, 1, 1, 2, True, 2.5),
    (8, 2, "softmax", False, 1, 1, 2, True, 1.0),
    (8, 2, "sigmoid", True, 4, 2, 2, True, 1.0),
    (9, 9, "sigmoid", False, 3, 2, 1, False, 0.5),
    (16, 4, "softmax", True, 8, 3, 1, False, 1.0),
    (24, 5, "sigmoid", True, 8, 8, 2, True, 1.0),
    (33, 2, "softmax", False, 11, 4, 2, True, 1.0),
    (60, 6, "softmax", True, 1, 1, 2, False, 3.0),
    (64, 8, "sigmoid", True, 8, 3, 2, True, 1.0),
    (128, 16, "softmax", False, 1, 1, 2, True, 1.0),
    (160, 6, "softmax", False, 8, 3, 1, False, 16.0),
    (256, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    (320, 7, "softmax", True, 64, 5, 2, True, 1.0),
    (1000, 4, "softmax", True, 1, 1, 2, True, 1.0),
    (1024, 16, "sigmoid", False, 32, 9, 2, False, 1.0),
]


def logits_of(rows, E, dtype, seed, masks=True):
    gen = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(rows, E, generator=gen)
    if masks:
        x[torch.rand(rows, E, generator=gen) < 0.05] = -math.inf
        if rows > 3:
            x[1] = -math.inf                                                      # nothing can be chosen
            x[2] = -math.inf; x[2, E // 2] = 0.3                                  # one can
            x[3] = torch.finfo(dtype).min                                         # the type's lowest value is no mask
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("E,k,score,has_bias,groups,keep,top,renorm,scale", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_experts_and_weights(E, k, score, has_bias, groups, keep, top, renorm, scale, dtype):
    from esc_gnn_amd import route_experts
    rows = 203
    x = logits_of(rows, E, dtype, 7 * E + k)
    bias = 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(E)) if has_bias else None
    if has_bias and E > 8:
        bias[E // 3] = -math.inf
    w, at = route_experts(x, k, score=score, bias=None if bias is None else bias.to(DEV), groups=groups, keep_groups=keep, group_top=top,
                          renormalize=renorm, scale=scale)
    assert w.dtype == torch.float32 and at.dtype == torch.int32 and w.shape == at.shape == (rows, k)
    b64 = None if bias is None else bias.double().numpy()
    if score == "softmax" and groups > 1 and bias is None:
        # row 3 (all the type's lowest): the plain loop's softmax is uniform, the groups tie, the lowest stay: as here
        pass
    want_at, want_w = plain(x.double().cpu().numpy(), k, score, b64, groups, keep, top, renorm, scale)
    assert np.array_equal(at.cpu().numpy(), want_at)
    assert (np.abs(w.double().cpu().numpy() - want_w) <= 64 * U * want_w + 1e-37).all()


@pytest.mark.parametrize("E,k,score,has_bias,groups,keep,top,renorm,scale", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient(E, k, score, has_bias, groups, keep, top, renorm, scale, dtype):
    """against the formulas' gradient by automatic differentiation in 64 bits"""
    from esc_gnn_amd import route_experts
    rows = 101
    x = logits_of(rows, E, dtype, 3 * E + k)
    x[3] = 0.25
    bias = 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(E)).to(DEV) if has_bias else None
    xg = x.clone().requires_grad_()
    w, at = route_experts(xg, k, score=score, bias=bias, groups=groups, keep_groups=keep, group_top=top, renormalize=renorm, scale=scale)
    up = torch.randn(rows, k, generator=torch.Generator().manual_seed(1)).to(DEV)
    got, = torch.autograd.grad(w, xg, up)
    assert got.dtype == dtype and not bool(torch.isnan(got).any())
    x64 = x.double().requires_grad_()
    idx, there = at.long().clamp(min=0), at >= 0
    # (a masked logit takes a finite stand-in: its score is 0 and so is its gradient)
    xs = torch.where(x64 == -math.inf, -1e4, x64)
    l = xs.gather(1, idx)
    if score == "softmax" and renorm:
        q = torch.softmax(torch.where(there, l, -1e5), 1)
    elif score == "softmax":
        q = torch.softmax(xs, 1).gather(1, idx)
    else:
        q = torch.sigmoid(l)
        if renorm:
            q = q / ((q * there).sum(1, keepdim=True) + 1e-20)
    q = scale * q * there
    want, = torch.autograd.grad(q, x64, up.double())
    want = torch.where(torch.isfinite(x), want, 0.0)
    size = (w.double() * up.double().abs()).amax(1, keepdim=True)                 # of the terms that meet in an entry
    tol = (64 + 4 * k) * U * size * 2 + torch.finfo(dtype).eps / 2 * want.abs() + 1e-37
    assert bool(((got.double() - want).abs() <= tol).all())


def test_gradient_against_differences():
    """central differences of the weights themselves, step 2^-6: the third derivative of a softmax or sigmoid weight is below 1
    in size, so each of a row's <= 4 terms errs by h^2 / 6, plus 64 u / h for the weights' own rounding"""
    from esc_gnn_amd import route_experts
    h = 2.0 ** -6
    for score, renorm in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        x = torch.randn(40, 12, generator=torch.Generator().manual_seed(2)).to(DEV)
        x[:, :4] += 5.0                                                           # the choice does not change under the step
        up = torch.randn(40, 4, generator=torch.Generator().manual_seed(3)).to(DEV)
        xg = x.clone().requires_grad_()
        w, at = route_experts(xg, 4, score=score, renormalize=renorm)
        got, = torch.autograd.grad(w, xg, up)
        # weights by expert, so that a change of the order among the four does not matter
        f = lambda y: (lambda r: torch.zeros(40, 12, device=DEV).scatter_(1, r[1].long(), r[0]).double())(route_experts(y, 4, score=score, renormalize=renorm))  # noqa: E731
        byexp = torch.zeros(40, 12, device=DEV).scatter_(1, at.long(), up).double()
        for e in range(12):
            d = torch.zeros_like(x); d[:, e] = h
            num = ((f(x + d) - f(x - d)) * byexp).sum(1) / (2 * h)
            assert float((got[:, e].double() - num).abs().max()) <= 4 * 4 * (h * h / 6 + 64 * U / h)


def test_ties_and_near_ties_go_by_the_exact_value():
    from esc_gnn_amd import route_experts
    x = torch.zeros(5, 64, device=DEV)
    for kw in (dict(), dict(bias=torch.zeros(64, device=DEV)), dict(score="sigmoid", groups=8, keep_groups=2)):
        w, at = route_experts(x, 4, **kw)
        assert at.tolist() == [[0, 1, 2, 3]] * 5 and bool((w == 0.25).all())
    # s + bias equal but for 2^-40 of it: 32 bits cannot tell them apart
    l = torch.tensor([0.7, 0.7000001, 0.3, -0.2, 0.9, 0.1], dtype=torch.float32)
    s = torch.sigmoid(l.double())
    bias = (0.95 - s).float()                                                     # keys within rounding of 0.95
    key = s + bias.double()
    order = torch.sort(key, descending=True, stable=True).indices.tolist()
    assert len(set(key.float().tolist())) < 6                                     # equal in 32 bits
    w, at = route_experts(l.to(DEV).repeat(300, 1), 6, score="sigmoid", bias=bias.to(DEV))
    assert at.tolist() == [order] * 300


def test_not_finite():
    from esc_gnn_amd import route_experts
    x = torch.randn(4, 16, generator=torch.Generator().manual_seed(0)).to(DEV)
    x[0, 5] = float("nan"); x[1, 6] = float("inf"); x[2] = float("nan")
    for kw in (dict(), dict(score="sigmoid"), dict(bias=torch.zeros(16, device=DEV)), dict(score="sigmoid", groups=4, keep_groups=2)):
        w, at = route_experts(x, 2, **kw)
        assert at[0, 0] == 5
        assert bool(torch.isnan(w[0]).any()) and bool(torch.isnan(w[2]).all()) and bool(torch.isfinite(w[3]).all())
        assert bool((at >= 0).all()) and bool((at < 16).all())
        if kw.get("score") == "sigmoid":
            assert at[1, 0] == 6 and bool(torch.isfinite(w[1]).all())
        else:
            assert bool(torch.isnan(w[1]).any())


def test_shapes_strides_streams_and_repeats():
    from esc_gnn_amd import route_experts
    for rows in (0, 1, 63, 64, 65, 257):
        w, at = route_experts(torch.randn(rows, 24, device=DEV), 3)
        assert w.shape == (rows, 3)
    base = torch.randn(300, 48, device=DEV)
    for view in (base[:, ::2], base[1:, 3:27], base.t()[:24].t(), base.view(-1)[1:1 + 24 * 500].view(500, 24)):
        a, b = route_experts(view, 3), route_experts(view.clone().contiguous(), 3)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = torch.randn(70001, 24, device=DEV)
    first = route_experts(x, 3, score="sigmoid", bias=torch.zeros(24, device=DEV), groups=4, keep_groups=2)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = route_experts(x, 3, score="sigmoid", bias=torch.zeros(24, device=DEV), groups=4, keep_groups=2)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])

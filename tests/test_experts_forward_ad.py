"""Forward-mode differentiation is not served by the experts' operators: it has to say so, never to give a result without a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


def test_a_tangent_goes_by_the_autograd_function():
    from esc_gnn_amd.experts import _wants_grad
    x, e = torch.ones(3), torch.zeros(3, dtype=torch.int32)
    assert not _wants_grad((x, None, e)) and _wants_grad((None, e, torch.ones(3, requires_grad=True)))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert not dual.requires_grad
        assert _wants_grad((e, None, dual)) and not _wants_grad((x, None, e))
        with torch.no_grad():                                                     # (tangents do not stop there)
            assert _wants_grad((dual,)) and not _wants_grad((torch.ones(3, requires_grad=True),))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3000])
@pytest.mark.parametrize("width", [3, 40])
def test_calls_with_a_tangent_are_refused(rows, width):
    from esc_gnn_amd import expert_mlp, route_experts
    g = torch.Generator().manual_seed(rows)
    t = {n: torch.randn(*s, generator=g).to("cuda:0") for n, s in dict(x=(rows, width), weights=(rows, 2), w1=(4, 24, width), b1=(4, 24), w2=(4, 16, 24), b2=(4, 16)).items()}
    experts = torch.randint(0, 4, (rows, 2), generator=g, dtype=torch.int32).to("cuda:0")
    run = lambda q: expert_mlp(q["x"], q["weights"], experts, q["w1"], q["b1"], q["w2"], q["b2"])      # noqa: E731
    want = run(t)
    for n in t:
        with forward_ad.dual_level():
            assert torch.equal(run(t), want)
            with pytest.raises(NotImplementedError):
                run({**t, n: forward_ad.make_dual(t[n], torch.ones_like(t[n]))})
            with torch.no_grad(), pytest.raises(NotImplementedError):
                run({**t, n: forward_ad.make_dual(t[n], torch.ones_like(t[n]))})
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        route_experts(forward_ad.make_dual(t["x"], torch.ones_like(t["x"])), 2)
    assert torch.equal(run(t), want)

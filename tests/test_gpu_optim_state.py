"""
GPU tests of the optimizer's states over their life: taken from torch's AdamW in mid-run, copied, captured.
u = 2^-24, half a step of fp32.
"""
import copy
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"


def _grads(ps, it):
    for i, p in enumerate(ps):
        p.grad = torch.randn(p.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(100 * it + i)).to(p.dtype)


@pytest.mark.parametrize("kw", [dict(), dict(fused=True), dict(capturable=True), dict(foreach=False)])
def test_goes_on_where_torchs_left_off(kw):
    """8 steps by torch, 5 more by both.  A step errs by some 30 u of its update (|update| <= 5 lr = 0.025) and 4 u of the parameter, and
    what the moments are off by (8 u a step) passes on to the next: 5 steps stay under 1000 u of max(|p|, 1).  A count that is not
    taken over would show as a third or more of an update, 1e-3"""
    from esc_gnn_amd import AdamW
    torch.manual_seed(0)
    a = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in ((33, 7), (300,), (1,), (64, 65))]
    groups = lambda ps: [{"params": ps[:2]}, {"params": ps[2:], "lr": 5e-3, "betas": (0.8, 0.95)}]               # noqa: E731
    ref = torch.optim.AdamW(groups(a), lr=1e-3, **kw)
    for it in range(8):
        _grads(a, it); ref.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    opt = AdamW(groups(b), lr=0.5)                                                  # (the loaded groups' settings count)
    opt.load_state_dict(ref.state_dict())
    for it in range(8, 13):
        _grads(a, it); ref.step()
        _grads(b, it); opt.step()
        for x, y in zip(a, b):
            assert float((x - y).detach().abs().max()) <= 1000 * U * max(1.0, float(x.detach().abs().max())), it
    assert all(int(opt.state[p]["step"]) == 13 for p in b)


def test_a_count_of_another_type_is_refused_at_the_step():
    from esc_gnn_amd import AdamW
    p = torch.nn.Parameter(torch.ones(5, device=DEV))
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    before = p.detach().clone()
    for bad in (torch.ones(1, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32)):
        opt.state[p]["step"] = bad
        with pytest.raises(ValueError, match="step"):
            opt.step()
        assert torch.equal(p, before)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copy_goes_on_by_itself(bits):
    """a deep copy (with its own parameters) makes the same steps, bit for bit, and neither counts for the other"""
    from esc_gnn_amd import AdamW
    ps = [torch.nn.Parameter(torch.randn(n, device=DEV)) for n in (700, 33)]
    opt = AdamW(ps, state_bits=bits, max_grad_norm=0.3, seed=5)
    for it in range(2):
        _grads(ps, it); opt.step()
    other = copy.deepcopy(opt)
    assert torch.equal(other.grad_norm, opt.grad_norm)
    qs = other.param_groups[0]["params"]
    for it in range(2, 4):
        _grads(ps, it); opt.step()
    assert int(other.state[qs[0]]["step"]) == 2
    for it in range(2, 4):
        _grads(qs, it); other.step()
    for p, q in zip(ps, qs):
        assert p is not q and torch.equal(p, q) and all(torch.equal(opt.state[p][n], other.state[q][n]) for n in opt.state[p])


def test_a_capture_that_would_make_states_is_refused():
    """states and counts made inside a capture would be made anew by every replay: the step has to refuse, and to go on afterwards"""
    from esc_gnn_amd import AdamW
    ps = [torch.nn.Parameter(torch.randn(n, device=DEV)) for n in (700, 33)]
    for p in ps:
        p.grad = torch.ones_like(p)
    before = [p.detach().clone() for p in ps]
    opt = AdamW(ps)
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, before))
    opt.step()
    # a parameter that stays behind makes the others' count their own
    ps[1].grad = None
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert int(opt.state[ps[0]]["step"]) == int(opt.state[ps[1]]["step"]) == 1
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    ref = copy.deepcopy(opt)
    for k in range(3):
        graph.replay()
        for q, p in zip(ref.param_groups[0]["params"], ps):
            q.grad = None if p.grad is None else p.grad.clone()
        ref.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, ref.param_groups[0]["params"]))
        assert int(opt.state[ps[0]]["step"]) == 3 + k and int(opt.state[ps[1]]["step"]) == 1


@pytest.mark.parametrize("kw", [dict(), dict(fused=True), dict(capturable=True), dict(foreach=False)])
def test_torch_goes_on_where_this_one_left_off(kw):
    """the other way: 8 steps here, then 5 by both; the bound is counted in the test above"""
    from esc_gnn_amd import AdamW
    torch.manual_seed(1)
    a = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in ((33, 7), (300,), (1,), (64, 65))]
    opt = AdamW(a, lr=1e-3)
    for it in range(8):
        _grads(a, it); opt.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ref = torch.optim.AdamW(b, lr=0.5, **kw)
    saved = copy.deepcopy(opt.state_dict())
    for g, own in zip(saved["param_groups"], ref.param_groups):
        g.update({n: v for n, v in own.items() if n not in g})                        # (how torch is to run it)
    ref.load_state_dict(saved)
    for it in range(8, 13):
        _grads(a, it); opt.step()
        _grads(b, it); ref.step()
        for x, y in zip(a, b):
            assert float((x - y).detach().abs().max()) <= 1000 * U * max(1.0, float(y.detach().abs().max())), it
    assert all(int(ref.state[p]["step"]) == 13 for p in b)

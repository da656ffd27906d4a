"""
GPU tests of calls to the head's operators (esc_gnn_amd/optim.py, experts.py, train_dp.NodeExperts) that their documents allow and the
operators' own tests do not make: many groups, several threads, graphs side by side, a second backward, autocast, checkpoints, the edges of the sort.
Where a result is compared with another call's, the bits have to be equal; else the operators' own counted tolerances apply.
"""
import copy
import threading
import pytest
import torch

from .test_gpu_experts import DEV, NAMES, check, formula, make

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def call(t, **other):
    from esc_gnn_amd import expert_mlp
    q = {**t, **other}
    return expert_mlp(q["x"], q["weights"], q["experts"], q["w1"], q["b1"], q["w2"], q["b2"])


def both(t):
    a = {n: t[n].detach().clone().requires_grad_() for n in NAMES}
    y = call({**t, **a})
    return [y.detach(), *torch.autograd.grad(y, [a[n] for n in NAMES], t["up"])]


@pytest.mark.parametrize("bits", [32, 8])
def test_more_groups_than_a_call_holds(bits):
    """20 groups of settings against torch (fp32 states: five steps, 30 u of an update <= 5 lr and 4 u of the parameter each: 1000 u of
    max(|p|, 1)), and a captured step of them against the eager one, bit for bit"""
    from esc_gnn_amd import AdamW
    torch.manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(50 + 37 * i, device=DEV)) for i in range(20)] + [torch.nn.Parameter(torch.randn((), device=DEV))]
    groups = lambda q: [{"params": [p] + ([q[20]] if i == 19 else []), "lr": 1e-3 * (1 + i), "betas": (0.9 - 0.01 * i, 0.99)} for i, p in enumerate(q[:20])]      # noqa: E731
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, ref = AdamW(groups(ps), state_bits=bits, max_grad_norm=2.0), torch.optim.AdamW(groups(qs))
    for it in range(5):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad = torch.randn(p.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(100 * it + i))
            q.grad = p.grad.clone()
        want = torch.nn.utils.clip_grad_norm_(qs, 2.0)
        ref.step(); opt.step()
        assert abs(float(opt.grad_norm) - float(want)) <= 1e-5 * float(want)
        if bits == 32:
            for p, q in zip(ps, qs):
                assert float((p - q).detach().abs().max()) <= 1000 * U * max(1.0, float(q.detach().abs().max()))
    assert all(int(opt.state[p]["step"]) == 5 for p in ps)
    eager = copy.deepcopy(opt)
    rs = [p for g in eager.param_groups for p in g["params"]]
    for r, p in zip(rs, [p for g in opt.param_groups for p in g["params"]]):
        r.grad = p.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(3):
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        for r, p in zip(rs, [p for g in opt.param_groups for p in g["params"]]):
            assert torch.equal(p, r) and int(opt.state[p]["step"]) == 6 + k


def test_closures_and_scalars():
    from esc_gnn_amd import AdamW
    p = torch.nn.Parameter(torch.tensor(3.0, device=DEV))
    opt = AdamW([p], lr=0.1, weight_decay=0.0)

    def closure():
        opt.zero_grad()
        loss = (p - 1) ** 2
        loss.backward()
        return loss
    assert float(opt.step(closure).detach()) == 4.0
    assert abs(float(p.detach()) - 2.9) <= 1e-6 and float(p.grad) == 4.0


@pytest.mark.parametrize("shape", [(5, 40, 72, 56, 5, 2), (900, 40, 72, 56, 5, 2), (9000, 40, 72, 56, 2, 2)])
def test_threads_with_streams_of_their_own(shape):
    ts = [make(*shape, torch.bfloat16, True, seed=s) for s in range(4)]
    want = [both(t) for t in ts]
    torch.cuda.synchronize()
    got, errors = [[] for _ in ts], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i].append(both(ts[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                                     # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(ts))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for w, gs in zip(want, got):
        assert len(gs) == 5 and all(torch.equal(a, b) for g in gs for a, b in zip(w, g))


def test_two_graphs_side_by_side():
    """two captured passes replayed on two streams at once"""
    ts = [make(3000, 40, 72, 56, 5, 2, torch.float32, True, seed=s) for s in (1, 2)]
    want = [both(t) for t in ts]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in ts]
    for t in ts:
        g = torch.cuda.CUDAGraph()
        a = {n: t[n].detach().clone().requires_grad_() for n in NAMES}
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            y = call({**t, **a})
            outs.append([y, *torch.autograd.grad(y, [a[n] for n in NAMES], t["up"])])
        graphs.append((g, a))
    for _ in range(4):
        for st, (g, _) in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(a, b) for a, b in zip(w, o))
        both(ts[0])                                                               # eager work between the replays


@pytest.mark.parametrize("shape", [(3, 40, 72, 56, 5, 2), (700, 700, 72, 56, 5, 2), (9000, 40, 72, 56, 2, 2)])
def test_a_second_backward_of_the_same_pass(shape):
    t = make(*shape, torch.bfloat16, True, seed=3)
    a = {n: t[n].detach().clone().requires_grad_() for n in NAMES}
    y = call({**t, **a})
    one = torch.autograd.grad(y, [a[n] for n in NAMES], t["up"], retain_graph=True)
    other = torch.autograd.grad(y, [a[n] for n in NAMES], t["up"].flip(0), retain_graph=True)
    two = torch.autograd.grad(y, [a[n] for n in NAMES], t["up"])
    assert all(torch.equal(p, q) for p, q in zip(one, two)) and not torch.equal(one[0], other[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(call({**t, **a}), a["x"], t["up"], create_graph=True)[0].sum(), a["x"])       # no second derivative


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [6, 1500])
def test_rows_that_begin_one_element_into_a_buffer(dtype, rows):
    t = make(rows, 37, 45, 51, 6, 2, dtype, True, seed=rows)

    def off(v):
        b = torch.zeros(v.numel() + 1, dtype=v.dtype, device=DEV)[1:].view(v.shape)
        return b.copy_(v)
    want, got = both(t), both({n: off(v) for n, v in t.items()})
    assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.parametrize("shape", [(2600, 20, 24, 16, 1, 9), (2600, 20, 24, 16, 1, 10), (2600, 20, 24, 16, 1, 11), (4095, 20, 24, 16, 1, 2), (12288, 12, 24, 16, 2, 5), (12287, 12, 24, 16, 2, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_edges_of_the_sort_by_combination(shape, dtype):
    """one expert many times over: as many digits as a key has; rows at and below the least that it takes"""
    check(make(*shape, dtype, True, seed=sum(shape)), dtype)


def test_as_many_combinations_as_there_may_be():
    """31 experts, k = 2: 1024 keys, from 2048 rows for each of 496 groups on"""
    t = make(2048 * 496, 8, 8, 8, 31, 2, torch.bfloat16, True, seed=7)
    got = both(t)
    want, size = formula(t), formula(t, True)
    most = int(torch.bincount(t["experts"].flatten().clamp(min=0).long(), minlength=31).max())
    v = 2.0 ** -8
    for n, g in zip(("y",) + NAMES, got):
        terms = {"y": 18, "weights": 24, "x": 26}.get(n, 16 + most)
        tol = ((2 * terms + 64) * U + (0.0 if n in ("b2", "weights") else 2 * v)) * size[n] + (0.0 if n == "weights" else v) * want[n].abs() + 1e-30
        assert bool(((g.double() - want[n]).abs() <= tol).all()), n


@pytest.mark.parametrize("t16", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [4, 900])
def test_autocast(t16, rows):
    """fp32 tensors under autocast: the call in the 16-bit type, gradients back in fp32"""
    t = make(rows, 40, 72, 56, 5, 2, torch.float32, True, seed=8)
    a = {n: t[n].detach().clone().requires_grad_() for n in NAMES}
    with torch.autocast("cuda", dtype=t16):
        y = call({**t, **a})
    assert y.dtype is t16
    got = torch.autograd.grad(y, [a[n] for n in NAMES], t["up"].to(t16))
    low = {n: v if n in ("weights", "experts") else v.to(t16) for n, v in t.items()}
    want = both(low)
    assert torch.equal(y, want[0])
    for n, g, w in zip(NAMES, got, want[1:]):
        assert g.dtype is torch.float32 and torch.equal(g, w.float()), n


def test_a_checkpointed_layer():
    from torch.utils.checkpoint import checkpoint
    from esc_gnn_amd.train_dp import NodeExperts
    torch.manual_seed(6)
    layer = NodeExperts(24, 6, 2).to(DEV)
    x, up = torch.randn(2000, 24, device=DEV).requires_grad_(), torch.randn(2000, 24, device=DEV)
    ps = [x, *layer.parameters()]
    want = torch.autograd.grad(layer(x), ps, up)
    got = torch.autograd.grad(checkpoint(layer, x, use_reentrant=False), ps, up)
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_counts_of_any_shape():
    from esc_gnn_amd import expert_counts
    e = torch.randint(-2, 9, (300, 7), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    want = torch.bincount(e[(e >= 0) & (e < 6)].long(), minlength=6)
    for view in (e, e.t(), e.view(-1), e.view(10, 30, 7), e[:, :, None].expand(-1, -1, 1)):
        assert torch.equal(expert_counts(view, 6).long(), want)
    assert torch.equal(expert_counts(e[:, ::2], 6).long(), torch.bincount(e[:, ::2][(e[:, ::2] >= 0) & (e[:, ::2] < 6)].long(), minlength=6))
    assert expert_counts(torch.tensor(3, dtype=torch.int32, device=DEV), 6).tolist() == [0, 0, 0, 1, 0, 0]


def test_routing_in_threads_and_graphs():
    from esc_gnn_amd import route_experts
    x = torch.randn(5000, 64, device=DEV)
    bias = 0.1 * torch.randn(64, device=DEV)
    kw = dict(score="sigmoid", bias=bias, groups=8, keep_groups=3)
    up = torch.randn(5000, 4, device=DEV)

    def step(q):
        w, e = route_experts(q, 4, **kw)
        return w, e, torch.autograd.grad(w, q, up)[0]
    want = [v.detach() for v in step(x.clone().requires_grad_())]
    static = x.clone().requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for _ in range(3):
        graph.replay()
        step(x.clone().requires_grad_())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.no_grad():
        static.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[1], want[1].flip(0)) and torch.equal(out[0], want[0].flip(0))

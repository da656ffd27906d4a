"""
GPU tests of the training step with experts in the head and the multi-tensor AdamW (train_dp.DPTrainer's options).
"""
import os
import socket
import subprocess
import sys
import time
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def batch(B=48, n=64, seed=3):
    from esc_gnn_amd import synthetic
    from esc_gnn_amd.process_pyg_data import build_PQ_batch
    clouds = synthetic.ellipsoid_clouds(B, n, seed=seed)
    pos = torch.from_numpy(clouds.reshape(-1, 3)).to(DEV)
    gp = torch.arange(B + 1, dtype=torch.int32, device=DEV) * n
    b = build_PQ_batch(pos, gp, 5, {"kernel": "gaussian", "gaussian_eps": 0.05})
    gid = torch.arange(B, device=DEV).repeat_interleave(n)
    target = torch.from_numpy((clouds.max(1) - clouds.min(1)).max(1).astype(np.float32)).to(DEV)
    pc = b["P"].csr(); rp = pc.rowptr.long()
    rows = torch.repeat_interleave(torch.arange(pc.n, device=DEV), rp[1:] - rp[:-1]); cols = pc.col.long()
    edge_index = torch.stack([cols[rows != cols], rows[rows != cols]])
    return pos, pos, b["P"], b["Q"], gid, B, target, edge_index


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("optimizer,clip", [("torch", 1.0), ("escat", None), ("escat", 1.0), ("escat8", 1.0)])
def test_step_runs_with_experts(optimizer, clip, amp):
    from esc_gnn_amd.train_dp import DPTrainer, NodeExperts
    data = batch()
    torch.manual_seed(0)
    tr = DPTrainer(C=3, diffusion_kwargs=dict(scales_type="dyadic", J=3, include_lowpass=True), device=DEV, amp_bf16=amp, experts=6,
                   optimizer=optimizer, max_grad_norm=clip)
    before = [p.detach().clone() for p in tr.model.parameters()]
    losses = [float(tr.step(*data).detach()) for _ in range(4)]
    assert all(np.isfinite(losses))
    m = [m for m in tr.model.mlp if isinstance(m, NodeExperts)][0]
    assert int(m.load.sum()) == 0 and float(m.balance.abs().max()) <= 4 * m.rate + 1e-9
    for (name, p), q in zip(tr.model.named_parameters(), before):
        assert bool(torch.isfinite(p).all()) and not torch.equal(p, q), name
    assert all(p.grad.data_ptr() >= tr.bucket.flat.data_ptr() for p in tr.model.parameters())
    if optimizer != "torch":
        assert (tr.opt.grad_norm is None) == (clip is None)


def test_gradients_of_the_layer_against_64_bits():
    """NodeExperts against the same formula in 64 bits on the experts that it chose; sums of <= 700 x 32 products, relative to the
    largest entry 2000 u (u = 2^-24) holds with room"""
    from esc_gnn_amd import route_experts
    from esc_gnn_amd.train_dp import NodeExperts
    torch.manual_seed(2)
    layer = NodeExperts(32, 5, 2).to(DEV)
    layer.balance.copy_(torch.tensor([0.02, -0.02, 0.0, 0.01, -0.01]))
    x = torch.randn(700, 32, device=DEV).requires_grad_()
    up = torch.randn(700, 32, device=DEV)
    y = layer(x)
    ps = dict(layer.named_parameters())
    got = dict(zip(["x", *ps], torch.autograd.grad(y, [x, *ps.values()], up)))
    w, e = route_experts(torch.nn.functional.linear(x, layer.router.weight).detach(), 2, bias=layer.balance)
    assert int(layer.load.sum()) == 1400
    q = {"x": x.detach().double().requires_grad_(), **{n: p.detach().double().requires_grad_() for n, p in ps.items()}}
    w64 = torch.softmax((q["x"] @ q["router.weight"].t()).gather(1, e.long()), 1)
    z = torch.stack([torch.nn.functional.silu(q["x"] @ q["w1"][i].t() + q["b1"][i]) @ q["w2"][i].t() + q["b2"][i] for i in range(5)], 1)
    y64 = q["x"] + (w64[..., None] * z.gather(1, e.long()[..., None].expand(-1, -1, 32))).sum(1)
    want = dict(zip(q, torch.autograd.grad(y64, list(q.values()), up.double())))
    for n in want:
        assert float((got[n].double() - want[n]).abs().max()) <= 2000 * 2.0 ** -24 * float(want[n].abs().max()), n


def test_balance_bias_pulls_the_loads_together():
    from esc_gnn_amd.train_dp import NodeExperts
    torch.manual_seed(1)
    layer = NodeExperts(16, 8, 2, rate=0.02).to(DEV)
    x = torch.randn(4000, 16, device=DEV) + 0.5
    spread = []
    with torch.no_grad():
        for _ in range(60):
            layer(x)
            spread.append(float(layer.load.float().std()))
            layer.update_balance()
    assert spread[-1] < 0.5 * spread[0]


def test_default_head_is_as_before():
    from esc_gnn_amd.train_dp import ScatteringHead
    torch.manual_seed(0)
    h = ScatteringHead(7, 9)
    assert [tuple(p.shape) for p in h.parameters()] == [(16,), (16,), (256, 16), (256,), (256, 256), (256,), (1, 256), (1,)]


@pytest.mark.parametrize("optimizer", ["escat", "escat8"])
def test_two_ranks_keep_the_same_parameters(tmp_path, optimizer):
    """two processes share the GPU over gloo, each with clouds of its own: parameters and the balance bias stay equal bit for bit"""
    with socket.socket() as sk:
        sk.bind(("127.0.0.1", 0))
        port = sk.getsockname()[1]
    here = os.path.dirname(os.path.abspath(__file__))
    outs = [str(tmp_path / f"r{r}.pt") for r in range(2)]
    logs = [open(str(tmp_path / f"r{r}.log"), "w+") for r in range(2)]
    procs = [subprocess.Popen([sys.executable, os.path.join(here, "dp_experts_worker.py"), outs[r], optimizer], stdout=logs[r], stderr=subprocess.STDOUT,
                              env=dict(os.environ, RANK=str(r), LOCAL_RANK=str(r), WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))) for r in range(2)]
    try:
        end = time.monotonic() + 90
        while any(p.poll() is None for p in procs) and time.monotonic() < end and not any(p.poll() not in (None, 0) for p in procs):
            time.sleep(0.1)
    finally:
        for p in procs:
            if p.poll() is None:
                p.kill()
            p.wait(timeout=30)
    for p, f in zip(procs, logs):
        f.seek(0)
        assert p.returncode == 0, f.read()[-3000:]
    a, b = (torch.load(o, weights_only=True) for o in outs)
    assert list(a) == list(b) and any("balance" in n for n in a)
    for n in a:
        if "running_" not in n:                                   # (BatchNorm's statistics are each rank's own, with experts or without)
            assert torch.equal(a[n], b[n]), n


def test_a_captured_training_step_of_the_layer():
    """routing, experts, gradients and the optimizer's step in one graph: replays on new rows, with eager work between, equal the eager steps"""
    from esc_gnn_amd import adamw_step, expert_mlp, new_state8, route_experts
    from esc_gnn_amd.train_dp import NodeExperts
    torch.manual_seed(5)
    layer = NodeExperts(40, 6, 2).to(DEV)
    names = [n for n, _ in layer.named_parameters()]
    rows = [torch.randn(900, 40, device=DEV) for _ in range(4)]
    ups = [torch.randn(900, 40, device=DEV) for _ in range(4)]

    def fresh():
        ps = {n: p.detach().clone().requires_grad_() for n, p in layer.named_parameters()}
        sizes = [p.numel() for p in ps.values()]
        return ps, [new_state8(k, p.device) for k, p in zip(sizes, ps.values())], [new_state8(k, p.device) for k, p in zip(sizes, ps.values())], torch.zeros(1, dtype=torch.int32, device=DEV)

    def step(state, x, up):
        ps, m, v, count = state
        w, e = route_experts(torch.nn.functional.linear(x, ps["router.weight"]), 2, bias=layer.balance)
        y = x + expert_mlp(x, w, e, ps["w1"], ps["b1"], ps["w2"], ps["b2"])
        grads = torch.autograd.grad(y, [ps[n] for n in names], up)
        adamw_step([ps[n].detach() for n in names], list(grads), m, v, count, lr=1e-2, max_grad_norm=1.0)
        return y.detach()
    eager, caught, warm = fresh(), fresh(), fresh()
    x, up = rows[0].clone(), ups[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(warm, x, up)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(caught, x, up)
    for i in range(4):
        x.copy_(rows[i]); up.copy_(ups[i])
        graph.replay()
        want = step(eager, rows[i], ups[i])                         # (eager work between the replays)
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
        for n in names:
            assert torch.equal(caught[0][n], eager[0][n]), (i, n)
    assert int(caught[3]) == 4


def test_a_backward_behind_the_optimizers_step_is_refused():
    """what a graph saved and the step has changed since: an error, as with torch's optimizers"""
    from esc_gnn_amd import AdamW
    p = torch.nn.Parameter(torch.randn(64, device=DEV))
    opt = AdamW([p], lr=0.1)
    (p * 2).sum().backward()
    y = (p * p).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()

"""
GPU tests of the head's operators where offsets pass 32 bits: more than 2^31 elements in the logits, the rows, the hidden rows, a parameter.
What is checked is the last rows (elements), against the formula in 64 bits; tolerances as in the operators' own tests, counted for these sums.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def need(gib):
    free, _ = torch.cuda.mem_get_info()
    if free < gib << 30:
        pytest.skip(f"{gib} GiB of free GPU memory needed")


def test_route():
    from esc_gnn_amd import route_experts
    need(20)
    rows, E, k = (1 << 24) + 3, 136, 4
    x = torch.empty(rows, E, dtype=torch.float16, device=DEV).uniform_(-2, 2, generator=torch.Generator(DEV).manual_seed(1)).requires_grad_()
    assert x.numel() > 1 << 31
    w, e = route_experts(x, k)
    up = torch.zeros(rows, k, device=DEV)
    up[-5:] = torch.randn(5, k, device=DEV)
    g, = torch.autograd.grad(w, x, up)
    w = w.detach()
    t = x[-5:].detach().double().requires_grad_()
    order = torch.sort(t.detach(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(e[-5:].long(), order)
    w64 = torch.softmax(t.gather(1, order), 1)
    g64, = torch.autograd.grad(w64, t, up[-5:].double())
    assert float((w[-5:].double() - w64).abs().max()) <= 1e-6                     # a handful of fp32 operations on values <= 1
    assert float((g[-5:].double() - g64).abs().max()) <= 2.0 ** -11 * float(g64.abs().max()) + 1e-6
    assert not bool(g[:-5].any())


def test_experts():
    from esc_gnn_amd import expert_mlp
    need(60)
    rows, d, h, o, E = (1 << 23) + 77, 264, 264, 8, 3
    gen = torch.Generator(DEV).manual_seed(2)
    r = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)                # noqa: E731
    x = r(rows, d).requires_grad_()
    w1, w2 = ((r(E, h, d) / d ** 0.5).detach().requires_grad_(), (r(E, o, h) / h ** 0.5).detach().requires_grad_())
    weights = torch.rand(rows, 1, generator=gen, device=DEV)
    experts = torch.randint(0, E, (rows, 1), generator=gen, device=DEV, dtype=torch.int32)
    assert x.numel() > 1 << 31 and rows * h > 1 << 31
    y = expert_mlp(x, weights, experts, w1, None, w2, None)
    up = torch.zeros(rows, o, dtype=torch.bfloat16, device=DEV)
    up[-200:] = r(200, o)
    dx, dw1, dw2 = torch.autograd.grad(y, [x, w1, w2], up)
    t = {"x": x[-200:].detach().double().requires_grad_(), "w1": w1.detach().double().requires_grad_(), "w2": w2.detach().double().requires_grad_()}
    e = experts[-200:, 0].long()
    u = torch.bmm(t["w1"][e], t["x"][:, :, None])[:, :, 0]
    y64 = weights[-200:].double() * torch.bmm(t["w2"][e], torch.nn.functional.silu(u)[:, :, None])[:, :, 0]
    want = dict(zip(t, torch.autograd.grad(y64, list(t.values()), up[-200:].double())))
    # roundings of the hidden row (or du) and of the result, 2^-9 relative each, over random signs: 0.01 of the norm holds with room
    for got, ref in ((y[-200:], y64.detach()), (dx[-200:], want["x"]), (dw1, want["w1"]), (dw2, want["w2"])):
        assert float((got.double() - ref).norm()) <= 0.01 * float(ref.norm())
    assert not bool(dx[:-200].any())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(bits):
    from esc_gnn_amd import adamw_step, dequantize_state, new_state8
    need(50)
    n = (1 << 31) + 4097 * 3
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g[-9000:] = 1.0
    g[:9000] = -1.0
    m, v = (new_state8(n, p.device), new_state8(n, p.device)) if bits == 8 else (torch.zeros(n, device=DEV), torch.zeros(n, device=DEV))
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    norm = adamw_step([p], [g], [m], [v], step, lr=0.5, weight_decay=0.0, max_grad_norm=1e9)
    assert abs(float(norm) - 18000 ** 0.5) < 1e-3
    assert int(step) == 1
    # the first step moves by lr g / (|g| + eps); 8-bit states do not enter the first step's update but by what is stored
    assert bool((p[-9000:] == -0.5).all()) and bool((p[:9000] == 0.5).all()) and not bool(p[9000:-9000].any())
    mm = dequantize_state(*m, True) if bits == 8 else m
    assert bool((mm[9000:-9000] == 0).all())
    assert float((mm[-9000:] - 0.1).abs().max()) <= (0.1 / 8 if bits == 8 else 1e-8) and float((mm[:9000] + 0.1).abs().max()) <= (0.1 / 8 if bits == 8 else 1e-8)

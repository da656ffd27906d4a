"""
GPU tests of the experts' products (esc_gnn_amd/experts.py, csrc/escat_experts*.hip) against the formulas in 64 bits.

Tolerances, per element, counted before the first run.  u = 2^-24; v = half a step of the operands' type (fp32: u).  An fp32
sum of n terms errs by at most n u of the sum of their sizes.  With S(...) the same formula on sizes (absolute values):
  hidden      du <= (d + 2) u S(|W1||x| + |b1|);  h = silu(u): |silu'| <= 1.1, and 8 u of |h| for its own operations (fp32's expf; the
              hardware exponential of 16-bit types errs by |u| u more: |u| <= 30 here);  then w h rounded: v + u
  y           (h + k + 2) u S(..) + v' S(w |W2| |h|) with v' = v + the hidden row's relative error;  then rounded to the type: v |y|
  gradients   the same with G = W2^T dy: (o + 2) u S, du = w G silu'(u): |silu''| <= 0.5, rounded v; sums over n rows: n u S.
The tests use the coarser  c1 u S + c2 v S + v |result|  with c1 = twice the number of summed terms + 64 and c2 = 2, S = the
formula on sizes with silu replaced by |u| + (its argument's error is then in c1).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"


def make(rows, d, h, o, E, k, dtype, bias, seed=0, drop=0.05):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)                                       # noqa: E731
    t = dict(x=r(rows, d), weights=torch.rand(rows, k, generator=g), w1=r(E, h, d) / d ** 0.5, b1=0.1 * r(E, h) if bias else None,
             w2=r(E, o, h) / h ** 0.5, b2=0.1 * r(E, o) if bias else None, up=r(rows, o))
    t = {n: None if v is None else (v if n == "weights" else v.to(dtype)).to(DEV) for n, v in t.items()}
    e = torch.randint(0, E, (rows, k), generator=g)
    e = torch.where(torch.rand(rows, k, generator=g) < drop, -1, e)
    t["experts"] = e.to(torch.int32).to(DEV)
    return t


NAMES = ("x", "weights", "w1", "b1", "w2", "b2")


def formula(t, sizes=False):
    """outputs and gradients in 64 bits; sizes: of absolute values, silu(u) -> |u|, silu' -> 1.1"""
    c = {n: None if t[n] is None else (t[n].double().abs() if sizes else t[n].double()) for n in NAMES + ("up",)}
    E = t["w1"].shape[0]
    out = {"y": torch.zeros(t["up"].shape, dtype=torch.float64, device=DEV)}
    out.update({n: None if c[n] is None else torch.zeros_like(c[n]) for n in NAMES})
    for e in range(E):
        row, slot = torch.nonzero(t["experts"] == e, as_tuple=True)
        if not row.numel():
            continue
        u = c["x"][row] @ c["w1"][e].t()
        if c["b1"] is not None:
            u = u + c["b1"][e]
        s = torch.ones_like(u) if sizes else torch.sigmoid(u)
        hh = u * s
        slope = torch.full_like(u, 1.1) if sizes else s * (1 + u * (1 - s))
        z = hh @ c["w2"][e].t()
        if c["b2"] is not None:
            z = z + c["b2"][e]
        w = c["weights"][row, slot][:, None]
        out["y"].index_add_(0, row, w * z)
        dy = c["up"][row]
        out["weights"].index_put_((row, slot), (z * dy).sum(1))
        out["w2"][e] = (w * dy).t() @ hh
        G = dy @ c["w2"][e]
        du = w * G * slope
        if sizes:
            du = du + 0.5 * w * G * u                                                  # silu''
        out["x"].index_add_(0, row, du @ c["w1"][e])
        out["w1"][e] = du.t() @ c["x"][row]
        if c["b1"] is not None:
            out["b1"][e], out["b2"][e] = du.sum(0), (w * dy).sum(0)
    return out


def check(t, dtype):
    from esc_gnn_amd import expert_mlp
    a = {n: None if t[n] is None else t[n].detach().clone().requires_grad_() for n in NAMES}
    y = expert_mlp(a["x"], a["weights"], t["experts"], a["w1"], a["b1"], a["w2"], a["b2"])
    names = [n for n in NAMES if a[n] is not None]
    got = dict(zip(names, torch.autograd.grad(y, [a[n] for n in names], t["up"])))
    got["y"] = y.detach()
    want, size = formula(t), formula(t, True)
    rows, d = t["x"].shape
    E, o, h = t["w2"].shape
    k = t["experts"].shape[1]
    most = int(torch.bincount(t["experts"].flatten().clamp(min=0).long(), minlength=E).max()) if rows else 0
    terms = {"y": d + h + k, "weights": d + h + o, "x": d + o + h + k, "w1": d + o + most, "b1": d + o + most, "w2": d + most, "b2": most}
    v = torch.finfo(dtype).eps / 2
    for n in ["y"] + names:
        assert got[n].shape == want[n].shape and got[n].dtype == (torch.float32 if n == "weights" else dtype), n
        mid = 2 * v if dtype != torch.float32 and n != "b2" and n != "weights" else 0.0      # dw and db2 see no 16-bit value of ours
        end = 0.0 if n == "weights" else v
        tol = ((2 * terms[n] + 64) * U + mid) * size[n] + end * want[n].abs() + (6e-8 if dtype == torch.float16 else 1e-30)
        bad = (got[n].double() - want[n]).abs() > tol
        assert not bool(bad.any()), (n, int(bad.sum()), float(((got[n].double() - want[n]).abs() / tol).max()))


SHAPES = [  # rows, d, h, o, E, k
    (1, 1, 1, 1, 1, 1),
    (1, 64, 64, 64, 4, 2),
    (3, 5, 7, 9, 2, 2),
    (2, 242, 256, 256, 8, 2),
    (127, 33, 65, 31, 3, 1),
    (129, 128, 128, 128, 1, 1),
    (300, 242, 256, 256, 8, 2),
    (257, 64, 129, 200, 5, 3),
    (1000, 17, 300, 40, 64, 4),
    (2500, 130, 66, 258, 2, 2),
    (700, 1024, 40, 24, 6, 2),
    (5000, 40, 72, 48, 3, 2),
    (64, 8, 520, 16, 300, 6),
    # few rows: the form without sorting
    (60, 242, 256, 250, 8, 2),
    (20, 1024, 40, 24, 6, 2),
    (33, 17, 300, 40, 64, 4),
    (100, 130, 66, 258, 2, 2),
    # more pairs than the form for few rows takes, by pair and with k = 1
    (3000, 33, 65, 31, 64, 2),
    (5000, 130, 129, 70, 40, 3),
    (6000, 50, 40, 60, 5, 1),
    # u kept by the forward with 16-bit types, by pair and by combination, ragged
    (700, 700, 140, 130, 6, 2),
    (7000, 650, 70, 40, 2, 2),
    # combinations of six, and of one expert with itself
    (15000, 20, 24, 16, 2, 6),
    (5000, 20, 24, 16, 1, 2),
    # many experts, many slots
    (6000, 24, 16, 24, 1024, 2),
    (6000, 24, 16, 24, 1024, 1),
    (40, 24, 40, 16, 100, 40),
    (900, 24, 40, 16, 7, 64),
    # enough rows for tiles by combination of experts (escat_experts.h): k = 2, 3; ragged sizes
    (7000, 40, 72, 136, 2, 2),
    (21000, 33, 47, 70, 3, 3),
    (21000, 242, 66, 130, 4, 2),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [True, False])
def test_outputs_and_gradients(shape, dtype, bias):
    check(make(*shape, dtype, bias, seed=sum(shape)), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unequal_loads(dtype):
    """all rows to one expert, none to the others; rows routed nowhere; numbers outside the experts; an expert twice in a row"""
    t = make(900, 48, 80, 56, 7, 2, dtype, True, seed=5)
    t["experts"][:] = 3
    check(t, dtype)
    t["experts"][::2] = -1
    t["experts"][1::6, 0] = 6
    check(t, dtype)
    bad = t["experts"].clone()
    t["experts"][t["experts"] == 6] = -1
    from esc_gnn_amd import expert_mlp
    bad[bad == 6] = 7
    args = [t["x"], t["weights"], None, t["w1"], t["b1"], t["w2"], t["b2"]]
    y = [expert_mlp(*args[:2], e, *args[3:]) for e in (t["experts"], bad, torch.where(bad == 7, -100, bad))]
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
    t["experts"][:] = -1
    check(t, dtype)


def test_no_rows():
    from esc_gnn_amd import expert_mlp, expert_counts
    t = make(0, 12, 20, 8, 3, 2, torch.float32, True)
    a = {n: t[n].requires_grad_() for n in NAMES}
    y = expert_mlp(a["x"], a["weights"], t["experts"], a["w1"], a["b1"], a["w2"], a["b2"])
    assert y.shape == (0, 8)
    for n, g in zip(NAMES, torch.autograd.grad(y, [a[n] for n in NAMES], t["up"])):
        assert g.shape == a[n].shape and not bool(g.any())
    assert expert_counts(t["experts"], 3).tolist() == [0, 0, 0]


def test_masked_rows_keep_what_is_not_finite_to_themselves():
    """a row that is routed nowhere may hold anything: it reaches neither y nor a gradient of another; a routed one shows in its own row
    and in the gradients of its expert only"""
    from esc_gnn_amd import expert_mlp
    for dtype in (torch.float32, torch.bfloat16):
        t = make(300, 40, 33, 20, 4, 2, dtype, True, seed=2, drop=0.0)
        t["experts"][7] = -1
        t["x"][7], t["up"][7], t["weights"][7] = float("nan"), float("inf"), float("nan")
        want = {n: None if t[n] is None else t[n].clone() for n in t}
        want["x"][7] = 0; want["up"][7] = 0; want["weights"][7] = 0
        res = []
        for q in (t, want):
            a = {n: q[n].detach().requires_grad_() for n in NAMES}
            y = expert_mlp(a["x"], a["weights"], q["experts"], a["w1"], a["b1"], a["w2"], a["b2"])
            res.append([y.detach(), *torch.autograd.grad(y, [a[n] for n in NAMES], q["up"])])
        for p, q in zip(*res):
            assert torch.equal(p, q) and bool(torch.isfinite(p).all())
        t["experts"][9] = 1; t["x"][9, 3] = float("nan")
        y = expert_mlp(t["x"], t["weights"], t["experts"], t["w1"], t["b1"], t["w2"], t["b2"])
        bad = torch.isnan(y).any(1)
        assert bool(bad[9]) and int(bad.sum()) == 1


def test_gradient_against_differences():
    """fp32: directional central differences along random directions.  f = <y, up> in 64 bits of fp32 outputs; step 2^-7 of a
    direction of norm 1 changes f by terms whose third derivative is below 10 here: h^2 10 / 6, and f's own rounding, 1e-6 |f-sizes| / h"""
    from esc_gnn_amd import expert_mlp
    t = make(50, 20, 24, 16, 4, 2, torch.float32, True, seed=8)
    a = {n: t[n].detach().requires_grad_() for n in NAMES}
    run = lambda q: expert_mlp(q["x"], q["weights"], t["experts"], q["w1"], q["b1"], q["w2"], q["b2"])        # noqa: E731
    grads = dict(zip(NAMES, torch.autograd.grad(run(a), [a[n] for n in NAMES], t["up"])))
    size = float(formula(t, True)["y"].abs().mul(t["up"].abs()).sum())
    h = 2.0 ** -7
    for n in NAMES:
        v = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(3)).to(DEV); v /= v.norm()
        f = [float((run({**t, n: t[n] + s * h * v}).double() * t["up"].double()).sum()) for s in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * h) - float((grads[n] * v).double().sum())) <= 10 * h * h / 6 + 1e-6 * size / h, n


def test_only_what_is_asked_for():
    from esc_gnn_amd import expert_mlp
    t = make(200, 24, 40, 16, 3, 2, torch.float32, True, seed=4)
    a = {n: t[n].detach().requires_grad_() for n in NAMES}
    full = dict(zip(NAMES, torch.autograd.grad(expert_mlp(a["x"], a["weights"], t["experts"], a["w1"], a["b1"], a["w2"], a["b2"]), [a[n] for n in NAMES], t["up"])))
    for n in NAMES:
        q = {m: t[m].detach().requires_grad_(m == n) for m in NAMES}
        g, = torch.autograd.grad(expert_mlp(q["x"], q["weights"], t["experts"], q["w1"], q["b1"], q["w2"], q["b2"]), q[n], t["up"])
        assert torch.equal(g, full[n]), n


def test_counts_and_the_same_bits_again():
    from esc_gnn_amd import expert_mlp, expert_counts
    for P, E in ((1, 1), (5000, 7), (70000, 64), (300, 1024), (262144, 3)):
        e = torch.randint(-1, E + 1, (P,), generator=torch.Generator().manual_seed(P), dtype=torch.int32).to(DEV)
        want = torch.bincount(e[(e >= 0) & (e < E)].long(), minlength=E)
        assert torch.equal(expert_counts(e, E).long(), want)
    t = make(32000, 64, 64, 64, 5, 2, torch.bfloat16, True, seed=6)
    outs = []
    st = torch.cuda.Stream()
    for i in range(3):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st if i == 2 else torch.cuda.current_stream()):
            a = {n: t[n].detach().requires_grad_() for n in NAMES}
            y = expert_mlp(a["x"], a["weights"], t["experts"], a["w1"], a["b1"], a["w2"], a["b2"])
            outs.append([y, *torch.autograd.grad(y, [a[n] for n in NAMES], t["up"])])
        torch.cuda.current_stream().wait_stream(st)
    for o in outs[1:]:
        for p, q in zip(outs[0], o):
            assert torch.equal(p, q)


def test_strided_arguments():
    from esc_gnn_amd import expert_mlp
    t = make(100, 24, 40, 16, 3, 2, torch.float32, True, seed=4)
    y = expert_mlp(t["x"], t["weights"], t["experts"], t["w1"], t["b1"], t["w2"], t["b2"])
    wide = torch.zeros(100, 48, device=DEV); wide[:, ::2] = t["x"]
    odd = torch.zeros(3 * 40 * 24 + 1, device=DEV)[1:].view(3, 40, 24); odd.copy_(t["w1"])
    z = expert_mlp(wide[:, ::2], t["weights"].t().contiguous().t(), t["experts"].t().contiguous().t(), odd, t["b1"], t["w2"], t["b2"])
    assert torch.equal(y, z)
    x = t["x"].requires_grad_()
    g0, = torch.autograd.grad(expert_mlp(x, t["weights"], t["experts"], t["w1"], t["b1"], t["w2"], t["b2"]).sum(), x)      # an expanded gradient
    g1, = torch.autograd.grad(expert_mlp(x, t["weights"], t["experts"], t["w1"], t["b1"], t["w2"], t["b2"]), x, torch.ones(100, 16, device=DEV))
    assert torch.equal(g0, g1)


def test_captured_forward_and_backward():
    """a captured pass is replayed with other routings and rows, eager work between the replays; every replay equals the eager pass"""
    from esc_gnn_amd import expert_mlp
    t = make(600, 40, 72, 56, 5, 2, torch.bfloat16, True, seed=9)
    a = {n: t[n].detach().clone().requires_grad_() for n in NAMES}
    e, up = t["experts"].clone(), t["up"].clone()

    def step(q, e, up):
        y = expert_mlp(q["x"], q["weights"], e, q["w1"], q["b1"], q["w2"], q["b2"])
        return [y, *torch.autograd.grad(y, [q[n] for n in NAMES], up)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            step(a, e, up)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, e, up)
    for i in range(3):
        o = make(600, 40, 72, 56, 5, 2, torch.bfloat16, True, seed=20 + i, drop=0.3 * i)
        with torch.no_grad():
            for n in NAMES:
                a[n].copy_(o[n])
        e.copy_(o["experts"]); up.copy_(o["up"])
        graph.replay()
        q = {n: o[n].detach().requires_grad_() for n in NAMES}
        want = step(q, o["experts"], o["up"])
        torch.cuda.synchronize()
        for g, w in zip(out, want):
            assert torch.equal(g, w)


def test_a_run_of_them_together():
    """router, experts, loss, clip and AdamW as a training step: gradients against 64-bit differentiation of the same formulas, and a step"""
    from esc_gnn_amd import AdamW, expert_mlp, route_experts
    g = torch.Generator().manual_seed(1)
    rows, d, h, E, k = 500, 30, 44, 6, 2
    x = torch.randn(rows, d, generator=g).to(DEV)
    ps = {n: torch.nn.Parameter(v.to(DEV)) for n, v in dict(gate=torch.randn(E, d, generator=g) / 5, w1=torch.randn(E, h, d, generator=g) / 6,
          b1=torch.zeros(E, h), w2=torch.randn(E, 3, h, generator=g) / 7, b2=torch.zeros(E, 3)).items()}
    target = torch.randn(rows, 3, generator=g).to(DEV)
    w, e = route_experts(x @ ps["gate"].t(), k)
    y = expert_mlp(x, w, e, ps["w1"], ps["b1"], ps["w2"], ps["b2"])
    ((y - target) ** 2).mean().backward()
    q = {n: p.detach().double().requires_grad_() for n, p in ps.items()}
    l = x.double() @ q["gate"].t()
    w64 = torch.softmax(l.gather(1, e.long()), 1)
    z = torch.stack([torch.nn.functional.silu(x.double() @ q["w1"][i].t() + q["b1"][i]) @ q["w2"][i].t() + q["b2"][i] for i in range(E)], 1)
    y64 = (w64[..., None] * z.gather(1, e.long()[..., None].expand(-1, -1, 3))).sum(1)
    ((y64 - target.double()) ** 2).mean().backward()
    for n in ps:
        # each entry sums <= 500 x 3 x 44 rounded products; relative to the largest entry 2000 u holds with room
        assert float((ps[n].grad.double() - q[n].grad).abs().max()) <= 2000 * U * float(q[n].grad.abs().max()), n
    before = {n: p.detach().clone() for n, p in ps.items()}
    opt = AdamW(ps.values(), lr=1e-2, state_bits=8, max_grad_norm=1.0)
    opt.step()
    assert all(bool(torch.isfinite(p).all()) and not torch.equal(p, before[n]) for n, p in ps.items())


@pytest.mark.parametrize("shape", [(11403, 106, 57, 200, 34, 1), (9000, 112, 34, 48, 20, 4), (9000, 40, 185, 144, 12, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_end_inside_a_piece_of_16_bytes(shape, dtype):
    """two or three elements behind the last whole piece of a hidden row, more rows than the form for few takes"""
    check(make(*shape, dtype, False, seed=11), dtype)


@pytest.mark.parametrize("width", range(57, 66))
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_every_remainder_of_a_row(width, dtype):
    check(make(2600, width, width + 3, width + 6, 6, 2, dtype, True, seed=width), dtype)


@pytest.mark.parametrize("shape", [(3000, 33, 65, 31, 64, 2), (5000, 40, 72, 48, 3, 1), (7000, 40, 72, 136, 2, 2)])
def test_only_what_is_asked_for_of_many_rows(shape):
    """each gradient alone, with and without the forward's hidden rows, equals the one among all"""
    from esc_gnn_amd import expert_mlp
    t = make(*shape, torch.bfloat16, True, seed=12)
    a = {n: t[n].detach().requires_grad_() for n in NAMES}
    full = dict(zip(NAMES, torch.autograd.grad(expert_mlp(a["x"], a["weights"], t["experts"], a["w1"], a["b1"], a["w2"], a["b2"]), [a[n] for n in NAMES], t["up"])))
    for n in NAMES:
        q = {m: t[m].detach().requires_grad_(m == n) for m in NAMES}
        g, = torch.autograd.grad(expert_mlp(q["x"], q["weights"], t["experts"], q["w1"], q["b1"], q["w2"], q["b2"]), q[n], t["up"])
        assert torch.equal(g, full[n]), n


class Guarded:
    """device memory of so many bytes between two runs of a pattern"""
    def __init__(self, nbytes):
        self.n = nbytes
        self.all = torch.full((nbytes + 8192,), 0x5A, dtype=torch.uint8, device=DEV)

    def ptr(self):
        return self.all.data_ptr() + 4096

    def view(self, dtype, shape):
        return self.all[4096:4096 + self.n].view(dtype).view(shape)

    def intact(self):
        return bool((self.all[:4096] == 0x5A).all()) and bool((self.all[4096 + self.n:] == 0x5A).all())


@pytest.mark.parametrize("shape", [(3, 17, 33, 9, 2, 2), (300, 242, 256, 250, 8, 2), (3000, 33, 65, 31, 64, 2), (5000, 41, 70, 45, 3, 1), (7000, 40, 77, 137, 2, 2),
                                   (700, 1030, 43, 24, 6, 2), (2500, 1030, 143, 24, 6, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keep", [False, True])
def test_nothing_is_written_outside(shape, dtype, keep):
    """every buffer that the library writes lies between two patterns; a workspace is exactly as large as it says, full of NaN before"""
    import ctypes
    from esc_gnn_amd import _lib
    lib = _lib.load()
    rows, d, h, o, E, k = shape
    t = make(*shape, dtype, True, seed=13)
    size = t["x"].element_size()
    dims = _lib.EscatExpertsDims(rows, 0 if dtype is torch.float32 else 1, d, h, o, E, k)
    at = ctypes.addressof(dims)
    p = {n: t[n].contiguous().data_ptr() for n in NAMES + ("up", "experts")}
    plan = Guarded(lib.escat_experts_plan_bytes(rows, k, E))
    _lib.check(lib.escat_experts_plan(p["experts"], rows, k, E, plan.ptr(), plan.n, 0, 0), "plan")
    sorts = bool(lib.escat_experts_fwd_needs_plan(at))
    hid = Guarded(lib.escat_experts_hidden_bytes(at)) if keep and sorts else None
    hp = hid.ptr() if hid else 0
    ws = [Guarded(lib.escat_experts_workspace_bytes(at, b, int(hid is not None))) for b in (0, 1)]
    for w in ws + ([hid] if hid else []):
        w.all[4096:4096 + w.n] = 0xFF
    y = Guarded(rows * o * size)
    _lib.check(lib.escat_experts_fwd(at, p["x"], p["weights"], p["experts"], p["w1"], p["b1"], p["w2"], p["b2"], plan.ptr(), y.ptr(), hp, ws[0].ptr(), ws[0].n, 0), "fwd")
    g = {n: Guarded(t[n].numel() * t[n].element_size()) for n in NAMES}
    _lib.check(lib.escat_experts_bwd(at, p["x"], p["weights"], p["w1"], p["b1"], p["w2"], p["b2"], plan.ptr(), hp, p["up"], g["x"].ptr(), g["weights"].ptr(), g["w1"].ptr(),
                                     g["b1"].ptr(), g["w2"].ptr(), g["b2"].ptr(), ws[1].ptr(), ws[1].n, 0), "bwd")
    torch.cuda.synchronize()
    for n, b in dict(g, plan=plan, y=y, fwd=ws[0], bwd=ws[1], **({"hidden": hid} if hid else {})).items():
        assert b.intact(), n
    want = formula(t)
    for n in NAMES + ("y",):
        got = (y if n == "y" else g[n]).view(torch.float32 if n == "weights" else dtype, want[n].shape)
        # (how near is the other tests' matter: here a wrong buffer would be nowhere near)
        assert float((got.double() - want[n]).norm()) <= 0.02 * float(want[n].norm()) + 1e-30, n

"""
GPU tests of AdamW with 32-bit and 8-bit states (esc_gnn_amd/optim.py, csrc/escat_adamw.hip) against the formulas in 64 bits.

Tolerances, counted before the first run.  Half a step of fp32 is u = 2^-24.
  m = b1 m + (1-b1) (c g): c, c g, the two products, their sum, and b1, 1-b1 as fp32 constants: <= 7 roundings of the terms' sizes.
  v: one more (the square).  p = p d - num / den: the update's size times roundings of num (m's 7, the scalar's, the product: 9)
  and den (v's 8 halved by the root, root, scalar, product, sum: 8) and the division: <= 18; p d: constant and product: 2; the
  difference: 1; then one rounding to the parameter's type.
"""
import math
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"
TOP = {True: 15.0 * 2 ** 14, False: 14.0 * 2 ** 30}


# ------------------------------------------------------------------ the 8-bit format, restated bit by bit
def values8(code, scale, signed):
    c = code.cpu().numpy().astype(np.int64)
    a = c & 127 if signed else c
    v = np.where(a < 8, a, (8 + a % 8) * 2.0 ** (a // 8 - 1))
    v = np.where(c == (128 if signed else 255), np.nan, v)
    if signed:
        v = np.where(c > 128, -v, v)
    return v * np.repeat(scale.cpu().numpy().astype(np.float64), 256)[:len(c)]


def mix(x):
    x = ((x ^ (x >> 16)) * 0x6C8E9CF5) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0x5851F42D) & 0xFFFFFFFF
    return x ^ (x >> 16)


def noise(seed, t, ordinal, n):
    key = mix(np.int64((t + seed * 0x2545F491) & 0xFFFFFFFF))
    key = mix((key + ordinal * 0x632BE5AB) & 0xFFFFFFFF)
    i = np.arange(n, dtype=np.int64)
    return mix(mix(((i >> 32) + key) & 0xFFFFFFFF) ^ (i & 0xFFFFFFFF))


def encode8(x, r16, signed):
    """x fp32 (numpy) -> codes, scales: the fp32 and integer operations of the format"""
    n = len(x)
    nb = -(-n // 256)
    pad = np.zeros(nb * 256, np.float32); pad[:n] = x
    fin = np.where(np.isfinite(pad), np.abs(pad), 0).reshape(nb, 256).max(1).astype(np.float32)
    fin = np.where((fin > 0) & (fin < 2.0 ** -90), np.float32(2.0 ** -90), fin).astype(np.float32)
    top = np.float32(TOP[signed])
    with np.errstate(all="ignore"):
        inv = np.where(fin > 0, (np.float32(1) / fin) * top, np.float32(0)).astype(np.float32)
        y = np.minimum(np.abs(pad) * np.repeat(inv, 256), top).astype(np.float32)[:n]
        hi = ((y.view(np.int32).astype(np.int64) + (r16 << 4)) >> 20) - (129 << 3)
        lo = np.where(y < 8, y + r16.astype(np.float32) * np.float32(2.0 ** -16), 0).astype(np.float32).astype(np.int64)
    c = np.where(y >= 8, hi, lo)
    if signed:
        c = np.minimum(c, 127); c = np.where((x < 0) & (c > 0), c | 128, c); c = np.where(np.isfinite(x), c, 128)
    else:
        c = np.minimum(c, 254); c = np.where(x > 0, np.maximum(c, 1), c); c = np.where(np.isfinite(x), c, 255)
    return c.astype(np.uint8), (fin * np.float32(np.float32(1) / top)).astype(np.float32)


# ------------------------------------------------------------------ the step in 64 bits
def step64(p, g, m, v, t, clip, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    g = g.double() * clip
    m = betas[0] * m.double() + (1 - betas[0]) * g
    v = betas[1] * v.double() + (1 - betas[1]) * g * g
    upd = lr / (1 - betas[0] ** t) * m / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p.double() * (1 - lr * weight_decay) - upd, m, v, upd


def make(n, dtype, gtype, seed, off=0):
    """a parameter, gradient and states that begin `off` elements into their buffers"""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda: torch.randn(n + off, generator=gen, device=DEV)                       # noqa: E731
    size = torch.exp(2 * r())
    p, g = (0.1 * r()).to(dtype)[off:], (r() * size * 1e-3).to(gtype)[off:]
    m, v = (0.3 * r() * size * 1e-3)[off:], (size * size * 1e-6 * torch.exp(r()))[off:]
    return p, g, m, v


def check32(p, m, v, p0, g, m0, v0, t, clip, **kw):
    P, M, V, upd = step64(p0, g, m0, v0, t, clip, **kw)
    b1, b2 = kw.get("betas", (0.9, 0.999))
    gs = g.double().abs() * clip
    assert bool(((m.double() - M).abs() <= 7 * U * (b1 * m0.double().abs() + (1 - b1) * gs) + 1e-45).all())
    assert bool(((v.double() - V).abs() <= 8 * U * (b2 * v0.double() + (1 - b2) * gs * gs) + 1e-45).all())
    size = 7 * U * (b1 * m0.double().abs() + (1 - b1) * gs) / M.abs().clamp(min=1e-300)        # m's own error, relative, where its terms cancel
    half = torch.finfo(p.dtype).eps / 2
    tol = (18 * U + size) * upd.abs() + 3 * U * (P.abs() + upd.abs())
    tiny = torch.finfo(p.dtype).smallest_normal * torch.finfo(p.dtype).eps
    assert bool(((p.double() - P).abs() <= tol + half * (P.abs() + tol) + tiny).all())


SIZES = [1, 3, 255, 256, 257, 1023, 1025, 4095, 4096, 4097, 10007]


@pytest.mark.parametrize("dtype,gtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("clip", [None, 0.01, 1e6])
def test_states_in_32_bits(dtype, gtype, clip):
    from esc_gnn_amd import adamw_step
    ts = [make(n, dtype, gtype, 10 + i, off=i % 4) for i, n in enumerate(SIZES)]
    old = [[x.clone() for x in t] for t in ts]
    step = torch.full((1,), 41, dtype=torch.int32, device=DEV)
    kw = dict(lr=3e-3, betas=(0.85, 0.99), eps=1e-6, weight_decay=0.1)
    norm = adamw_step(*zip(*ts), step, max_grad_norm=clip, **kw)
    assert int(step) == 42
    c = 1.0
    if clip is not None:
        want = math.sqrt(sum(float(t[1].double().square().sum()) for t in old))
        assert abs(float(norm) - want) <= 2 * U * want                               # the sum has 64 bits, the result one rounding
        c = min(1.0, clip / (want + 1e-6))
    else:
        assert norm is None
    for new, o in zip(ts, old):
        check32(new[0], new[2], new[3], *o, 42, c, **kw)
        assert torch.equal(new[1], o[1])                                             # the gradient is left as it is


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("clip", [None, 0.02])
def test_states_in_8_bits_are_the_formats_bits(dtype, clip):
    """codes and scales equal, bit for bit, what the format makes of the fp32 moments; parameters as with 32-bit states"""
    from esc_gnn_amd import adamw_step, dequantize_state
    ts = [make(n, dtype, dtype, 50 + i, off=i % 3) for i, n in enumerate(SIZES)]
    half = lambda n: np.full(n, 1 << 15, np.int64)                                   # noqa: E731
    ms, vs = [], []
    for i, (p, g, m, v) in enumerate(ts):
        for x, signed, out in ((m, True, ms), (v, False, vs)):
            c, s = encode8(x.cpu().numpy(), half(x.numel()), signed)
            code = torch.zeros(x.numel() + i % 3, dtype=torch.uint8, device=DEV)[i % 3:]
            code.copy_(torch.from_numpy(c))
            out.append((code, torch.from_numpy(s).to(DEV)))
    old_p = [t[0].clone() for t in ts]
    m0 = [dequantize_state(c, s, True) for c, s in ms]
    v0 = [dequantize_state(c, s, False) for c, s in vs]
    for (c, s), x in zip(ms, m0):
        assert np.array_equal(x.cpu().numpy().astype(np.float64), values8(c, s, True).astype(np.float32).astype(np.float64))
    for (c, s), x in zip(vs, v0):
        assert np.array_equal(x.cpu().numpy().astype(np.float64), values8(c, s, False).astype(np.float32).astype(np.float64))
    step = torch.full((1,), 9, dtype=torch.int32, device=DEV)
    norm = adamw_step([t[0] for t in ts], [t[1] for t in ts], ms, vs, step, max_grad_norm=clip, seed=77)
    c = 1.0
    if clip is not None:
        want = math.sqrt(sum(float(t[1].double().square().sum()) for t in ts))
        assert abs(float(norm) - want) <= 2 * U * want
        c = float(np.float32(min(1.0, clip / (want + 1e-6))))
    f = np.float32
    for i, (p, g, m, v) in enumerate(ts):
        gg = g.float().cpu().numpy() * f(c)
        m1 = m0[i].cpu().numpy() * f(0.9) + gg * f(1 - 0.9)
        v1 = v0[i].cpu().numpy() * f(0.999) + (gg * gg) * f(1 - 0.999)
        r = noise(77, 10, i, len(gg))
        for x, (code, scale), bits, signed in ((m1, ms[i], r & 0xFFFF, True), (v1, vs[i], r >> 16, False)):
            wc, wsc = encode8(x, bits, signed)
            assert np.array_equal(scale.cpu().numpy(), wsc) and np.array_equal(code.cpu().numpy(), wc), (i, signed)
        check32(p, torch.from_numpy(m1).to(DEV), torch.from_numpy(v1).to(DEV), old_p[i], g, m0[i], v0[i], 10, c)


def test_rounding_of_8_bit_states_is_unbiased_and_within_one_code():
    """4096 equal values per seed, 64 seeds: the mean of the stored values is the value (5 sigma), each within one code"""
    from esc_gnn_amd import adamw_step, dequantize_state, new_state8
    n = 4096
    g = torch.full((n,), 1e-3, device=DEV)
    g[::256] = 1.0                                                                   # fixes every block's scale
    got = []
    for seed in range(64):
        m, v = new_state8(n, DEV), new_state8(n, DEV)
        adamw_step([torch.zeros(n, device=DEV)], [g], [m], [v], torch.zeros(1, dtype=torch.int32, device=DEV), seed=seed)
        got.append((dequantize_state(*m, True), dequantize_state(*v, False)))
    keep = torch.ones(n, dtype=torch.bool, device=DEV); keep[::256] = False
    for k, want in ((0, 0.1 * 1e-3), (1, 0.001 * 1e-6)):
        x = torch.stack([q[k][keep] for q in got]).double()
        assert float((x - want).abs().max()) <= want / 8 * (1 + 1e-5)                # a code is at most 1/8 wide
        sd = float(x.std()) / math.sqrt(x.numel())
        assert abs(float(x.mean()) - want) <= 5 * sd + want * 2.0 ** -16, (k, float(x.mean()), want)


def test_second_moment_in_8_bits_follows_a_falling_gradient():
    """|g| falls by 100 for all but one element of each block: v follows to the new level, as with 32 bits.  (Stationary
    spread of a value on codes d = 1/8 apart that drifts by 1 - b2 a step: sd <= sqrt(d / 2) = 0.25; the mean of 4080 within 0.1)"""
    from esc_gnn_amd import adamw_step, dequantize_state, new_state8
    n = 4096
    m, v, p = new_state8(n, DEV), new_state8(n, DEV), torch.zeros(n, device=DEV)
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    big = torch.ones(n, device=DEV)
    small = torch.full((n,), 0.01, device=DEV); small[::256] = 1.0
    for g, times in ((big, 200), (small, 1500)):
        for _ in range(times):
            adamw_step([p], [g], [m], [v], step, betas=(0.9, 0.99))
    x = dequantize_state(*v, False)
    keep = torch.ones(n, dtype=torch.bool, device=DEV); keep[::256] = False
    assert abs(float(x[keep].mean()) / 1e-4 - 1) < 0.1
    assert float((x[~keep] - 1).abs().max()) < 0.2


def test_what_is_not_finite_stays_with_its_element():
    from esc_gnn_amd import adamw_step, dequantize_state, new_state8
    for bits in (32, 8):
        n = 700
        g = torch.full((n,), 0.5, device=DEV); g[3], g[300], g[301] = float("nan"), float("inf"), -float("inf")
        p = torch.ones(n, device=DEV)
        m, v = (new_state8(n, DEV), new_state8(n, DEV)) if bits == 8 else (torch.zeros(n, device=DEV), torch.zeros(n, device=DEV))
        step = torch.zeros(1, dtype=torch.int32, device=DEV)
        adamw_step([p], [g], [m], [v], step)
        if bits == 8:
            m, v = dequantize_state(*m, True), dequantize_state(*v, False)
        bad = torch.zeros(n, dtype=torch.bool, device=DEV); bad[[3, 300, 301]] = True
        for x in (m, v):
            assert not bool(torch.isfinite(x[bad]).any()) and bool(torch.isfinite(x[~bad]).all())
        assert bool(torch.isnan(p[bad]).all()) and bool(torch.isfinite(p[~bad]).all())


def test_extreme_sizes_of_states():
    """zero gradients keep zero states; the smallest and largest finite gradients stay finite and v never rounds to 0"""
    from esc_gnn_amd import adamw_step, dequantize_state, new_state8
    for g0 in (0.0, 1e-22, 1e-12, 1e18):
        n = 513
        g = torch.full((n,), g0, device=DEV)
        p, m, v = torch.ones(n, device=DEV), new_state8(n, DEV), new_state8(n, DEV)
        step = torch.zeros(1, dtype=torch.int32, device=DEV)
        for _ in range(3):
            adamw_step([p], [g], [m], [v], step, weight_decay=0.0)
        mv, vv = dequantize_state(*m, True), dequantize_state(*v, False)
        assert bool(torch.isfinite(p).all())
        if g0 == 0.0:
            assert not bool(mv.any()) and not bool(vv.any()) and bool((p == 1).all())
        if g0 * g0 * 0.001 >= 2.0 ** -120:
            assert bool((vv > 0).all())


def test_more_tensors_than_a_launch_holds_and_empty_ones():
    from esc_gnn_amd import adamw_step
    ns = [(i * 37) % 211 for i in range(130)]                                        # some are empty
    ts = [make(n, torch.float32, torch.float32, i) for i, n in enumerate(ns)]
    old = [[x.clone() for x in t] for t in ts]
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    norm = adamw_step(*zip(*ts), step, max_grad_norm=0.5)
    want = math.sqrt(sum(float(t[1].double().square().sum()) for t in old))
    assert abs(float(norm) - want) <= 2 * U * want
    for new, o in zip(ts, old):
        check32(new[0], new[2], new[3], *o, 1, min(1.0, 0.5 / (want + 1e-6)))
    empty = torch.zeros(0, device=DEV)
    step.zero_()
    norm = adamw_step([empty], [empty], [empty], [empty], step, max_grad_norm=1.0)
    assert float(norm) == 0.0 and int(step) == 1


def test_no_write_outside_the_tensors():
    from esc_gnn_amd import adamw_step
    for n in (1, 255, 4097):
        bufs = [torch.full((n + 512,), 7.0, device=DEV) for _ in range(4)]
        codes = [torch.full((n + 512,), 7, dtype=torch.uint8, device=DEV) for _ in range(2)]
        nb = -(-n // 256)
        scales = [torch.full((nb + 8,), 7.0, device=DEV) for _ in range(2)]
        cut = lambda b, k=n: b[256:256 + k]                                          # noqa: E731
        step = torch.zeros(1, dtype=torch.int32, device=DEV)
        adamw_step([cut(bufs[0])], [cut(bufs[1])], [cut(bufs[2])], [cut(bufs[3])], step)
        adamw_step([cut(bufs[0])], [cut(bufs[1])], [(cut(codes[0]), scales[0][4:4 + nb])], [(cut(codes[1]), scales[1][4:4 + nb])], step)
        for b in bufs + codes:
            assert bool((b[:256] == 7).all()) and bool((b[256 + n:] == 7).all())
        for s in scales:
            assert bool((s[:4] == 7).all()) and bool((s[4 + nb:] == 7).all())


def test_same_inputs_same_bits_and_another_stream():
    from esc_gnn_amd import adamw_step
    outs = []
    for k in range(3):
        ts = [make(n, torch.float32, torch.float32, i) for i, n in enumerate((100003, 77))]
        step = torch.zeros(1, dtype=torch.int32, device=DEV)
        st = torch.cuda.Stream() if k == 2 else torch.cuda.current_stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            norm = adamw_step(*zip(*ts), step, max_grad_norm=0.1)
        torch.cuda.current_stream().wait_stream(st)
        outs.append([norm, step] + [x for t in ts for x in t])
    for a, b in zip(outs[0], outs[1]):
        assert torch.equal(a, b)
    for a, b in zip(outs[0], outs[2]):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ the optimizer
def _pair(bits=32, **kw):
    from esc_gnn_amd import AdamW
    torch.manual_seed(0)
    a = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in ((33, 7), (300,), (1,), (64, 65))]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    return a, b, AdamW([{"params": a[:2]}, {"params": a[2:], "lr": 5e-3, "betas": (0.8, 0.95)}], state_bits=bits, **kw), \
        torch.optim.AdamW([{"params": b[:2]}, {"params": b[2:], "lr": 5e-3, "betas": (0.8, 0.95)}], lr=kw.get("lr", 1e-3))


def test_optimizer_follows_torchs():
    """ten steps with groups, a clip and a parameter that joins late and pauses.  Each step errs by some 30 u of its update
    (|update| <= 5 lr = 0.025) and 4 u of the parameter: 10 steps stay under 1000 u of max(|p|, 1)"""
    a, b, opt, ref = _pair(max_grad_norm=1.0)
    for it in range(10):
        for i, (x, y) in enumerate(zip(a, b)):
            if i == 1 and (it < 3 or it == 6):
                x.grad = y.grad = None
                continue
            g = torch.randn(x.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(100 * it + i))
            x.grad, y.grad = g.clone(), g.clone()
        want = torch.nn.utils.clip_grad_norm_(b, 1.0)
        ref.step()
        opt.step()
        assert abs(float(opt.grad_norm) - float(want)) <= 1e-5 * float(want)          # torch sums the squares in fp32
        for x, y in zip(a, b):
            # (torch's fp32 norm may be off by its summation error, some 1e-6: it scales m and sqrt(v) alike)
            assert float((x - y).detach().abs().max()) <= 1000 * U * max(1.0, float(y.detach().abs().max()))
    assert int(opt.state[a[0]]["step"]) == 10 and int(opt.state[a[1]]["step"]) == 6


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip_goes_on_with_the_same_bits(bits):
    from esc_gnn_amd import AdamW
    def grads(ps, it):
        for i, x in enumerate(ps):
            x.grad = torch.randn(x.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(100 * it + i)).to(x.dtype)
    ps = [torch.nn.Parameter(torch.randn(n, device=DEV).to(t)) for n, t in ((700, torch.float32), (513, torch.bfloat16), (5, torch.float16))]
    opt = AdamW(ps, state_bits=bits, max_grad_norm=1.0, seed=3)
    for it in range(3):
        grads(ps, it); opt.step()
    saved = {k: v for k, v in opt.state_dict().items()}
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = AdamW(qs, state_bits=bits, max_grad_norm=1.0, seed=3)
    other.load_state_dict(saved)
    for it in range(3, 6):
        grads(ps, it); opt.step()
        grads(qs, it); other.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        for k in opt.state[p]:
            assert torch.equal(opt.state[p][k], other.state[q][k]) and opt.state[p][k].dtype == other.state[q][k].dtype
    with pytest.raises(ValueError):
        AdamW(qs, state_bits=40 - bits).load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_counts_on(bits):
    """replays of a captured step (with eager steps of another optimizer between them) equal eager steps bit for bit"""
    from esc_gnn_amd import AdamW
    def build():
        torch.manual_seed(1)
        ps = [torch.nn.Parameter(torch.randn(n, device=DEV)) for n in (5000, 300)]
        for p in ps:
            p.grad = torch.randn_like(p)
        return ps, AdamW(ps, state_bits=bits, max_grad_norm=1.0)
    ps, opt = build()
    qs, ref = build()
    rs, noise_opt = build()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        opt.step()                                                                   # states exist before the capture
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    ref.step()
    for k in range(4):
        for p, q in zip(ps, qs):
            g = torch.randn(p.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(k))
            p.grad.copy_(g); q.grad.copy_(g)
        graph.replay()
        noise_opt.step()
        ref.step()
        torch.cuda.synchronize()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and int(opt.state[p]["step"]) == k + 2
    assert torch.equal(opt.grad_norm, ref.grad_norm)

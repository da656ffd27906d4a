"""Refusals of the experts' entry points: host checks, made before anything reaches the GPU."""
import pytest
import torch


@pytest.mark.parametrize("kw,error", [
    (dict(), RuntimeError),                                                       # CPU tensor
    (dict(logits=torch.zeros(4)), ValueError),
    (dict(logits=torch.zeros(4, 8, dtype=torch.float64)), ValueError),
    (dict(logits=torch.zeros(4, 0)), ValueError),
    (dict(logits=torch.zeros(4, 1025)), ValueError),
    (dict(k=0), ValueError),
    (dict(k=9), ValueError),
    (dict(logits=torch.zeros(4, 64), k=17), ValueError),
    (dict(score="tanh"), ValueError),
    (dict(groups=3), ValueError),
    (dict(logits=torch.zeros(4, 256), groups=128), ValueError),
    (dict(groups=4, keep_groups=5), ValueError),
    (dict(groups=4, keep_groups=0), ValueError),
    (dict(groups=4, group_top=3), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(bias=torch.zeros(7)), ValueError),
    (dict(bias=torch.zeros(8, dtype=torch.float64)), ValueError),
])
def test_route_experts_refuses(kw, error):
    from esc_gnn_amd import route_experts
    kw = dict(kw)
    logits, k = kw.pop("logits", torch.zeros(4, 8)), kw.pop("k", 2)
    with pytest.raises(error):
        route_experts(logits, k, **kw)


def test_route_library_checks_its_arguments():
    from esc_gnn_amd import _lib
    lib = _lib.load()
    ok = [0, 0, 0, 8, 2, 0, 0, 1, 1, 2, 1, 1.0, 0, 0, 0]
    assert lib.escat_route(*ok) == 0                                              # no rows: nothing to do
    for at, value, code in ((1, 5, -1), (2, -1, -1), (3, 0, -1), (4, 9, -1), (3, 2000, -2), (5, 2, -1), (7, 3, -1), (8, 2, -1), (9, 0, -1), (11, 0.0, -1), (2, 5, -1)):
        bad = list(ok); bad[at] = value
        assert lib.escat_route(*bad) == code, (at, value)
    okb = [0, 0, 0, 8, 2, 0, 1, 1.0, 0, 0, 0, 0, 0]
    assert lib.escat_route_bwd(*okb) == 0
    for at, value in ((1, 3), (2, 4), (4, 0), (5, -1), (7, -1.0)):
        bad = list(okb); bad[at] = value
        assert lib.escat_route_bwd(*bad) == -1, (at, value)


def _mlp(**change):
    from esc_gnn_amd import expert_mlp
    a = dict(x=torch.zeros(5, 6), weights=torch.zeros(5, 2), experts=torch.zeros(5, 2, dtype=torch.int32), w1=torch.zeros(3, 7, 6), b1=torch.zeros(3, 7),
             w2=torch.zeros(3, 4, 7), b2=torch.zeros(3, 4))
    a.update(change)
    return expert_mlp(*a.values())


@pytest.mark.parametrize("change,error", [
    (dict(), RuntimeError),                                                       # CPU tensors
    (dict(x=torch.zeros(5, 8)), ValueError),
    (dict(x=torch.zeros(5, 6, dtype=torch.float64)), ValueError),
    (dict(x=torch.zeros(5, 6, dtype=torch.bfloat16)), ValueError),
    (dict(x=torch.zeros(6)), ValueError),
    (dict(w2=torch.zeros(3, 4, 8)), ValueError),
    (dict(w2=torch.zeros(2, 4, 7)), ValueError),
    (dict(w1=torch.zeros(3, 6, 7).transpose(1, 2)), ValueError),
    (dict(b1=torch.zeros(3, 4)), ValueError),
    (dict(b2=torch.zeros(3, 4, dtype=torch.bfloat16)), ValueError),
    (dict(weights=torch.zeros(5, 3)), ValueError),
    (dict(weights=torch.zeros(5, 2, dtype=torch.bfloat16)), ValueError),
    (dict(weights=torch.zeros(5, 0), experts=torch.zeros(5, 0, dtype=torch.int32)), ValueError),
    (dict(weights=torch.zeros(5, 65), experts=torch.zeros(5, 65, dtype=torch.int32)), ValueError),
    (dict(experts=torch.zeros(5, 2, dtype=torch.int64)), ValueError),
    (dict(x=torch.zeros(5, 0), w1=torch.zeros(3, 7, 0)), ValueError),
])
def test_expert_mlp_refuses(change, error):
    with pytest.raises(error):
        _mlp(**change)


def test_expert_counts_refuses():
    from esc_gnn_amd import expert_counts
    for experts, E in ((torch.zeros(3, dtype=torch.int64), 4), (torch.zeros(3, dtype=torch.int32), 0), (torch.zeros(3, dtype=torch.int32), 1025)):
        with pytest.raises(ValueError):
            expert_counts(experts, E)
    with pytest.raises(RuntimeError):
        expert_counts(torch.zeros(3, dtype=torch.int32), 4)


def test_experts_library_checks_its_arguments():
    import ctypes
    from esc_gnn_amd import _lib
    lib = _lib.load()
    dims = lambda *a: ctypes.addressof(keep.append(_lib.EscatExpertsDims(*a)) or keep[-1])       # noqa: E731
    keep = []
    good = (4, 0, 8, 8, 8, 2, 1)
    assert lib.escat_experts_workspace_bytes(dims(*good), 1, 0) > lib.escat_experts_workspace_bytes(dims(*good), 0, 0) > 0
    for at, value in ((0, -1), (1, 3), (2, 0), (3, 0), (4, 0), (5, 0), (6, 0)):
        bad = list(good); bad[at] = value
        assert lib.escat_experts_workspace_bytes(dims(*bad), 0, 0) == 0
        assert lib.escat_experts_fwd(dims(*bad), *[0] * 11, 0, 0) == -1
    assert lib.escat_experts_fwd(dims(1 << 30, 0, 8, 8, 8, 2, 1), *[0] * 11, 0, 0) == -2
    assert lib.escat_experts_fwd(dims(4, 0, 8, 8, 8, 2000, 1), *[0] * 11, 0, 0) == -2
    assert lib.escat_experts_fwd(dims(4, 1, 8, 4, 8, 2, 1), *[0] * 11, 0, 0) == -2                # bf16 rows of 8 bytes
    assert lib.escat_experts_fwd(dims(*good), *[0] * 11, 0, 0) == -1                              # null pointers
    assert lib.escat_experts_fwd(dims(*good), *[16] * 9, 0, 16, 64, 0) == -3                        # small workspace
    assert lib.escat_experts_fwd(dims(0, 0, 8, 8, 8, 2, 1), *[0] * 11, 0, 0) == 0                 # no rows
    assert lib.escat_experts_bwd(dims(*good), *[16] * 7, 0, 16, 0, 0, 0, 16, 0, 0, 16, 1 << 20, 0) == -1          # db1 without dw1
    assert lib.escat_experts_plan(0, 5, 1, 4, 16, 1 << 20, 0, 0) == -1
    assert lib.escat_experts_plan(16, 5, 1, 4, 16, 8, 0, 0) == -3
    assert lib.escat_experts_plan(16, 1 << 31, 1, 4, 16, 8, 0, 0) == -2
    assert lib.escat_experts_plan(16, 5, 2, 4, 16, 1 << 20, 16, 0) == -1                          # counts of k = 2


def test_head_options_refuse():
    from esc_gnn_amd.train_dp import DPTrainer, NodeExperts, ScatteringHead
    kw = dict(diffusion_kwargs=dict(scales_type="dyadic", J=2, include_lowpass=True))
    with pytest.raises(ValueError):
        DPTrainer(C=3, optimizer="sgd", **kw)
    with pytest.raises(ValueError):
        NodeExperts(8, 2, 3)
    head = ScatteringHead(4, 4, experts=4)
    with pytest.raises(RuntimeError):                                             # CPU tensors
        head(torch.zeros(6, 4), torch.zeros(6, 4), torch.zeros(6, dtype=torch.int64), 1)

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

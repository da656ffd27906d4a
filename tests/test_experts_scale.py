"""route_experts' scale is an fp32 number in the kernels: what is none there is refused on the host."""
import pytest
import torch


@pytest.mark.parametrize("scale", [1e39, 1e-46, 5e-324, float("inf"), -1.0])
def test_a_scale_that_fp32_does_not_hold_is_refused(scale):
    from esc_gnn_amd import route_experts
    with pytest.raises(ValueError, match="scale"):
        route_experts(torch.zeros(4, 8), 2, scale=scale)


@pytest.mark.parametrize("scale", [1e38, 1e-37, 2.5])
def test_others_are_not(scale):
    from esc_gnn_amd import route_experts
    with pytest.raises(RuntimeError):                                             # (CPU tensors: the next check)
        route_experts(torch.zeros(4, 8), 2, scale=scale)


def test_the_library_refuses_an_infinite_scale():
    from esc_gnn_amd import _lib
    lib = _lib.load()
    for scale in (float("inf"), float("nan"), 0.0):
        assert lib.escat_route(0, 0, 0, 8, 2, 0, 0, 1, 1, 2, 1, scale, 0, 0, 0) == -1
        assert lib.escat_route_bwd(0, 0, 0, 8, 2, 0, 1, scale, 0, 0, 0, 0, 0) == -1

"""GPU tests of the load that NodeExperts counts for its balance bias (train_dp.py), with captured forwards too."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_replayed_forwards_count():
    """a captured training forward counts its nodes at every replay, before and after update_balance, which the eager code calls"""
    from esc_gnn_amd.train_dp import NodeExperts
    torch.manual_seed(3)
    layer = NodeExperts(16, 4, 2).to(DEV)
    x = torch.randn(500, 16, device=DEV)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x)
        torch.cuda.current_stream().wait_stream(side)
        one = layer.load.clone()
        assert int(one.sum()) == 1000
        layer.update_balance()
        layer.balance.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer(x)
        assert not bool(layer.load.any())
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layer.load, 3 * one)
        want = layer.rate * torch.sign(one.float().mean() - one.float())
        layer.update_balance()
        assert torch.equal(layer.balance, want) and not bool(layer.load.any())
        kept = layer.load
        graph.replay()
        torch.cuda.synchronize()
        assert layer.load is kept and int(layer.load.sum()) == 1000

"""one rank of tests/test_gpu_train_experts.py: three DPTrainer steps with experts and 8-bit states on its half of a batch"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def main(out):
    import torch.distributed as dist
    from test_gpu_train_experts import batch
    from esc_gnn_amd.train_dp import DPTrainer
    world, rank = int(os.environ["WORLD_SIZE"]), int(os.environ["RANK"])
    torch.cuda.set_device(0)
    if world > 1:
        dist.init_process_group("gloo")
    torch.manual_seed(0)
    tr = DPTrainer(C=3, diffusion_kwargs=dict(scales_type="dyadic", J=3, include_lowpass=True), device="cuda:0", experts=6, optimizer=sys.argv[2], max_grad_norm=1.0)
    data = batch(seed=3 + rank)
    for _ in range(3):
        tr.step(*data)
    torch.cuda.synchronize()
    torch.save({n: v.cpu() for n, v in tr.model.state_dict().items()}, out)
    if world > 1:
        dist.destroy_process_group()


if __name__ == "__main__":
    main(sys.argv[1])

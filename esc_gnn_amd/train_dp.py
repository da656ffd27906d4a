"""
Minimal data-parallel ESc-GNN training step.

What a step does, per rank (one process per GPU, graphs sharded, RCCL only for the gradients):
  1. orders-0/1/2 scattering of both tracks on the rank's batch -- esc_gnn_amd.scatter (the hot path; like the
     reference, x and the operators carry no grad, so the chain sits outside the autograd graph,
     training/train.py:303-321, models/escgnn_modular.py:674-685);
  2. the vector track's invariants for track mixing -- esc_gnn_amd.invariants.get_vector_invariants
     (models/escgnn_modular.py:403-504: per-wavelet norms + pooled neighbour cosines), then a small head on
     [scalar coefficients | invariants] (~1e5 parameters like the reference's mixers + readout), graph-mean readout,
     MSE loss;
  3. backward into ONE flat fp32 gradient bucket, one all-reduce (sum) / world, AdamW step.
Optional (off by default): `experts` = E widens the head at the cost per node of k of its E small MLPs (route_experts +
expert_mlp, kept in balance by a selection bias that an all-reduce of E counts follows); `optimizer` = "escat" / "escat8" takes the multi-tensor AdamW of
esc_gnn_amd.optim with states in 32 / 8 bits; `max_grad_norm` clips as the reference does (training/train.py:411-415).
The reference gets 3 from Accelerate/DDP (training/train.py:408, :483-492); the heads themselves are plain PyTorch
but for the optional operators.
"""
from typing import Dict
import torch
import torch.nn as nn

from .dist_utils import FlatGradBucket, allreduce_sum_
from .experts import expert_counts, expert_mlp, route_experts
from .optim import AdamW
from .scatter import scatter
from .invariants import get_vector_invariants


class NodeExperts(nn.Module):
    """x + sum over a node's k experts: a router (softmax over the chosen, selection steered by a balance bias) and the
    experts' MLPs.  `balance` follows the load: after a step, update_balance() raises the bias of the experts that got fewer
    nodes than the mean and lowers the others' by `rate` (it only steers the choice: no gradient, no part in the weights)."""

    def __init__(self, width: int, n_experts: int, per_node: int = 2, hidden: int = None, rate: float = 1e-3):
        super().__init__()
        hidden = hidden or width
        if not 1 <= per_node <= n_experts:
            raise ValueError(f"escat: {per_node} of {n_experts} experts per node")
        u = lambda fan_in, *shape: nn.Parameter(torch.empty(*shape).uniform_(-fan_in ** -0.5, fan_in ** -0.5))       # noqa: E731
        self.per_node, self.rate = per_node, rate
        self.router = nn.Linear(width, n_experts, bias=False)
        self.w1, self.b1 = u(width, n_experts, hidden, width), u(width, n_experts, hidden)
        self.w2, self.b2 = u(hidden, n_experts, width, hidden), u(hidden, n_experts, width)
        self.register_buffer("balance", torch.zeros(n_experts))
        self.register_buffer("load", torch.zeros(n_experts, dtype=torch.int32), persistent=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        with torch.autocast("cuda", enabled=False):                       # which expert is decided in fp32
            logits = nn.functional.linear(x.float(), self.router.weight.float())
        weights, experts = route_experts(logits, self.per_node, bias=self.balance)
        if self.training:
            self.load += expert_counts(experts, self.balance.numel())        # in place: a captured forward goes on counting here
        return x + expert_mlp(x, weights, experts, self.w1, self.b1, self.w2, self.b2)

    @torch.no_grad()
    def update_balance(self):
        load = allreduce_sum_(self.load).float()
        self.balance += self.rate * torch.sign(load.mean() - load)
        self.load.zero_()


class ScatteringHead(nn.Module):
    def __init__(self, n_scalar_feats: int, n_vector_feats: int, hidden: int = 256, experts: int = 0, experts_per_node: int = 2):
        super().__init__()
        self.bn = nn.BatchNorm1d(n_scalar_feats + n_vector_feats)
        middle = [nn.Linear(hidden, hidden), nn.SiLU()] if experts == 0 else [NodeExperts(hidden, experts, experts_per_node)]
        self.mlp = nn.Sequential(nn.Linear(n_scalar_feats + n_vector_feats, hidden), nn.SiLU(), *middle, nn.Linear(hidden, 1))

    def forward(self, Ws: torch.Tensor, inv: torch.Tensor, graph_id: torch.Tensor, n_graphs: int) -> torch.Tensor:
        N = Ws.shape[0]
        feats = torch.cat([Ws.reshape(N, -1), inv], dim=1)                             # (N, C*W + W*(1+m))
        y = self.mlp(self.bn(feats)).squeeze(-1).float()
        out = torch.zeros(n_graphs, device=y.device, dtype=y.dtype).index_add_(0, graph_id, y)
        cnt = torch.zeros(n_graphs, device=y.device, dtype=y.dtype).index_add_(0, graph_id, torch.ones_like(y))
        return out / cnt.clamp(min=1)


class DPTrainer:
    POOL_STATS = ('percentiles', 'min', 'max', 'mean')        # the reference's default neighbor_kwargs (:431-434)

    def __init__(self, C: int, diffusion_kwargs: Dict, lr: float = 1e-3, device=None, amp_bf16: bool = False, experts: int = 0,
                 experts_per_node: int = 2, optimizer: str = "torch", max_grad_norm: float = None):
        from .scales import plan_chain
        from .invariants import quantile_levels
        F = plan_chain(**{k: v for k, v in diffusion_kwargs.items()}).F
        W = 1 + F + F * (F - 1) // 2
        m = 3 + len(quantile_levels(0.2))
        self.kw = {"diffusion_kwargs": diffusion_kwargs}
        self.amp_bf16 = amp_bf16          # head GEMMs in bf16 (Accelerate's mixed_precision='bf16'); scattering stays fp32
        if optimizer not in ("torch", "escat", "escat8"):
            raise ValueError(f"escat: optimizer must be 'torch', 'escat' or 'escat8': {optimizer!r}")
        self.model = ScatteringHead(C * W, W * (1 + m), experts=experts, experts_per_node=experts_per_node).to(device)
        self.bucket = FlatGradBucket(self.model.parameters())
        self.max_grad_norm = max_grad_norm
        if optimizer == "torch":
            self.opt = torch.optim.AdamW(self.model.parameters(), lr=lr)
        else:
            self.opt = AdamW(self.model.parameters(), lr=lr, state_bits=8 if optimizer == "escat8" else 32, max_grad_norm=max_grad_norm)

    def n_params(self) -> int:
        return self.bucket.flat.numel()

    def step(self, x_s, x_v, P, Q, graph_id, n_graphs, target, edge_index) -> float:
        with torch.no_grad():
            Ws = scatter(track="scalar", x0=x_s, P_or_Q=P, kwargs=self.kw)               # (N, C, W)
            Wv = scatter(track="vector", x0=x_v, P_or_Q=Q, kwargs=self.kw)               # (N, 1, 3, W)
            inv = get_vector_invariants(Wv.permute(0, 3, 1, 2).contiguous(), edge_index, self.POOL_STATS, 0.2)   # (N, W', 1, d) in
        self.bucket.zero()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=self.amp_bf16):
            pred = self.model(Ws, inv, graph_id, n_graphs)
        loss = torch.nn.functional.mse_loss(pred.float(), target)
        loss.backward()                       # grads land in the flat bucket (p.grad are views of it)
        self.bucket.allreduce_mean()          # the step's only collective but for the experts' loads below
        if self.max_grad_norm is not None and isinstance(self.opt, torch.optim.AdamW):
            torch.nn.utils.clip_grad_norm_(self.model.parameters(), self.max_grad_norm)
        self.opt.step()
        for m in self.model.mlp:
            if isinstance(m, NodeExperts):
                m.update_balance()
        return loss

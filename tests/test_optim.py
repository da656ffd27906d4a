"""Refusals of the AdamW entry points: all of them are host checks, made before anything reaches the GPU."""
import pytest
import torch


def _call(n=5, **change):
    from esc_gnn_amd import adamw_step
    a = dict(params=[torch.zeros(n)], grads=[torch.zeros(n)], exp_avgs=[torch.zeros(n)], exp_avg_sqs=[torch.zeros(n)],
             step=torch.zeros(1, dtype=torch.int32))
    kw = dict(lr=1e-3)
    for k, v in change.items():
        (a if k in a else kw)[k] = v
    return adamw_step(*a.values(), **kw)


@pytest.mark.parametrize("change,error", [
    (dict(), RuntimeError),                                                        # CPU tensors
    (dict(params=[torch.zeros(5), torch.zeros(5)]), ValueError),
    (dict(step=torch.zeros(1)), ValueError),
    (dict(step=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(lr=-1.0), ValueError),
    (dict(lr=torch.tensor(1e-3)), TypeError),
    (dict(betas=(1.0, 0.9)), ValueError),
    (dict(eps=float("nan")), ValueError),
    (dict(max_grad_norm=0.0), ValueError),
    (dict(grads=[torch.zeros(4)]), ValueError),
    (dict(params=[torch.zeros(5, dtype=torch.float64)]), TypeError),
    (dict(grads=[torch.zeros(5, dtype=torch.bfloat16)]), TypeError),               # fp32 parameter, bf16 gradient
    (dict(grads=[torch.zeros(5).to_sparse()]), ValueError),
    (dict(params=[torch.zeros(5, 2).t()], grads=[torch.zeros(2, 5)], exp_avgs=[torch.zeros(10)], exp_avg_sqs=[torch.zeros(10)]), ValueError),
    (dict(exp_avgs=[torch.zeros(5, dtype=torch.bfloat16)]), ValueError),
    (dict(exp_avgs=[torch.zeros(4)]), ValueError),
    (dict(exp_avgs=[(torch.zeros(5, dtype=torch.uint8), torch.zeros(1))]), ValueError),          # one 8-bit, one 32-bit moment
    (dict(exp_avgs=[(torch.zeros(5, dtype=torch.uint8), torch.zeros(2))], exp_avg_sqs=[(torch.zeros(5, dtype=torch.uint8), torch.zeros(1))]), ValueError),
    (dict(exp_avgs=[(torch.zeros(5, dtype=torch.int8), torch.zeros(1))], exp_avg_sqs=[(torch.zeros(5, dtype=torch.uint8), torch.zeros(1))]), ValueError),
])
def test_adamw_step_refuses(change, error):
    with pytest.raises(error):
        _call(**change)


def test_adamw_refuses_a_tensor_listed_twice():
    from esc_gnn_amd import adamw_step
    p, z = torch.zeros(5), lambda: torch.zeros(5)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([p, p], [z(), z()], [z(), z()], [z(), z()], torch.zeros(1, dtype=torch.int32))
    m = z()
    with pytest.raises(ValueError, match="twice"):
        adamw_step([z(), z()], [z(), z()], [m, m], [z(), z()], torch.zeros(1, dtype=torch.int32))


def test_optimizer_refuses():
    from esc_gnn_amd import AdamW, dequantize_state
    p = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(state_bits=16), dict(max_grad_norm=-1.0), dict(lr=-1.0), dict(betas=(0.9, 1.0))):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    opt = AdamW([p])
    opt.step()                                            # no gradient anywhere: nothing to do
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError):
        opt.step()
    with pytest.raises(ValueError):
        dequantize_state(torch.zeros(300, dtype=torch.uint8), torch.zeros(1), True)
    with pytest.raises(RuntimeError):
        dequantize_state(torch.zeros(300, dtype=torch.uint8), torch.zeros(2), True)


def test_library_checks_its_arguments():
    from esc_gnn_amd import _lib
    lib = _lib.load()
    z = 0
    assert lib.escat_adamw_begin(z, -1, 0, 0.0, 0, 1, z, 0, z, z, z, 0, z) == -1
    assert lib.escat_adamw_begin(z, 0, 7, 0.0, 0, 1, z, 0, z, z, z, 0, z) == -1
    assert lib.escat_adamw_begin(z, 0, 0, 0.0, 0, 1, z, 0, z, z, z, 0, z) == -3
    assert lib.escat_adamw_begin(z, 0, 0, 0.0, 0, 1, z, 0, z, z, 8, 256, z) == -1                  # no group
    assert lib.escat_adamw_update(z, 0, 0, 1, 32, z, 0, 0, z, z, z) == -1                          # fp32 parameter, bf16 gradient
    assert lib.escat_adamw_update(z, 0, 0, 0, 16, z, 0, 0, z, z, z) == -1
    assert lib.escat_state8_values(z, z, 5, 1, z, z) == -1
    assert lib.escat_state8_values(z, z, 0, 1, z, z) == 0
    assert lib.escat_adamw_workspace_bytes(1) < lib.escat_adamw_workspace_bytes(1000)

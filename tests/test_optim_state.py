"""State dicts that the optimizer takes and refuses: host work, no GPU."""
import copy
import pytest
import torch


def _torch_dict(kind=torch.optim.AdamW, steps=100, dtype=torch.float32, **kw):
    ps = [torch.nn.Parameter(torch.ones(n, dtype=dtype)) for n in (3, 300)]
    opt = kind(ps, lr=2e-3, **kw)
    for _ in range(steps):
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
    return ps, opt.state_dict()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_torchs_state_dict_is_taken_as_what_it_means(dtype):
    """torch counts steps in fp32 and holds the moments in the parameter's type: here int32 and fp32, the values the same"""
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(dtype=dtype)
    opt = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps])
    opt.load_state_dict(copy.deepcopy(saved))
    assert opt.param_groups[0]["lr"] == 2e-3
    for i, p in enumerate(opt.param_groups[0]["params"]):
        st = opt.state[p]
        assert set(st) == {"step", "exp_avg", "exp_avg_sq"}
        assert st["step"].dtype is torch.int32 and st["step"].shape == (1,) and int(st["step"]) == 100
        for name in ("exp_avg", "exp_avg_sq"):
            assert st[name].dtype is torch.float32 and torch.equal(st[name], saved["state"][i][name].float())
    assert opt.state[opt.param_groups[0]["params"][0]]["step"] is opt.state[opt.param_groups[0]["params"][1]]["step"]


def test_a_count_may_be_a_number_and_must_be_a_whole_one():
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(steps=3)
    saved["state"][0]["step"] = 3
    opt = AdamW(ps)
    opt.load_state_dict(saved)
    assert int(opt.state[ps[0]]["step"]) == 3
    for bad in (2.5, -1, float("nan"), 2 ** 31, torch.zeros(2)):
        saved["state"][0]["step"] = bad
        with pytest.raises(ValueError, match="step"):
            opt.load_state_dict(saved)
        assert int(opt.state[ps[0]]["step"]) == 3                                  # a refused load changes nothing


@pytest.mark.parametrize("kind,kw", [(torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.AdamW, dict(maximize=True)),
                                     (torch.optim.Adam, dict(weight_decay=0.1)), (torch.optim.SGD, dict(momentum=0.9)), (torch.optim.RAdam, dict(weight_decay=0.1))])
def test_states_of_another_step_are_refused(kind, kw):
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(kind, 2, **kw)
    opt = AdamW(ps, lr=7e-3)
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 7e-3 and not opt.state


def test_plain_adam_without_decay_is_the_same_step():
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(torch.optim.Adam, 2)
    opt = AdamW(ps)
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["weight_decay"] == 0 and int(opt.state[ps[0]]["step"]) == 2


def test_missing_or_wrong_entries_are_refused():
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(steps=2)
    opt = AdamW(ps)
    for change in (lambda st: st.pop("exp_avg_sq"), lambda st: st.update(exp_avg=torch.zeros(4)), lambda st: st.pop("step")):
        other = copy.deepcopy(saved)
        change(other["state"][0])
        with pytest.raises(ValueError):
            opt.load_state_dict(other)


def test_torch_takes_this_optimizers_state_dict():
    """the other way: the names and values are what torch's AdamW reads"""
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(steps=4)
    mine = AdamW(ps, lr=2e-3)
    mine.load_state_dict(copy.deepcopy(saved))
    outs = []
    for source in (saved, mine.state_dict()):
        qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        opt = torch.optim.AdamW(qs, lr=2e-3)
        opt.load_state_dict(copy.deepcopy(source))
        for q in qs:
            q.grad = torch.full_like(q, 0.3)
        opt.step()
        assert all(float(opt.state[q]["step"]) == 5 for q in qs)
        outs.append(qs)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def _copies():
    import io
    import pickle

    def by_torch(o):
        f = io.BytesIO(); torch.save(o, f); f.seek(0)
        return torch.load(f, weights_only=False)                                   # (written two lines above)
    return [("deepcopy", copy.deepcopy), ("pickle", lambda o: pickle.loads(pickle.dumps(o))), ("torch.save", by_torch)]


@pytest.mark.parametrize("how", _copies(), ids=lambda h: h[0])
def test_a_copy_keeps_its_settings(how):
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(steps=2)
    opt = AdamW(ps, max_grad_norm=0.5, seed=11)
    opt.load_state_dict(saved)
    other = how[1](opt)
    assert (other.state_bits, other.max_grad_norm, other.seed, other.grad_norm) == (32, 0.5, 11, None)
    qs = other.param_groups[0]["params"]
    assert other.state[qs[0]]["step"] is other.state[qs[1]]["step"] and int(other.state[qs[0]]["step"]) == 2
    assert other.state[qs[0]]["step"] is not opt.state[ps[0]]["step"]
    other.load_state_dict(opt.state_dict())                                        # (loading leaves the settings alone)
    assert (other.state_bits, other.max_grad_norm, other.seed) == (32, 0.5, 11)


def test_adamw_refuses_scales_and_a_count_that_are_listed_twice():
    """states of two tensors, or of both moments, that share their scales; a count that is one of the states"""
    from esc_gnn_amd import adamw_step
    z, c = lambda n=300: torch.zeros(n), lambda: torch.zeros(300, dtype=torch.uint8)     # noqa: E731
    s, step = torch.zeros(2), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([z()], [z()], [(c(), s)], [(c(), s)], step)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([z(), z()], [z(), z()], [(c(), s), (c(), s)], [(c(), z(2)), (c(), z(2))], step)
    one = torch.zeros(1)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([one], [z(1)], [z(1)], [z(1)], one.view(torch.int32))
    g = z()
    with pytest.raises(ValueError, match="twice"):
        adamw_step([z()], [g], [g], [z()], step)                                      # a gradient that the step would write


def test_a_count_in_the_dict_is_as_torch_keeps_it():
    from esc_gnn_amd import AdamW
    ps, saved = _torch_dict(steps=4)
    for n in (4, 2 ** 24, 2 ** 24 + 1, 2 ** 31 - 1):
        saved["state"][0]["step"] = saved["state"][1]["step"] = n
        opt = AdamW(ps)
        opt.load_state_dict(saved)
        out = opt.state_dict()["state"]
        for st in out.values():
            assert st["step"].shape == () and st["step"].device.type == "cpu" and st["step"].dtype is (torch.float32 if n <= 2 ** 24 else torch.float64)
            assert int(st["step"]) == n
        assert out[0]["step"] is not out[1]["step"] and out[0]["exp_avg"] is opt.state[ps[0]]["exp_avg"]
        again = AdamW(ps)
        again.load_state_dict(opt.state_dict())
        assert int(again.state[ps[0]]["step"]) == n and again.state[ps[0]]["step"].dtype is torch.int32

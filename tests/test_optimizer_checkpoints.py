"""Loading optimizer states as torch.optim.Optimizer does: hooks, types (CPU)."""
import copy

import pytest
import torch

from zorse_amd import optim


def _saved(bits=32, dt=torch.float32):
    """(parameter, state dict) after a step: moments 0.5 and 2."""
    p = torch.nn.Parameter(torch.ones(6, dtype=dt))
    opt = optim.FusedAdamW([p], state_bits=bits)
    st = opt._init_state(p)
    st["step"] = 3
    st["exp_avg"].fill_(0.5 if bits == 32 else 5)
    st["exp_avg_sq"].fill_(2)
    return p, opt.state_dict()


@pytest.mark.parametrize("in_place", [False, True])
def test_pre_hooks_decide_what_is_loaded(in_place):
    p, saved = _saved()

    def tenfold(opt, sd):
        state = {k: {**v, "exp_avg": v["exp_avg"] * 10} for k, v in sd["state"].items()}
        if in_place:  # the dictionary is torch's own copy
            sd["state"] = state
            return None
        return {**sd, "state": state}

    opt = optim.FusedAdamW([p])
    opt.register_load_state_dict_pre_hook(tenfold)
    opt.load_state_dict(saved)
    assert bool((opt.state[p]["exp_avg"] == 5.0).all()) and opt.state[p]["step"] == 3
    assert bool((saved["state"][0]["exp_avg"] == 0.5).all())
    opt.load_state_dict(saved)  # again: no hook of the load itself stays behind
    assert bool((opt.state[p]["exp_avg"] == 5.0).all())
    assert len(opt._optimizer_load_state_dict_pre_hooks) == 1
    assert len(opt._optimizer_load_state_dict_post_hooks) == 0


def test_pre_hooks_may_convert_other_moments():
    """A checkpoint of another width that a hook makes fit is not refused; one
    that a hook makes unfit is, and leaves the optimizer alone."""
    p, narrow = _saved(8)
    _, wide = _saved(32)
    opt = optim.FusedAdamW([p])
    with pytest.raises(ValueError, match="state_bits"):
        opt.load_state_dict(narrow)
    assert not opt.state and not opt._optimizer_load_state_dict_pre_hooks
    hook = opt.register_load_state_dict_pre_hook(lambda o, sd: copy.deepcopy(wide))
    opt.load_state_dict(narrow)
    assert bool((opt.state[p]["exp_avg"] == 0.5).all())
    hook.remove()
    opt.register_load_state_dict_pre_hook(lambda o, sd: copy.deepcopy(narrow))
    with pytest.raises(ValueError, match="state_bits"):
        opt.load_state_dict(wide)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_post_hooks_find_and_change_the_state(dt):
    p, saved = _saved(dt=dt)
    seen = []

    def halve(opt):
        seen.append(opt.state[p]["exp_avg"].dtype)
        opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"] / 2

    opt = optim.FusedAdamW([p])
    opt.register_load_state_dict_post_hook(halve)
    opt.load_state_dict(saved)
    assert seen == [torch.float32]
    assert bool((opt.state[p]["exp_avg"] == 0.25).all())
    assert opt.state[p]["exp_avg"].dtype == torch.float32


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("param", [torch.float32, torch.bfloat16])
def test_moments_saved_in_another_float_type(dt, param):
    """As torch casts them for fp32 parameters; fp32 for 16-bit ones too."""
    p, saved = _saved(dt=param)
    st = saved["state"][0] = dict(saved["state"][0])
    for k in ("exp_avg", "exp_avg_sq", "master"):
        if k in st:
            st[k] = torch.linspace(0.1, 1, 6).to(dt)
    opt = optim.FusedAdamW([p])
    opt.load_state_dict(saved)
    for k in ("exp_avg", "exp_avg_sq", "master"):
        if k in st:
            got = opt.state[p][k]
            assert got.dtype == torch.float32 and torch.equal(got, st[k].float())
    if param == torch.float32:
        theirs = torch.optim.Adam([p])
        theirs.load_state_dict(saved)
        assert torch.equal(theirs.state[p]["exp_avg"], opt.state[p]["exp_avg"])


def test_seeds_of_counts_that_are_tensors():
    """torch's own optimizers save the step count as a tensor."""
    p, _ = _saved(8)
    opt = optim.FusedAdamW([p, torch.nn.Parameter(torch.ones(2))], state_bits=8)
    group = opt.param_groups[0]
    want = opt._seeds(group, group["params"], [3, 70000])
    for dt in (torch.float32, torch.int64):
        counts = [torch.tensor(n, dtype=dt) for n in (3, 70000)]
        assert opt._seeds(group, group["params"], counts) == want


def test_layers_round_with_bits_of_their_own():
    """The one parameter of each layer's optimizer has the same place in it; the
    seed is saved, and checkpoints without one repeat what they began with."""
    from zorse_amd.stage import StageRunner
    layers = [torch.nn.Linear(3, 3, bias=False) for _ in range(3)]
    stage = StageRunner(layers, state_bits=8)
    later = StageRunner(layers, state_bits=8, seed=3)

    def seeds(opt, step=5):
        group = opt.param_groups[0]
        return opt._seeds(group, group["params"], [step])[0]

    opts = stage.optimizers + later.optimizers
    drawn = {seeds(o, t) for o in opts for t in range(1, 50)}
    assert len(drawn) == 6 * 49
    first, other = stage.optimizers[:2]
    alone = optim.FusedAdamW(list(layers[0].parameters()), state_bits=8)
    assert seeds(first) == seeds(alone) == (5 * 0xC2B2AE3D) & 0xFFFFFFFF
    alone.load_state_dict(other.state_dict())
    assert seeds(alone) == seeds(other) != seeds(first)
    old = other.state_dict()
    del old["param_groups"][0]["seed"]
    other.load_state_dict(old)
    assert seeds(other) == seeds(first)
    with pytest.raises(TypeError):
        optim.FusedAdamW(layers[0].parameters(), state_bits=8, seed=1.5)
    wide = optim.FusedAdam(list(layers[0].parameters()))
    assert "seed" not in wide.param_groups[0]
    assert optim.FusedAdam(layers[0].parameters(), state_bits=8, seed=7).param_groups[0]["seed"] == 7


@pytest.mark.gpu
def test_seeds_change_the_second_moment_alone(dev):
    """Equal layers with equal gradients: other roundings, with another seed."""
    g = torch.linspace(1e-3, 1, 5000, device=dev)
    state = []
    for seed in (0, 0, 1):
        p = torch.nn.Parameter(torch.ones_like(g))
        opt = optim.FusedAdamW([p], state_bits=8, seed=seed)
        p.grad = g.clone()
        opt.step()
        state.append((p.detach(), *opt.moments(p)))
    for a, b in zip(state[0], state[1]):
        assert torch.equal(a, b)
    assert torch.equal(state[0][0], state[2][0]) and torch.equal(state[0][1], state[2][1])
    # rounded apart where a draw lies between the fraction's two sides: a third
    # of the elements on average
    apart = int((state[0][2] != state[2][2]).sum())
    assert 1000 < apart < 2500

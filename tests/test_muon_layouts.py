"""Muon's layouts of parameters, its arguments and its saved states (CPU)."""
import copy

import pytest
import torch

from zorse_amd import llama_simple, optim


def _layer(dtype=torch.float32):
    cfg = llama_simple.llama_config(hidden_size=64, num_attention_heads=4, num_key_value_heads=2,
                                    intermediate_size=96, rope_theta=1e4)
    return llama_simple.LlamaDecoderLayer(cfg, 0, param_dtype=dtype)


def test_a_layer_s_matrices():
    layer = _layer()
    mats = optim.flat_matrices(layer)
    assert [m[1:] for m in mats] == [(64, 64), (32, 64), (32, 64), (64, 64), (96, 64), (96, 64), (64, 96)]
    for (a, r, c), name in zip(mats, ("q", "k", "v", "o", "gate", "up", "down")):
        view = layer.param_view(name)
        assert view.data_ptr() == layer.flat_param.data_ptr() + 4 * a and view.shape == (r, c)
    opt = optim.Muon([layer.flat_param], matrices=mats)
    where, rest = opt._layout(opt.param_groups[0], layer.flat_param)
    assert where == mats and rest == [(layer.spec.numel - 128, 128)]
    st = opt._init_state(layer.flat_param)
    assert st["momentum_buffer"].numel() == layer.spec.numel - 128 and st["exp_avg"].numel() == 128
    with pytest.raises(ValueError, match="one flat parameter"):
        optim.flat_matrices(torch.nn.Linear(2, 2))


def test_layouts():
    w, b, t = (torch.nn.Parameter(torch.zeros(s)) for s in ((4, 6), (5,), (2, 3, 4)))
    opt = optim.Muon([{"params": [w, b, t]}, {"params": [torch.nn.Parameter(torch.zeros(7, 3))],
                                              "matrices": []}])
    g = opt.param_groups[0]
    assert opt._layout(g, w) == ([(0, 4, 6)], [])
    assert opt._layout(g, b) == ([], [(0, 5)]) and opt._layout(g, t) == ([], [(0, 24)])
    g = opt.param_groups[1]
    assert opt._layout(g, g["params"][0]) == ([], [(0, 21)])
    for bad in ([(0, 3, 3), (8, 2, 2)], [(15, 2, 4)], [(-1, 2, 2)], [(0, -2, -2)]):
        with pytest.raises(ValueError, match="overlap or leave"):
            optim.Muon([torch.nn.Parameter(torch.zeros(20))], matrices=bad)
    with pytest.raises(ValueError, match="overlap or leave"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))], "matrices": [(0, 2, 2)]})
    assert len(opt.param_groups) == 2


def test_arguments():
    p = [torch.nn.Parameter(torch.zeros(3, 3))]
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-1.0), dict(adjust="x"),
               dict(adam_betas=(1.0, 0.9)), dict(adam_eps=-1.0), dict(adam_lr=-0.1), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            optim.Muon(p, **kw)
    with pytest.raises(TypeError):
        optim.Muon(p, ns_steps=2.5)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_saved_states_load_again(dt):
    layer = _layer(dt)
    opt = optim.Muon([layer.flat_param], matrices=optim.flat_matrices(layer))
    st = opt._init_state(layer.flat_param)
    st["step"] = 4
    for i, k in enumerate(("momentum_buffer", "exp_avg", "exp_avg_sq")):
        st[k].fill_(i + 0.5)
    saved = copy.deepcopy(opt.state_dict())
    other = optim.Muon([layer.flat_param], matrices=optim.flat_matrices(layer))
    half = {**saved, "state": {0: {k: v.half() if torch.is_tensor(v) else v
                                   for k, v in saved["state"][0].items()}}}
    other.load_state_dict(half)
    new = other.state[layer.flat_param]
    assert new["step"] == 4
    for i, k in enumerate(("momentum_buffer", "exp_avg", "exp_avg_sq")):
        assert new[k].dtype == torch.float32 and bool((new[k] == i + 0.5).all())
    assert ("master" in new) == (dt != torch.float32)
    adam = optim.FusedAdamW([layer.flat_param])
    adam._init_state(layer.flat_param)
    with pytest.raises(ValueError, match="not Muon's"):
        other.load_state_dict(adam.state_dict())


def test_cpu_parameters_are_refused():
    p = torch.nn.Parameter(torch.zeros(3, 3))
    p.grad = torch.zeros(3, 3)
    opt = optim.Muon([p])
    with pytest.raises(ValueError, match="GPU tensors"):
        opt.step()
    assert opt.state[p]["step"] == 0


@pytest.mark.parametrize("name,more", [("momentum_buffer", 3), ("momentum_buffer", -1), ("exp_avg", 4),
                                       ("exp_avg_sq", -2), ("master", 8)])
def test_a_state_of_another_size_is_refused(name, more):
    layer = _layer(torch.bfloat16)
    p = layer.flat_param
    opt = optim.Muon([p], matrices=optim.flat_matrices(layer))
    opt._init_state(p)
    saved = copy.deepcopy(opt.state_dict())
    saved["state"][0][name] = torch.ones(saved["state"][0][name].numel() + more)
    opt.load_state_dict(saved)
    p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError, match=name):
        opt.step()
    assert opt.state[p]["step"] == 0

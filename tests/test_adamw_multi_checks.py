"""What the steps over lists of tensors refuse, before any launch (CPU), and
the optimizer's handling of their states."""
import ctypes

import pytest
import torch

from zorse_amd import _abi, kernels, optim

HYPER = (1e-3, 0.9, 0.999, 1e-8, 0.0)


def _table(*rows):
    flat = [v for r in rows for v in r]
    return (ctypes.c_int64 * max(1, len(flat)))(*flat)


def test_entry_points_refuse():
    lib = _abi.lib()
    #       param grad  m    v   lowp  n step g  low
    good = [256, 256, 256, 256, 256, 0, 1, 2, 2]

    def at(i, v, row=good):
        return [*row[:i], v, *row[i + 1:]]

    def multi(*rows, hyper=HYPER):
        return lib.zk_adamw_multi(_table(*rows), len(rows), *hyper, None)

    assert multi(good) == 0 and multi() == 0  # nothing to step: no launch
    assert lib.zk_adamw_multi(None, 1, *HYPER, None) == -1
    assert lib.zk_adamw_multi(None, -1, *HYPER, None) == -1
    assert multi(good, at(6, 0)) == -1 and multi(at(5, -1)) == -1
    assert multi(at(7, 3)) == -2 and multi(at(8, -1)) == -2 and multi(at(8, -1, at(4, 0))) == 0
    assert multi(at(0, 0, at(5, 8))) == -1 and multi(at(3, 0, at(5, 8))) == -1
    assert multi(at(0, 258)) == -3 and multi(at(1, 257)) == -3 and multi(at(2, 257)) == -3
    assert multi(at(4, 257)) == -3
    assert b"tensor 0" in lib.zk_last_error()
    for i, bad in enumerate((-1.0, 1.0, 1.0, -1e-8, -0.1)):
        assert multi(good, hyper=(*HYPER[:i], bad, *HYPER[i + 1:])) == -1
    #        param grad  m    v  base lowp  n step seed g low
    good8 = [256, 256, 257, 257, 256, 256, 0, 1, 9, 0, 1]

    def multi8(*rows):
        return lib.zk_adamw8_multi(_table(*rows), len(rows), *HYPER, None)

    assert multi8(good8) == 0
    assert multi8(at(7, 0, good8)) == -1 and multi8(at(9, 4, good8)) == -2
    assert multi8(at(4, 0, at(6, 8, good8))) == -1 and multi8(at(4, 257, good8)) == -3

    def values(row, dt=0):
        return lib.zk_adamw8_values(_table(row), 1, dt, None)

    view = [257, 257, 256, 256, 256, 0]
    assert values(view) == 0 and values(view, 2) == 0 and values(view, 1) == -2
    assert values(at(5, -1, view)) == -1 and values(at(3, 0, at(5, 8, view))) == -1
    assert values(at(3, 258, view)) == -3 and values(at(3, 258, view), 2) == 0
    assert lib.zk_adamw8_values(None, 2, 0, None) == -1


def test_wrappers_refuse():
    t, b = torch.zeros(4), torch.zeros(1, 2, dtype=torch.int16)
    c = torch.zeros(4, dtype=torch.uint8)
    h = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0)
    with pytest.raises(ValueError, match="GPU"):
        kernels.adamw_multi([t], [t], [t], [t], [1], **h)
    with pytest.raises(ValueError, match="length"):
        kernels.adamw_multi([t], [t], [t], [], [1], **h)
    with pytest.raises(ValueError, match="length"):
        kernels.adamw8_multi([t], [t], [c], [c], [b], [1], seeds=[], **h)
    with pytest.raises(ValueError, match="GPU"):
        kernels.adamw8_values([c], [c], [b])
    with pytest.raises(ValueError, match="fp32 or bf16"):
        kernels.adamw8_values([c], [c], [b], dtype=torch.float16)
    kernels.adamw_multi([], [], [], [], [], **h)  # an empty list is no work
    assert kernels.adamw8_values([], [], []) == ([], [])


def test_states_keep_their_types_through_a_checkpoint():
    """16-bit parameters' fp32 masters and moments, and 8-bit codes, survive
    load_state_dict (torch's own casts them to the parameter's type)."""
    for bits, moment in ((32, torch.float32), (8, torch.uint8)):
        p = torch.nn.Parameter(torch.randn(300).bfloat16())
        opt = optim.FusedAdamW([p], state_bits=bits)
        st = opt._init_state(p)
        st["step"] = 7
        for k in ("exp_avg", "exp_avg_sq"):
            st[k] = torch.arange(300).to(moment)
        st["master"] = torch.randn(300)
        q = torch.nn.Parameter(p.detach().clone())
        other = optim.FusedAdamW([q], lr=5.0, state_bits=bits)
        other.load_state_dict(opt.state_dict())
        got = other.state[q]
        assert got.keys() == st.keys() and other.param_groups[0]["lr"] == 1e-3
        for k, v in st.items():
            if torch.is_tensor(v):
                assert got[k].dtype == v.dtype and torch.equal(got[k], v)
                assert got[k].data_ptr() != v.data_ptr()
            else:
                assert got[k] == v
        wrong = optim.FusedAdamW([q], state_bits=40 - bits)
        with pytest.raises(ValueError, match="state_bits"):
            wrong.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="state_bits"):
        optim.FusedAdamW([p], state_bits=16)


def test_spans_that_meet():
    meet = kernels.spans_meet
    assert not meet([], [], 4) and not meet([0, 0, 0], [0, 0, 0], 4) and not meet([64], [8], 4)
    assert not meet([64, 32, 96], [8, 8, 1], 4) and not meet([64, 64], [8, 0], 4)
    assert meet([64, 64], [8, 8], 4) and meet([64, 32], [8, 9], 4) and meet([96, 0, 64], [1, 1, 9], 4)
    assert meet([0, 4, 100], [100, 0, 1], 4)


def test_step_counts_load_as_torch_loads_them():
    """torch.optim.Adam's, whose step count is a tensor (left to torch to place)."""
    p = torch.nn.Parameter(torch.randn(6))
    opt = torch.optim.Adam([p])
    p.grad = torch.ones(6)
    opt.step()
    ours = optim.FusedAdamW([p])
    ours.load_state_dict(opt.state_dict())
    assert int(ours.state[p]["step"]) == 1
    assert torch.equal(ours.state[p]["exp_avg"], opt.state[p]["exp_avg"])

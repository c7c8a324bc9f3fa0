"""What packed attention and the rotation by several axes refuse, before any
launch (CPU)."""
import ctypes

import pytest
import torch

from zorse_amd import _abi, functional as F, kernels as K

P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(258)


def _packed(**kw):
    d = _abi.PackedDesc(T=8, Hq=2, Hkv=1, d=64, scale=0.125, causal=1, dtype=2)
    for name in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        setattr(d, name + "_s", 128)
        setattr(d, name + "_h", 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def test_attention_entry_points_refuse():
    lib = _abi.lib()

    def fwd(q=P, k=P, v=P, plan=P, o=P, lse=P, **kw):
        return lib.zk_attn_packed_fwd(_packed(**kw), q, k, v, plan, o, lse, None)

    def bwd(dq=P, ws=P, nbytes=1 << 20, **kw):
        return lib.zk_attn_packed_bwd(_packed(**kw), P, P, P, P, P, P, P, dq, P, P, ws, nbytes, None)

    assert lib.zk_attn_packed_fwd(None, P, P, P, P, P, P, None) == -1
    for call in (fwd, bwd):
        assert call(dtype=3) == -2
        assert call(T=-1) == -1 and call(T=1 << 30) == -1
        assert call(Hq=3, Hkv=2) == -1 and call(Hq=0) == -1 and call(Hkv=0) == -1
        assert call(window=-1) == -1 and call(window=3, causal=0) == -1
        assert call(scale=0.0) == -1 and call(scale=float("nan")) == -1 and call(scale=-1.0) == -1
        assert call(scale=float("inf")) == -1
        assert call(d=130) == -4 and call(d=63) == -4 and call(d=0) == -4
        assert call(q_s=-8) == -4 and call(k_s=1 << 23) == -4
        assert call(q_h=63) == -3
        assert call(T=1 << 24, Hq=64) == -4
        assert call(T=0) == 0
    assert fwd(q=None) == -1 and fwd(o=None) == -1 and fwd(plan=None) == -1 and fwd(lse=None) == -1
    assert fwd(q=ODD) == -3 and fwd(lse=ODD) == -3 and fwd(dtype=0, v=ODD) == -3
    assert bwd(dq=None) == -1 and bwd(dq=ODD) == -3 and bwd(do_s=129) == -3
    assert bwd(ws=None) == -5 and bwd(nbytes=2 * 2 * 8 * 4) == -5
    assert lib.zk_attn_packed_bwd_workspace(_packed()) >= 2 * 2 * 8 * 4


def test_plans_refuse():
    lib = _abi.lib()
    assert lib.zk_packed_plan_bytes(-1) == -1 and lib.zk_packed_plan_bytes(1 << 30) == -1
    need = lib.zk_packed_plan_bytes(100)
    assert need >= 4 * (1 + 200 + 3)
    assert lib.zk_packed_plan(P, 0, 1, 100, P, need - 1, None, None) == -5
    assert lib.zk_packed_plan(None, 0, 1, 100, P, need, None, None) == -1
    assert lib.zk_packed_plan(P, 0, -1, 100, P, need, None, None) == -1
    assert lib.zk_packed_plan(P, 1, 1, 100, P, need, ctypes.c_void_p(260), None) == -3
    for bad in ([1, 5], [0, 5, 4], [], [[0, 5]], [0.0, 5.0]):
        with pytest.raises(ValueError):
            F.PackedSequences(bad, 100, device="cpu")
    with pytest.raises(ValueError, match="more than"):
        F.PackedSequences([0, 101], 100, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        K.packed_plan(torch.tensor([0, 5]), 5)


def test_wrappers_refuse():
    q, k = torch.zeros(8, 2, 64), torch.zeros(8, 1, 64)
    plan = torch.zeros(K.packed_plan_words(8), dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensors"):
        K.attn_packed_fwd(q, k, k, plan)
    with pytest.raises(ValueError, match="must be"):
        K.attn_packed_fwd(q[None], k[None], k[None], plan)
    cos = torch.zeros(4, 32)
    pos = torch.zeros(2, 8, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU tensors"):
        F.rope_axes(q, k, cos, cos, pos, F.pair_axes_of((16, 16)))
    with pytest.raises(ValueError, match=r"\[tokens, H, d\]"):
        F.rope_axes(q[0], k, cos, cos, pos, F.pair_axes_of((16, 16)))
    for sections in ((), (-1, 3), (1,) * 257):
        with pytest.raises(ValueError):
            F.pair_axes_of(sections)


def test_rotation_entry_point_refuses():
    lib = _abi.lib()

    def call(q=P, k=P, qo=P, ko=P, cos=P, pos=P, axes=bytes(32), **kw):
        d = _abi.AxesDesc(B=1, S=8, Hq=2, Hkv=1, d=64, n_pos=4, n_axes=2, dtype=2)
        for name, v in kw.items():
            setattr(d, name, v)
        return lib.zk_rope_axes(ctypes.byref(d), q, k, qo, ko, cos, P, pos, axes, None)

    assert call(dtype=9) == -2 and call(pairing=2) == -1
    assert call(B=-1) == -1 and call(S=-1) == -1 and call(Hq=0) == -1 and call(Hkv=-1) == -1
    assert call(B=1 << 20, S=1 << 20) == -1 and call(S=1 << 31) == -1
    assert call(d=63) == -4 and call(d=0) == -4 and call(d=514) == -4
    assert call(n_axes=0) == -1 and call(n_axes=257) == -1 and call(n_pos=0) == -1
    assert call(axes=bytes([1] * 31 + [2])) == -1 and call(axes=None) == -1
    assert call(q=None) == -1 and call(k=None) == -1 and call(ko=None) == -1 and call(pos=None) == -1
    assert call(q=ctypes.c_void_p(257)) == -3 and call(pos=ctypes.c_void_p(260)) == -3
    assert call(S=0) == 0

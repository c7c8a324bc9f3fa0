"""What the norm of query and key heads refuses, before any launch (CPU)."""
import ctypes

import pytest
import torch

from zorse_amd import _abi, kernels


def _desc(**kw):
    d = _abi.QkDesc(B=1, S=4, Hq=2, Hkv=1, d=8, n_pos=4, eps=1e-6, dtype=2, w_dtype=0)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def test_entry_points_refuse():
    lib = _abi.lib()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(257)

    def fwd(q=p, k=p, wq=p, wk=p, qo=p, ko=p, cos=p, sin=p, pos=None, **kw):
        return lib.zk_qk_norm_rope_fwd(_desc(**kw), q, k, wq, wk, qo, ko, cos, sin, pos, None)

    assert fwd(dtype=5) == -2 and fwd(w_dtype=-1) == -2
    assert fwd(pairing=2) == -1 and fwd(eps=-1.0) == -1
    assert fwd(d=7) == -1 and fwd(d=0) == -1 and fwd(d=1026) == -4
    assert fwd(Hq=0) == -1 and fwd(B=-1) == -1
    assert fwd(n_pos=3) == -1 and fwd(n_pos=0, pos=p) == -1
    assert fwd(k=None) == -1 and fwd(wk=None) == -1 and fwd(ko=None) == -1 and fwd(qo=None) == -1
    assert fwd(cos=None) == -1 and fwd(q=odd) == -3 and fwd(qo=odd) == -3 and fwd(pos=odd) == -3
    assert fwd(S=0) == 0 and fwd(B=0, k=None, wk=None, ko=None, Hkv=0) == 0
    assert lib.zk_qk_norm_rope_fwd(None, p, p, p, p, p, p, p, p, None, None) == -1

    ws = lib.zk_qk_norm_rope_bwd_workspace(8)
    assert ws > 0 and lib.zk_qk_norm_rope_bwd_workspace(0) < 0
    assert lib.zk_qk_norm_rope_bwd_workspace(1026) < 0

    def bwd(dwk=p, dy=p, w=p, n=ws, **kw):
        return lib.zk_qk_norm_rope_bwd(_desc(**kw), p, p, p, p, dy, p, p, p, p, dwk, p, p, None, w,
                                       n, None)

    assert bwd(dwk=None) == -1 and bwd(dy=None) == -1 and bwd(w=None) == -1
    assert bwd(n=ws - 1) == -5 and bwd(dy=odd) == -3 and bwd(d=1026) == -4


def test_wrapper_refuses():
    q, k, w = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 1, 8), torch.ones(8)
    t = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="GPU"):
        kernels.qk_norm_rope_fwd(q, k, w, w, t, t)
    with pytest.raises(ValueError, match="belong together"):
        kernels.qk_norm_rope_fwd(q, k, w, None, t, t)
    with pytest.raises(ValueError, match="gradient for each"):
        kernels.qk_norm_rope_bwd(q, None, q, k, w, w, t, t)

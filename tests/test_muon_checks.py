"""What the orthogonal updates refuse, before any launch (CPU)."""
import ctypes

import pytest
import torch

from zorse_amd import _abi, kernels as K

P = ctypes.c_void_p(4096)


def _row(**kw):
    m = _abi.MuonMatrix(grad=4096, out=8192, rows=8, cols=6, ld_grad=6, ld_out=6, ld_param=6,
                        ld_momentum=6, grad_dtype=2, out_dtype=2)
    for k, v in kw.items():
        setattr(m, k, v)
    return m


def _factors(n=1, ws=P, nbytes=1 << 30, steps=5, coef=(3.4445, -4.775, 2.0315), eps=1e-7, **kw):
    return _abi.lib().zk_orthogonalize(ctypes.byref(_row(**kw)), n, steps, *coef, eps, ws, nbytes, None)


def _step(lr=0.1, mu=0.9, wd=0.0, adjust=0, **kw):
    row = _row(**{"param": 12288, "momentum": 16384, **kw})
    return _abi.lib().zk_muon_multi(ctypes.byref(row), 1, 5, 3.4445, -4.775, 2.0315, 1e-7, lr, mu, wd, 1,
                                    adjust, P, 1 << 30, None)


def test_entry_points_refuse():
    lib = _abi.lib()
    assert _factors(n=0) == 0 and lib.zk_orthogonalize(None, 1, 5, 3, -4, 2, 0, P, 9, None) == -1
    for call in (_factors, _step):
        assert call(rows=0) == -1 and call(cols=-1) == -1 and call(rows=1 << 20) == -1
        assert call(rows=(1 << 20) - 1, cols=1 << 13, ld_grad=1 << 13, ld_out=1 << 13, ld_param=1 << 13,
                    ld_momentum=1 << 13) == -1
        assert call(grad_dtype=7) == -2 and call(out_dtype=-1) == -2
        assert call(grad=None) == -1 and call(ld_grad=5) == -1 and call(ld_out=5) == -1
        assert call(grad=4097) == -3 and call(out=8193) == -3
    assert _factors(out=None) == -1 and _factors(param=12288) == -1
    assert _factors(steps=0) == -1 and _factors(steps=101) == -1 and _factors(eps=-1.0) == -1
    assert _factors(eps=float("nan")) == -1
    assert _factors(coef=(5.0, 1.0, 0.0)) == -1 and _factors(coef=(float("nan"), 0, 0)) == -1
    assert _factors(ws=None) == -5 and _factors(nbytes=64) == -5
    assert _step(param=None) == -1 and _step(momentum=None) == -1 and _step(ld_param=3) == -1
    assert _step(param=12290) == -3
    assert _step(lr=-1.0) == -1 and _step(mu=1.0) == -1 and _step(wd=-0.1) == -1 and _step(adjust=2) == -1
    assert _step(lr=float("nan")) == -1


def test_workspace_holds_the_list():
    lib = _abi.lib()
    rows = (_abi.MuonMatrix * 3)(*(_row(rows=r, cols=c) for r, c in ((300, 500), (500, 300), (4096, 64))))
    need = lib.zk_muon_workspace(rows, 3)
    assert need >= 4 * 2 * (300 * 500 * 2)
    assert lib.zk_muon_workspace(None, 3) == 0 and lib.zk_muon_workspace(rows, 0) == 0


def test_wrappers_refuse():
    x = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="GPU tensors"):
        K.orthogonalize([x])
    with pytest.raises(TypeError, match="lists of tensors"):
        K.orthogonalize([3])
    with pytest.raises(ValueError, match="adjust"):
        K.muon_multi([x], [x], [x], lr=0.1, momentum=0.9, weight_decay=0.0, adjust="none")
    assert K.orthogonalize([]) == []


def test_a_call_without_a_workspace_checks_the_rest():
    row = _row(param=12288, momentum=16384)

    def call(lr=0.1, mu=0.9, n=1):
        return _abi.lib().zk_muon_multi(ctypes.byref(row), n, 5, 3.4445, -4.775, 2.0315, 1e-7, lr, mu, 0.0, 1,
                                        0, None, 0, None)

    assert call() == -5 and call(lr=-1.0) == -1 and call(mu=1.0) == -1 and call(n=0) == 0

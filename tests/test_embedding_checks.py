"""What the token embedding refuses, before anything is launched (CPU)."""
import ctypes

import pytest
import torch

from zorse_amd import _abi, functional, kernels


def test_entry_points_refuse():
    lib = _abi.lib()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(257)
    fwd, bwd = lib.zk_embedding_fwd, lib.zk_embedding_bwd
    assert fwd(p, 1, 4, p, 8, 16, p, 1.0, 9, 0, None) == -2
    assert fwd(p, 1, 4, p, 8, 16, p, 1.0, 0, 7, None) == -2
    assert fwd(p, 1, -1, p, 8, 16, p, 1.0, 0, 0, None) == -1
    assert fwd(p, 1, 4, p, 0, 16, p, 1.0, 0, 0, None) == -1
    assert fwd(p, 1, 4, p, 8, 0, p, 1.0, 0, 0, None) == -1
    assert fwd(p, 1, 1 << 29, p, 8, 16, p, 1.0, 0, 0, None) == -1
    assert fwd(p, 1, 4, p, 1 << 28, 16, p, 1.0, 0, 0, None) == -1
    assert fwd(None, 1, 4, p, 8, 16, p, 1.0, 0, 0, None) == -1
    assert fwd(p, 1, 4, odd, 8, 16, p, 1.0, 2, 0, None) == -3
    assert fwd(None, 1, 0, None, 8, 16, None, 1.0, 0, 0, None) == 0  # no tokens
    ws = lib.zk_embedding_bwd_workspace(400, 8, 16)
    assert ws > 0 and lib.zk_embedding_bwd_workspace(4, 0, 16) < 0
    assert lib.zk_embedding_bwd_workspace(1 << 29, 8, 16) < 0
    args = (p, 1, 400, p, 0, p, 0, 8, 16, 1.0, -1, 0)
    assert bwd(*args, p, ws - 1, None) == -5
    assert bwd(*args, None, ws, None) == -1
    assert bwd(*args, ctypes.c_void_p(264), ws, None) == -3
    assert lib.zk_embedding_bwd_workspace(4, 8, 16) == 0  # few tokens need none
    assert bwd(p, 1, 4, None, 0, p, 0, 8, 16, 1.0, -1, 0, p, ws, None) == -1
    assert bwd(p, 1, 4, p, 5, p, 0, 8, 16, 1.0, -1, 0, p, ws, None) == -2
    # nothing to add: no launch
    assert bwd(None, 1, 0, None, 0, p, 0, 8, 16, 1.0, -1, 1, p, ws, None) == 0


def test_wrappers_refuse_cpu_tensors_and_bad_arguments():
    ids, w = torch.zeros(3, dtype=torch.int64), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="GPU"):
        kernels.embedding_fwd(ids, w)
    with pytest.raises(ValueError, match="GPU"):
        kernels.embedding_bwd(ids, torch.zeros(3, 4), 8)
    for bad in (8, -9):
        with pytest.raises(ValueError, match="padding_idx"):
            functional.embedding(ids, w, padding_idx=bad)


def test_models_embed_on_the_cpu_as_before():
    """The models' embedding module on CPU tensors is nn.Embedding's."""
    from zorse_amd.llama_simple import TokenEmbedding
    torch.manual_seed(0)
    m = TokenEmbedding(11, 6, padding_idx=2)
    ref = torch.nn.Embedding(11, 6, padding_idx=2)
    ref.load_state_dict(m.state_dict())
    ids = torch.tensor([[1, 2, 10], [2, 2, 0]])
    a, b = m(ids), ref(ids)
    a.square().sum().backward()
    b.square().sum().backward()
    assert torch.equal(a, b) and torch.equal(m.weight.grad, ref.weight.grad)

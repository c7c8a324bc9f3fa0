"""Outputs that the caller gives to the norm of query and key heads: one for
each of q and k or none, refused before any launch (CPU)."""
import pytest
import torch

from zorse_amd import kernels


@pytest.mark.parametrize("missing", [0, 1])
def test_one_output_of_two_is_refused(missing):
    """A view given for one of them must not be left unwritten, nor its strides
    used for a new tensor."""
    q, w, t = torch.zeros(1, 4, 2, 8), torch.ones(8), torch.zeros(4, 4)
    k = torch.zeros(1, 4, 24)[..., 16:].unflatten(-1, (1, 8))
    out = [torch.zeros_like(q), k]
    out[missing] = None
    with pytest.raises(ValueError, match="output for each of q and k"):
        kernels.qk_norm_rope_fwd(q, k, w, w, t, t, out=tuple(out))
    with pytest.raises(ValueError, match="output for each of q and k"):
        kernels.qk_norm_rope_bwd(q, k, q, k, w, w, t, t, out=tuple(out))


@pytest.mark.parametrize("q_given", [False, True])
def test_output_of_an_absent_k_is_refused(q_given):
    q, w, t = torch.zeros(1, 4, 2, 8), torch.ones(8), torch.zeros(4, 4)
    out = (torch.zeros_like(q) if q_given else None, torch.zeros(1, 4, 1, 8))
    with pytest.raises(ValueError, match="output for each of q and k"):
        kernels.qk_norm_rope_fwd(q, None, w, None, t, t, out=out)
    with pytest.raises(ValueError, match="output for each of q and k"):
        kernels.qk_norm_rope_bwd(q, None, q, None, w, None, t, t, out=out)

"""Forward-mode derivatives of the token embedding: the lookup is linear in the
table, and the table's gradient in dy."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


def _inputs(dev, V=12, h=24):
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, V, (5, 40), generator=g).to(dev)
    return ids, *(torch.randn(V, h, generator=g).to(dev) for _ in range(2))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tangent_of_the_lookup(dev, grad, dtype):
    """Detached and under no_grad, where no node is made, and with one."""
    from zorse_amd import functional
    ids, w, t = _inputs(dev)
    w.requires_grad_(grad)
    kw = dict(scale=0.5, padding_idx=3, dtype=dtype)
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        y, ty = fwad.unpack_dual(functional.embedding(ids, fwad.make_dual(w, t), **kw))
        assert ty is not None and ty.dtype == dtype
        assert torch.equal(y, functional.embedding(ids, w, **kw))
        assert torch.equal(ty, functional.embedding(ids, t, **kw))
        # an expanded tangent
        row = torch.linspace(-1, 1, 24, device=dev).to(torch.float32)
        _, ty = fwad.unpack_dual(functional.embedding(ids, fwad.make_dual(w, row.expand(12, 24)), **kw))
        assert torch.equal(ty, (0.5 * row).to(dtype).expand(5, 40, 24))


def test_tangent_through_the_models_table(dev):
    """As nn.Embedding's, whose module the models' one replaces."""
    from zorse_amd.llama_simple import TokenEmbedding
    ids, w, t = _inputs(dev)
    ours = TokenEmbedding(12, 24, padding_idx=3, device=dev)
    theirs = torch.nn.Embedding(12, 24, padding_idx=3, device=dev)
    for no_grad in (False, True):
        with fwad.dual_level(), torch.set_grad_enabled(not no_grad):
            dual = {"weight": fwad.make_dual(w, t)}
            got, want = (fwad.unpack_dual(torch.func.functional_call(m, dual, (ids,)))
                         for m in (ours, theirs))
            assert torch.equal(got.primal, want.primal) and torch.equal(got.tangent, want.tangent)


def test_tangent_of_the_gradient(dev):
    """Forward over reverse: of sum(y^2) / 2 the gradient is n_r w_r for a row
    that n_r tokens name, its tangent n_r t_r, sums of equal numbers: each of the
    n_r additions is off by at most 2^-24 of the sum."""
    from zorse_amd import functional
    ids, w, t = _inputs(dev)
    n = torch.bincount(ids.flatten(), minlength=12).double()
    n[3] = 0
    w.requires_grad_()
    with fwad.dual_level():
        y = functional.embedding(ids, fwad.make_dual(w, t), padding_idx=3)
        for create in (True, False):
            g, tg = fwad.unpack_dual(torch.autograd.grad((y * y).sum() / 2, w, retain_graph=True,
                                                         create_graph=create)[0])
            for got, row in ((g, w), (tg, t)):
                ref = n[:, None] * row.detach().double()
                assert bool(((got.double() - ref).abs() <= (n.max() + 2) * 2.0 ** -24 * ref.abs()).all())

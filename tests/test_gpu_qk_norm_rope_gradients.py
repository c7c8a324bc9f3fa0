"""Gradients of the norm of query and key heads at their edges."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(dev, heads, kv_heads, d=16, S=5):
    g = torch.Generator().manual_seed(heads + d)
    q, k = (torch.randn(2, S, h, d, generator=g).to(dev) for h in (heads, kv_heads))
    wq, wk = ((1 + 0.1 * torch.randn(d, generator=g)).to(dev) for _ in range(2))
    ang = torch.arange(S)[:, None] * 1e4 ** (-torch.arange(0, d, 2) / d)
    return q, k, wq, wk, ang.cos().to(dev), ang.sin().to(dev)


@pytest.mark.parametrize("wdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [16, 130])
def test_key_weight_without_key_heads(dev, wdt, d):
    """k [B, S, 0, d]: its weight's gradient is zero (and is written: the memory
    that it gets held NaN before), q's are those without a k."""
    from zorse_amd import functional, kernels
    q, k, wq, wk, cos, sin = _inputs(dev, 3, 0, d)
    wq, wk = wq.to(wdt), wk.to(wdt)
    dq = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).to(dev)
    want = kernels.qk_norm_rope_bwd(dq, None, q, None, wq, None, cos, sin)
    junk = [torch.full((d,), float("nan"), device=dev, dtype=wdt) for _ in range(8)]
    del junk
    got = kernels.qk_norm_rope_bwd(dq, k, q, k, wq, wk, cos, sin)
    assert got[1].shape == k.shape and torch.equal(got[3], torch.zeros_like(wk))
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    junk = [torch.full((d,), float("nan"), device=dev, dtype=wdt) for _ in range(8)]
    del junk
    y = functional.qk_norm_rope(*leaves, cos, sin)
    assert y[1].shape == k.shape
    grads = torch.autograd.grad(y, leaves, (dq, k))
    assert torch.equal(grads[3], torch.zeros_like(wk)) and torch.equal(grads[2], want[2])


@pytest.mark.parametrize("which", range(4))
def test_penalty_of_gradients_is_refused(dev, which):
    """A gradient for a constant dy depends on q, k and the weights all the same:
    with create_graph it has a node that says that it cannot be differentiated,
    instead of counting as a constant."""
    from zorse_amd import functional
    *args, cos, sin = _inputs(dev, 4, 2)
    x = args[which].requires_grad_()
    y = functional.qk_norm_rope(*args, cos, sin)
    total = y[0].sum() + y[1].square().sum().detach() + y[1].sum()
    plain, = torch.autograd.grad(total, x, retain_graph=True)
    dx, = torch.autograd.grad(total, x, create_graph=True)
    assert torch.equal(dx, plain) and dx.requires_grad
    with pytest.raises(RuntimeError, match="differentiated once"):
        (total + dx.square().sum()).backward()


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(dev, which, grad):
    """A tangent of any input, instead of being dropped."""
    import torch.autograd.forward_ad as fwad
    from zorse_amd import functional
    args = [t.requires_grad_(grad and i < 4) for i, t in enumerate(_inputs(dev, 4, 2))]
    with fwad.dual_level():
        args[which] = fwad.make_dual(args[which].detach(), torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward"):
            functional.qk_norm_rope(*args)


def test_forward_over_reverse_is_refused(dev):
    import torch.autograd.forward_ad as fwad
    from zorse_amd import functional
    q, k, wq, wk, cos, sin = _inputs(dev, 4, 2)
    q.requires_grad_()
    y = functional.qk_norm_rope(q, k, wq, wk, cos, sin)
    with fwad.dual_level():
        dy = fwad.make_dual(torch.ones_like(y[0]), torch.ones_like(y[0]))
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(y[0], q, dy)

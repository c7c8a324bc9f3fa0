"""A step of Muon that is refused has changed nothing, whichever part is at fault."""
import pytest
import torch

from zorse_amd import optim

pytestmark = pytest.mark.gpu

BF, F4 = torch.bfloat16, torch.float32


def _model(dev, dt):
    g = torch.Generator().manual_seed(4)
    shapes = ((40, 30), (300,), (20, 50), (7,))
    ps = [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).to(dev, dt)) for s in shapes]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).to(dev, dt)
    return ps


def _state(opt, ps):
    tensors = [p.detach() for p in ps]
    for p in ps:
        tensors += [t for t in opt.state[p].values() if torch.is_tensor(t)]
    return [t.clone() for t in tensors], [opt.state[p]["step"] for p in ps], [p._version for p in ps]


@pytest.mark.parametrize("dt", [F4, BF])
@pytest.mark.parametrize("fault", ["adam_lr", "vector", "lr", "matrix", "coefficients"])
def test_a_refused_step_changes_nothing(dev, dt, fault):
    ps = _model(dev, dt)
    opt = optim.Muon(ps, lr=0.02, adam_lr=1e-3)
    stepped = []
    for p in ps:
        opt.add_step_hook(p, lambda q: stepped.append(q))
    opt.step()
    before, counts, versions = _state(opt, ps)
    stepped.clear()
    group, grads = opt.param_groups[0], [p.grad for p in ps]
    if fault == "adam_lr":
        group["adam_lr"] = -1.0
    elif fault == "lr":
        group["lr"] = -1.0
    elif fault == "coefficients":
        group["ns_coefficients"] = (9.0, 0.0, 0.0)
    elif fault == "vector":  # a gradient that shares memory with another parameter, which is written
        ps[3].grad = ps[1].detach()[:7]
    else:
        ps[0].grad = ps[0].detach()
    with pytest.raises((ValueError, RuntimeError)):
        opt.step()
    torch.cuda.synchronize()
    after, counts2, versions2 = _state(opt, ps)
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert counts == counts2 and versions == versions2 and not stepped
    # and the right call is a step as any other
    group.update(adam_lr=1e-3, lr=0.02, ns_coefficients=(3.4445, -4.775, 2.0315))
    for p, g in zip(ps, grads):
        p.grad = g
    opt.step()
    twins = _model(dev, dt)
    other = optim.Muon(twins, lr=0.02, adam_lr=1e-3)
    other.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(ps, twins)) and len(stepped) == len(ps)


def test_a_step_checked_before_it_runs(dev):
    from zorse_amd import kernels as K
    p, g, m = (torch.randn(30, 40, device=dev) for _ in range(3))
    kw = dict(lr=0.1, momentum=0.9, weight_decay=0.0)
    p2, m2 = p.clone(), m.clone()
    step = K.muon_step([p], [g], [m], **kw)
    assert torch.equal(p, p2) and torch.equal(m, m2)
    step.run()
    K.muon_multi([p2], [g], [m2], **kw)
    assert torch.equal(p, p2) and torch.equal(m, m2)
    K.muon_step([], [], [], **kw).run()
    with pytest.raises(RuntimeError, match="ZK_EINVAL"):
        K.muon_step([p], [g], [m], lr=-1.0, momentum=0.9, weight_decay=0.0)

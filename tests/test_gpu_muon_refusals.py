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


def test_columns_of_one_buffer(dev):
    """Matrices beside each other share no element, though their spans meet."""
    from zorse_amd import kernels as K
    cuts = (0, 30, 70, 71, 100)

    def columns(seed):
        buf = torch.randn(50, 100, device=dev, generator=torch.Generator(dev).manual_seed(seed))
        return buf, [buf[:, a:b] for a, b in zip(cuts, cuts[1:])]

    kw = dict(lr=0.1, momentum=0.9, weight_decay=0.1)
    (pb, ps), (gb, gs), (mb, ms) = (columns(i) for i in range(3))
    twins = [[t.clone() for t in ts] for ts in (ps, gs, ms)]
    K.muon_multi(ps, gs, ms, **kw)
    K.muon_multi(*twins, **kw)
    for a, b in zip((*ps, *ms), (*twins[0], *twins[2])):
        assert torch.equal(a, b)
    # parameter, gradient and momentum in one buffer, and a single row between others
    buf = torch.randn(50, 100, device=dev)
    K.muon_multi([buf[:, :30]], [buf[:, 30:60]], [buf[:, 60:90]], **kw)
    K.orthogonalize([buf[:, :30], buf[3:4, 90:95]], outs=[buf[:, 30:60], buf[9:10, 60:65]])
    for bad in ([buf[:, :30], buf[:, 29:50]], [buf[:, 20:40], buf[1:, 10:21]], [buf[:, :30], buf[7:8, 25:35]],
                [buf[:, 80:], buf[:20, :30].as_strided((20, 30), (101, 1), 85)]):
        grads = [torch.zeros_like(t) for t in bad]
        with pytest.raises(ValueError, match="overlaps"):
            K.muon_multi(bad, grads, [torch.zeros_like(t) for t in bad], **kw)

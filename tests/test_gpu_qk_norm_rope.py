"""The norm of query and key heads with the rotation, against the formulas in
64 bits.

With u = 2^-24: a row's mean square has up to 16 + 6 additions of positive
terms, a product and the addition of eps behind it, so r is off by 14 u of
itself; a rotated element has three more products and a sum, 20 u of the sum of
its products' magnitudes.  dn is off by 2 u of its products' magnitudes,
mean(g x) by 30 u of the mean of its terms' magnitudes and r^2 by 28 u.  A
weight's gradient sums n rows in some order: (n + 30) u of the magnitudes'
sum.  Then half a step of the output's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
TINY = {BF: 2.0 ** -134, FP: 2.0 ** -25, F4: 2.0 ** -150}


def _tables(n, d, theta=1e4):
    inv = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _turn(x, c, s, inter):
    """Rotated pairs, and the sum of their products' magnitudes."""
    if inter:
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = x.chunk(2, -1)
    y = (a * c - b * s, b * c + a * s)
    m = ((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs())
    if inter:
        return torch.stack(y, -1).flatten(-2), torch.stack(m, -1).flatten(-2)
    return torch.cat(y, -1), torch.cat(m, -1)


def _half(t, dt):
    return torch.finfo(dt).eps / 2 * t.abs() + TINY[dt]


def _check(got, ref, before, dt, what):
    got = got.detach().cpu().double()
    bound = before * (1 + torch.finfo(dt).eps) + _half(ref, dt)
    bad = (got - ref).abs() > bound
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}"


def _reference(x, w, dy, c, s, eps, inter):
    """(y, dx, dw) in 64 bits, each with what may be lost before its rounding."""
    x, w, dy = x.double(), w.double(), dy.double()
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    y, m = _turn(x * r * w, c, s, inter)
    dn, dm = _turn(dy, c, -s, inter)
    g, gm = dn * w, dm * w.abs()
    mean = (g * x).mean(-1, keepdim=True)
    mag = (gm * x.abs()).mean(-1, keepdim=True)
    dx = r * (g - x * r * r * mean)
    lost = r * U * (24 * gm + 80 * x.abs() * r * r * mag)
    n = x.numel() // x.shape[-1]
    dw = (dn * x * r).flatten(0, -2).sum(0)
    return ((y, 20 * U * m), (dx, lost),
            (dw, (n + 30) * U * (dm * x.abs() * r).flatten(0, -2).sum(0)))


CASES = [
    # B, S, Hq, Hkv, d, activations, weights, interleaved, positions, eps
    (1, 1, 1, 1, 2, F4, F4, False, None, 1e-6),
    (3, 1, 32, 8, 128, BF, BF, False, "rows", 1e-6),
    (1, 5, 3, 3, 64, FP, FP, True, None, 1e-5),
    (2, 129, 4, 1, 128, BF, F4, True, "shared", 1e-6),
    (1, 2500, 5, 1, 16, BF, BF, False, None, 1e-6),
    (1, 67, 32, 32, 100, F4, F4, True, None, 1e-6),
    (2, 31, 7, 7, 110, BF, BF, False, "rows", 1e-6),
    (1, 2100, 9, 2, 6, FP, F4, False, "shared", 1e-6),
    (1, 40, 2, 1, 256, BF, BF, False, None, 1e-6),
    (1, 33, 1, 1, 1024, F4, BF, True, None, 1e-6),
    (1, 19, 2, 0, 48, BF, BF, False, None, 1e-6),
    (2, 4099, 40, 8, 128, BF, BF, False, "rows", 1e-6),
]


def _inputs(dev, B, S, Hq, Hk, d, dt, wdt, pos):
    g = torch.Generator().manual_seed(S * d + Hq)
    qkv = torch.randn(B, S, (Hq + 2 * Hk) * d + 3, generator=g)
    qkv[0, S // 2, :d] = 0  # a head without any value
    qkv[0, 0, :d] *= 1e3
    qkv = qkv.to(dt)
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(wdt) for _ in range(2))
    dq = torch.randn(B, S, Hq, d, generator=g).to(dt)
    dk = torch.randn(B, S, Hk, d, generator=g).to(dt)
    n_pos = S + 37
    p = None
    if pos == "shared":
        p = torch.randint(0, n_pos, (S,), generator=g)
    elif pos == "rows":
        p = torch.randint(0, n_pos, (B, S), generator=g)
    cos, sin = _tables(n_pos, d)
    return qkv, wq, wk, dq, dk, p, cos, sin


@pytest.mark.parametrize("B,S,Hq,Hk,d,dt,wdt,inter,pos,eps", CASES)
def test_forward_and_gradients(dev, B, S, Hq, Hk, d, dt, wdt, inter, pos, eps):
    from zorse_amd import functional
    qkv, wq, wk, dq, dk, p, cos, sin = _inputs(dev, B, S, Hq, Hk, d, dt, wdt, pos)
    buf = qkv.to(dev).requires_grad_()
    ws = [w.to(dev).requires_grad_() for w in (wq, wk)]
    q = buf[..., :Hq * d].unflatten(-1, (Hq, d))  # views of one buffer, odd row stride
    k = buf[..., Hq * d:(Hq + Hk) * d].unflatten(-1, (Hk, d)) if Hk else None
    out = functional.qk_norm_rope(q, k, ws[0], ws[1] if Hk else None, cos.to(dev), sin.to(dev),
                                  positions=None if p is None else p.to(dev), eps=eps,
                                  interleaved=inter)
    torch.autograd.backward([o for o in out if o is not None],
                            [t.to(dev) for t, o in ((dq, out[0]), (dk, out[1])) if o is not None])
    at = torch.arange(S) if p is None else p
    c, s = (t.double()[at].unsqueeze(-2) for t in (cos, sin))
    grad = buf.grad.cpu()
    for i, (h0, H, w, dy) in enumerate(((0, Hq, wq, dq), (Hq, Hk, wk, dk))):
        if not H:
            assert out[1] is None
            continue
        x = qkv[..., h0 * d:(h0 + H) * d].unflatten(-1, (H, d))
        y, dx, dw = _reference(x, w, dy, c, s, eps, inter)
        assert out[i].is_contiguous() and out[i].dtype == dt
        _check(out[i], *y, dt, "y")
        _check(grad[..., h0 * d:(h0 + H) * d].unflatten(-1, (H, d)), *dx, dt, "dx")
        _check(ws[i].grad, *dw, wdt, "dw")
    assert not bool(grad[..., (Hq + Hk) * d:].any())  # v and the padding


@pytest.mark.parametrize("inter", [False, True])
def test_gradients_against_differences(dev, inter):
    """Central differences of the kernel's own forward in fp32."""
    from zorse_amd import functional
    g = torch.Generator().manual_seed(11)
    B, S, H, d, step = 1, 3, 2, 12, 2.0 ** -8
    x, w = torch.randn(B, S, H, d, generator=g), 1 + 0.3 * torch.randn(d, generator=g)
    v = torch.randn(B, S, H, d, generator=g)
    cos, sin = (t.to(dev) for t in _tables(S, d))

    def f(xx, ww):
        y, _ = functional.qk_norm_rope(xx.to(dev), None, ww.to(dev), None, cos, sin,
                                       interleaved=inter)
        return float((y.cpu().double() * v.double()).sum())

    xd, wd = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    y, _ = functional.qk_norm_rope(xd, None, wd, None, cos, sin, interleaved=inter)
    y.backward(v.to(dev))
    # rounding: sum of |y v| times 20 u / step; truncation: step^2 / 6 of a
    # third derivative of order 10
    tol = 20 * U * float((y.detach().cpu() * v).abs().sum()) / step + 20 * step ** 2
    for i in range(0, x.numel(), 5):
        e = torch.zeros(x.numel()).index_fill_(0, torch.tensor([i]), step).view_as(x)
        assert abs((f(x + e, w) - f(x - e, w)) / (2 * step) - float(xd.grad.flatten()[i])) <= tol
    for i in range(d):
        e = torch.zeros(d).index_fill_(0, torch.tensor([i]), step)
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * step) - float(wd.grad[i])) <= tol


def test_in_place_and_positions_outside_the_tables(dev):
    from zorse_amd import kernels
    qkv, wq, wk, dq, dk, _, cos, sin = _inputs(dev, 2, 50, 6, 2, 64, BF, BF, None)
    q = qkv[..., :6 * 64].unflatten(-1, (6, 64)).to(dev)
    k = qkv[..., 6 * 64:8 * 64].unflatten(-1, (2, 64)).to(dev)
    a = (wq.to(dev), wk.to(dev), cos.to(dev), sin.to(dev))
    want = kernels.qk_norm_rope_fwd(q, k, *a)
    grads = kernels.qk_norm_rope_bwd(dq.to(dev), dk.to(dev), q, k, *a)
    gq, gk = dq.to(dev), dk.to(dev)
    same = kernels.qk_norm_rope_bwd(gq, gk, q, k, *a, out=(gq, gk))
    assert same[0] is gq and all(torch.equal(x, y) for x, y in zip(grads, same))
    q2, k2 = q.clone(), k.clone()
    kernels.qk_norm_rope_fwd(q2, k2, *a, out=(q2, k2))
    assert torch.equal(q2, want[0]) and torch.equal(k2, want[1])
    pos = torch.arange(50, device=dev)
    pos[7], pos[9] = -1, cos.shape[0]
    bad, _ = kernels.qk_norm_rope_fwd(q, k, *a, positions=pos)
    off = torch.zeros(50, dtype=torch.bool, device=dev)
    off[[7, 9]] = True
    assert bool(bad[:, off].isnan().all()) and torch.equal(bad[:, ~off], want[0][:, ~off])
    dxq, _, dwq, _ = kernels.qk_norm_rope_bwd(dq.to(dev), dk.to(dev), q, k, *a, positions=pos)
    assert bool(dxq[:, off].isnan().all()) and torch.equal(dxq[:, ~off], grads[0][:, ~off])
    assert bool(dwq.isnan().all())


def test_refusals_and_empty_batches(dev):
    from zorse_amd import functional, kernels
    w = torch.ones(8, device=dev)
    cos, sin = (t.to(dev) for t in _tables(4, 8))
    q, k = torch.randn(1, 4, 2, 8, device=dev), torch.randn(1, 4, 1, 8, device=dev)
    for args in ((q, k[:, :3], w, w, cos, sin), (q, k, w[:6], w, cos, sin),
                 (q, k.bfloat16(), w, w, cos, sin), (q, k, w, w, cos[:3], sin[:3]),
                 (q, k, w, w, cos, sin[:3]), (q, k, w, w, cos.double(), sin.double()),
                 (q.transpose(2, 3), k, w, w, cos, sin), (q[0], k, w, w, cos, sin)):
        with pytest.raises(ValueError):
            kernels.qk_norm_rope_fwd(*args)
    with pytest.raises(ValueError):
        kernels.qk_norm_rope_fwd(q, k, w, w, cos, sin, positions=torch.zeros(3, device=dev).long())
    with pytest.raises(ValueError):
        kernels.qk_norm_rope_fwd(q, k, w, w, cos, sin, out=(q, k.expand(1, 4, 2, 8)))
    with pytest.raises(ValueError, match="overlaps"):
        kernels.qk_norm_rope_fwd(q, k, w, w, cos, sin, out=(q[:, :1].expand(1, 4, 2, 8), k))
    e = q[:0].requires_grad_()
    we = w.clone().requires_grad_()
    y, _ = functional.qk_norm_rope(e, None, we, None, cos, sin)
    y.sum().backward()
    assert y.shape == e.shape and e.grad.shape == e.shape and not bool(we.grad.any())


def test_expanded_gradients_and_heads(dev):
    """y.sum() hands a gradient with strides of zero on; one key head expanded
    to all query heads gets the sum of their gradients."""
    from zorse_amd import functional
    cos, sin = (t.to(dev) for t in _tables(6, 16))
    w = torch.ones(16, device=dev, requires_grad=True)
    k = torch.randn(2, 6, 1, 16, device=dev, requires_grad=True)
    y, _ = functional.qk_norm_rope(k.expand(2, 6, 4, 16), None, w, None, cos, sin)
    y.sum().backward()
    k2 = k.detach().clone().requires_grad_()
    y2, _ = functional.qk_norm_rope(k2, None, w.detach(), None, cos, sin)
    y2.backward(torch.full_like(y2, 4.0))
    # four equal fp32 terms of about r (|g| + |mean|) added, and scaled by 4
    assert float((k.grad - k2.grad).abs().max()) <= 64 * U * float(k2.grad.abs().max() + 4)


def test_captured_pass_replays_with_new_values(dev):
    from zorse_amd import kernels
    qkv, wq, wk, dq, dk, _, cos, sin = _inputs(dev, 1, 300, 8, 2, 128, BF, BF, None)
    q = torch.empty(1, 300, 8, 128, device=dev, dtype=BF)
    k = torch.empty(1, 300, 2, 128, device=dev, dtype=BF)
    a = (wq.to(dev), wk.to(dev), cos.to(dev), sin.to(dev))
    dq, dk = dq.to(dev), dk.to(dev)

    def both():
        return (*kernels.qk_norm_rope_fwd(q, k, *a), *kernels.qk_norm_rope_bwd(dq, dk, q, k, *a))

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        q.copy_(torch.randn(q.shape, generator=g))
        k.copy_(torch.randn(k.shape, generator=g))

    fill(0)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for seed in (1, 2, 3):
        fill(seed)
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_second_differentiation_is_refused(dev):
    from zorse_amd import functional
    q = torch.randn(1, 3, 2, 16, device=dev, requires_grad=True)
    w = torch.ones(16, device=dev, requires_grad=True)
    cos, sin = (t.to(dev) for t in _tables(3, 16))
    y, _ = functional.qk_norm_rope(q, None, w, None, cos, sin)
    dq, = torch.autograd.grad(y, q, torch.ones_like(y, requires_grad=True), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        dq.sum().backward()


def test_gradient_of_one_output(dev):
    """A loss of q' alone: k and its weight have zero gradients, q's are those
    without k."""
    from zorse_amd import functional
    g = torch.Generator().manual_seed(5)
    q, k = (torch.randn(2, 7, h, 24, generator=g).to(dev).requires_grad_() for h in (3, 1))
    w = [torch.randn(24, generator=g).to(dev).requires_grad_() for _ in range(2)]
    cos, sin = (t.to(dev) for t in _tables(7, 24))
    dy = torch.randn(2, 7, 3, 24, generator=g).to(dev)
    y, _ = functional.qk_norm_rope(q, k, *w, cos, sin)
    dq, dk, dwq, dwk = torch.autograd.grad(y, (q, k, *w), dy)
    alone, none = functional.qk_norm_rope(q, None, w[0], None, cos, sin)
    want = torch.autograd.grad(alone, (q, w[0]), dy)
    assert none is None and torch.equal(y, alone)
    assert torch.equal(dq, want[0]) and not bool(dk.any()) and not bool(dwk.any())
    # dw: the same 42 products, over as many workgroups' partial sums or other
    # ones: 42 roundings of sums below 42 max|dn x r|
    bound = 42 * 2.0 ** -24 * 42 * float((dy.abs().max() * 2) * 24 ** 0.5)
    assert bool(((dwq - want[1]).abs() <= bound).all())

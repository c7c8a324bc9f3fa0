"""The rotation by several axes against the formula in 64 bits: two products
and a sum in fp32, 2 * 2^-24 of the products' magnitudes, and half a step of the
output's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32


def _tables(n, d):
    inv = 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _want(x, cos, sin, positions, axes, inter, back=False):
    """(value, bound) for heads [..., tokens, H, d], positions [A, ..., tokens]."""
    pos = positions[list(axes)].movedim(0, -1)  # [..., tokens, d/2]
    pair = torch.arange(len(axes))
    ok = (pos >= 0) & (pos < cos.shape[0])
    at = pos.clamp(0, cos.shape[0] - 1)
    c = torch.where(ok, cos.double()[at, pair], torch.nan).unsqueeze(-2)
    s = torch.where(ok, sin.double()[at, pair], torch.nan).unsqueeze(-2) * (-1 if back else 1)
    y = x.double()
    a, b = (y[..., 0::2], y[..., 1::2]) if inter else y.chunk(2, -1)
    parts = (a * c - b * s, b * c + a * s)
    mags = ((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs())
    join = (lambda p: torch.stack(p, -1).flatten(-2)) if inter else (lambda p: torch.cat(p, -1))
    val, mag = join(parts), join(mags)
    half = torch.finfo(x.dtype).eps / 2
    return val, (2.0 ** -23 * mag) * (1 + half) + half * val.abs() + torch.finfo(x.dtype).tiny


def _near(got, want):
    got, (ref, bound) = got.cpu().double(), want
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fine = ~torch.isnan(ref)
    assert bool(((got - ref).abs()[fine] <= bound[fine]).all())


CASES = [
    # shape of tokens, Hq, Hkv, d, sections, turns, interleaved, type
    ((1,), 1, 1, 2, (1,), False, False, BF),
    ((3,), 32, 8, 128, (16, 24, 24), False, False, BF),
    ((2, 37), 4, 2, 64, (11, 11, 10), True, False, FP),
    ((129,), 16, 16, 100, (25, 25), True, True, F4),
    ((65,), 5, 1, 100, (20, 30), False, False, BF),
    ((65,), 5, 0, 80, (10, 0, 30), False, True, BF),
    ((33,), 3, 3, 512, (64, 64, 64, 64), False, False, F4),
    ((33,), 2, 1, 256, (100, 28), True, True, FP),
    ((300,), 9, 9, 6, (1, 1, 1), False, True, F4),
    ((1000,), 40, 8, 128, (64,), False, False, BF),
    ((2, 5, ), 1, 7, 14, (3, 4), True, False, BF),
    ((50,), 70, 30, 96, (16, 16, 16), False, False, FP),
]


@pytest.mark.parametrize("shape,Hq,Hk,d,sections,turns,inter,dt", CASES)
def test_against_64_bits(dev, shape, Hq, Hk, d, sections, turns, inter, dt):
    from zorse_amd import functional as F
    g = torch.Generator().manual_seed(d + Hq)
    axes = F.pair_axes_of(sections, turns=turns)
    cos, sin = _tables(50, d)
    positions = torch.randint(0, 50, (len(sections), *shape), generator=g)
    buf = torch.randn(*shape, (Hq + 2 * Hk) * d, generator=g).to(dt)  # q | k | v
    dbuf = buf.to(dev)

    def parts(t):
        q = t[..., :Hq * d].unflatten(-1, (Hq, d))
        return q, t[..., Hq * d:(Hq + Hk) * d].unflatten(-1, (Hk, d)) if Hk else None

    q, k = parts(buf)
    dq, dk = parts(dbuf)
    leaves = [t.detach().requires_grad_() for t in (dq, dk) if t is not None]
    y = F.rope_axes(leaves[0], leaves[1] if Hk else None, cos.to(dev), sin.to(dev),
                    positions.to(dev), axes, interleaved=inter)
    ups = []
    for got, x in zip(y, (q, k)):
        if x is None:
            assert got is None
            continue
        _near(got, _want(x, cos, sin, positions, axes, inter))
        ups.append(torch.randn(x.shape, generator=g).to(dt))
    grads = torch.autograd.grad([t for t in y if t is not None], leaves, [u.to(dev) for u in ups])
    for got, u in zip(grads, ups):
        _near(got, _want(u, cos, sin, positions, axes, inter, back=True))


def test_positions_outside_and_values(dev):
    from zorse_amd import functional as F
    cos, sin = _tables(9, 16)
    axes = F.pair_axes_of((3, 5))
    positions = torch.tensor([[0, 8, 9, -1, 3], [2, 2, 2, 10 ** 12, 8]])
    x = torch.randn(5, 2, 16)
    x[4, 1, 3] = float("inf")
    x[4, 1, 11] = 1.0
    y, none = F.rope_axes(x.to(dev), None, cos.to(dev), sin.to(dev), positions.to(dev), axes)
    assert none is None
    want, bound = _want(x, cos, sin, positions, axes, False)
    got = y.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert bool(((got - want).abs()[fine] <= bound[fine]).all())
    assert torch.equal(got[~fine].nan_to_num(5), want[~fine].nan_to_num(5))


@pytest.mark.parametrize("dt", [BF, F4])
def test_in_place_and_back(dev, dt):
    from zorse_amd import functional as F, kernels as K
    cos, sin = (t.to(dev) for t in _tables(40, 64))
    axes = F.pair_axes_of((10, 22))
    pos = torch.randint(0, 40, (2, 77), device=dev)
    q, k = torch.randn(77, 4, 64, device=dev).to(dt), torch.randn(77, 2, 64, device=dev).to(dt)
    a, b = K.rope_axes(q, k, cos, sin, pos, axes)
    c, e = q.clone(), k.clone()
    K.rope_axes(c, e, cos, sin, pos, axes, q_out=c, k_out=e)
    assert torch.equal(a, c) and torch.equal(b, e)
    K.rope_axes(c, e, cos, sin, pos, axes, inverse=True, q_out=c, k_out=e)
    # there and back: two roundings of a pair of norm sqrt(2) at most its largest
    tol = 3 * torch.finfo(dt).eps * (q.float().abs().max() * 2)
    assert bool(((c - q).float().abs() <= tol).all())


def test_one_axis_is_the_rotation_of_the_layers(dev):
    """fp32: the same formula as flash_attention's rotation."""
    from zorse_amd import functional as F, kernels as K
    S, d = 90, 128
    cos, sin = F.rope_tables(S, d, 1e4, F4, dev)
    q, k = torch.randn(2, S, 3, d, device=dev), torch.randn(2, S, 1, d, device=dev)
    pos = torch.arange(S, device=dev).expand(1, 2, S).contiguous()
    for inter in (False, True):
        a, b = F.rope_axes(q, k, cos, sin, pos, F.pair_axes_of((64,)), interleaved=inter)
        c, e = q.clone(), k.clone()
        K.rope_(c, e, cos, sin, interleaved=inter)
        assert torch.allclose(a, c, rtol=0, atol=2e-6) and torch.allclose(b, e, rtol=0, atol=2e-6)


def test_differentiated_twice_and_captured(dev):
    from zorse_amd import functional as F
    cos, sin = (t.to(dev) for t in _tables(30, 32))
    axes, pos = F.pair_axes_of((8, 8)), torch.randint(0, 30, (2, 20), device=dev)
    q, k = torch.randn(20, 2, 32, device=dev), torch.randn(20, 1, 32, device=dev)
    lq, lk = q.clone().requires_grad_(), k.clone().requires_grad_()
    up = torch.randn_like(q).requires_grad_()
    y = F.rope_axes(lq, lk, cos, sin, pos, axes)
    g = torch.autograd.grad(y[0], lq, up, create_graph=True)[0]
    w = torch.randn_like(q)
    back = torch.autograd.grad(g, up, w)[0]  # the rotation again
    assert torch.equal(back, F.rope_axes(w, None, cos, sin, pos, axes)[0])
    side = torch.cuda.Stream()

    def step():
        a, b = (t.detach().requires_grad_() for t in (q, k))
        y = F.rope_axes(a, b, cos, sin, pos, axes)
        return [*(t.detach() for t in y), *torch.autograd.grad(y, (a, b), (w, k))]

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        torch.manual_seed(seed)
        for t in (q, k, w):
            t.copy_(torch.randn_like(t))
        pos.copy_(torch.randint(0, 30, (2, 20)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()


def test_more_than_2_24_workgroups(dev):
    """A token of 129 pairs takes a workgroup of 256 threads, and a launch fewer than
    2^32 of them along an axis."""
    from zorse_amd import functional as F, kernels as K
    T, d = (1 << 24) + 5, 258
    cos, sin = (t.to(dev) for t in _tables(50, d))
    axes = F.pair_axes_of((d // 2,))
    q = torch.empty(T, 1, d, device=dev, dtype=torch.bfloat16).normal_()
    pos = torch.randint(0, 50, (1, T), device=dev)
    parts = [slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)]
    want = [K.rope_axes(q[s].clone(), None, cos, sin, pos[:, s].contiguous(), axes)[0] for s in parts]
    K.rope_axes(q, None, cos, sin, pos, axes, q_out=q)
    for s, w in zip(parts, want):
        assert torch.equal(q[s], w)

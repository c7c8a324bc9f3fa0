"""Orthogonal factors by Newton-Schulz products, and the step that takes them,
against the polynomial in 64 bits.

The products round their operands to fp16, and small singular values grow 3.4
times a step, so what a rounding costs depends on the spectrum.  The bound is
therefore taken from the number format itself: `_rounded` computes the same
steps in 64 bits and rounds what the kernels store as they do (X in two fp16
numbers, of which the products take the first; G and P in one; with a side of at
most 128, or an fp32 result, all of them in two), without the kernels' sums in
fp32.  Their relative error, n 2^-24 of magnitudes for sums of n terms at worst,
about sqrt(n) 2^-24 as they are, lies a hundred times below fp16's half steps for
the sizes here, and at the level of two fp16 numbers' (2^-22): the norm of the
error may be 1.5 times that of `_rounded` in fp16, and 8 times it plus sqrt(n)
2^-22 in two numbers, beside half a step of the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32
A, B, C = 3.4445, -4.7750, 2.0315
S, R = 2.0 ** 7, 2.0 ** 13  # the powers of two of these coefficients


def _exact(u, steps=5, eps=1e-7, coef=(A, B, C)):
    a, b, c = coef
    x = u.double()
    x = x / (x.norm() + eps)
    if x.shape[0] > x.shape[1]:
        return _exact_t(x.T, steps, a, b, c).T
    return _exact_t(x, steps, a, b, c)


def _exact_t(x, steps, a, b, c):
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * g @ g) @ x
    return x


def _two(x):
    hi = x.half().double()
    return hi, (x - hi).half().double()


def _rounded(u, two, steps=5, eps=1e-7):
    x = u.double()
    x = x * float(torch.tensor(S / (float(x.norm()) + eps), dtype=F4))
    if x.shape[0] > x.shape[1]:
        x = x.T
    hi, lo = _two(x)

    def times(p, q):
        out = p[0] @ q[0]
        return out + p[0] @ q[1] + p[1] @ q[0] if two else out

    def t(p):
        return p[0].T, p[1].T

    for _ in range(steps):
        x = (hi, lo)
        g = _two(times(x, t(x)))
        if not two:
            g = (g[0], 0 * g[1])
        p = _two(C * R / S ** 4 * times(g, g) + B * R / S ** 2 * (g[0] + g[1]))
        if not two:
            p = (p[0], 0 * p[1])
        hi, lo = _two(A * (hi + lo) + times(p, x) / R)
    x = (hi + lo) / S
    return x.T if u.shape[0] > u.shape[1] else x


def _matrix(m, n, kind, seed, dt=F4):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g, dtype=torch.float64)
    if kind == "decay":
        k = min(m, n)
        u, _, v = torch.linalg.svd(x, full_matrices=False)
        x = u * torch.logspace(0, -4, k, dtype=torch.float64) @ v
    elif kind == "strong":  # a few directions over noise
        x = torch.randn(m, 4, generator=g, dtype=torch.float64) @ torch.randn(
            4, n, generator=g, dtype=torch.float64) + 0.01 * x
    elif kind == "scaled":  # rows of very different sizes
        x = x * torch.exp(2 * torch.randn(m, 1, generator=g, dtype=torch.float64))
    return (x * 1e-3).to(dt)


def _near(got, u, dt, what):
    got = got.cpu().double()
    two = min(u.shape) <= 128 or dt == F4
    ref, fmt = _exact(u), _rounded(u, two)
    norm = float(ref.norm())
    err = float((fmt - ref).norm())
    sums = math.sqrt(max(u.shape)) * 2.0 ** -22 * norm
    bound = (8 * err + sums if two else 1.5 * err) + torch.finfo(dt).eps / 2 * norm
    off = float((got - ref).norm())
    assert off <= bound, f"{what}: {off / norm:.2e} off, {bound / norm:.2e} allowed"
    assert float((got - ref).abs().max()) <= 40 * bound / math.sqrt(ref.numel()) + \
        torch.finfo(dt).eps * float(ref.abs().max())


CASES = [
    # rows, cols, spectrum, type, result
    (1, 1, "noise", F4, F4),
    (1, 50, "noise", BF, BF),
    (77, 1, "noise", FP, BF),
    (16, 16, "noise", F4, F4),
    (5, 700, "decay", BF, F4),
    (130, 64, "strong", F4, F4),
    (128, 128, "decay", BF, BF),
    (129, 200, "noise", BF, BF),
    (200, 129, "strong", F4, BF),
    (256, 256, "decay", FP, FP),
    (321, 577, "scaled", BF, BF),
    (577, 321, "strong", FP, FP),
    (512, 1024, "noise", BF, F4),
    (600, 320, "decay", F4, F4),
]


@pytest.mark.parametrize("m,n,kind,dt,out", CASES)
def test_against_64_bits(dev, m, n, kind, dt, out):
    from zorse_amd import kernels as K
    u = _matrix(m, n, kind, m + n, dt)
    got = K.orthogonalize([u.to(dev)], dtype=out)[0]
    assert got.dtype == out and got.shape == u.shape
    _near(got, u, out, f"{m} x {n} {kind}")


def test_a_list_of_all_sizes(dev):
    from zorse_amd import kernels as K
    shapes = [(256, 256), (40, 60), (300, 700), (700, 300), (3, 5), (256, 256), (1, 9), (640, 200),
              (130, 130), (64, 64), (150, 151), (151, 150)]
    us = [_matrix(m, n, "strong" if i % 2 else "noise", i, (F4, BF, FP)[i % 3])
          for i, (m, n) in enumerate(shapes)]
    outs = K.orthogonalize([u.to(dev) for u in us], dtype=BF)
    again = K.orthogonalize([u.to(dev) for u in us], dtype=BF)
    for u, o, p in zip(us, outs, again):
        _near(o, u, BF, f"{tuple(u.shape)}")
        assert torch.equal(o, p)
    assert K.orthogonalize([]) == []
    empty = torch.zeros(0, 5, device=dev)
    assert K.orthogonalize([empty, us[1].to(dev)])[0].shape == (0, 5)


@pytest.mark.parametrize("m,n,out", [(1024, 2816, BF), (2816, 1024, BF), (1500, 1500, FP)])
def test_large_tiles(dev, m, n, out):
    """Enough matrices for the 256 x 256 tiles; padded and whole sizes."""
    from zorse_amd import kernels as K
    us = [_matrix(m, n, "noise", i, BF) for i in range(4)]
    outs = K.orthogonalize([u.to(dev) for u in us], dtype=out)
    for u, o in zip(us[:2], outs):
        _near(o, u, out, f"{m} x {n}")


def test_views_and_outs(dev):
    from zorse_amd import kernels as K
    flat = torch.randn(300 * 500 + 7, device=dev)
    wide = torch.randn(200, 900, device=dev).to(BF)
    us = [flat[7:].view(300, 500), wide[:, 300:641]]
    outs = [torch.full((300, 800), 7.0, device=dev, dtype=BF)[:, 100:600],
            torch.empty(200, 341, device=dev, dtype=F4)]
    K.orthogonalize(us, outs=outs)
    plain = K.orthogonalize([us[0].clone()], dtype=BF) + K.orthogonalize([us[1].contiguous()], dtype=F4)
    assert torch.equal(outs[0], plain[0]) and torch.equal(outs[1], plain[1])
    assert bool((outs[0]._base[:, :100] == 7).all()) and bool((outs[0]._base[:, 600:] == 7).all())


def test_scale_zero_and_odd_values(dev):
    from zorse_amd import kernels as K
    u = _matrix(200, 300, "noise", 1)
    for f in (1e-20, 1.0, 1e18):
        # without eps the factor does not depend on the size
        got = K.orthogonalize([(u * f).to(dev)], eps=0.0, dtype=F4)[0]
        ref = _exact(u.double(), eps=0.0)
        assert float((got.cpu().double() - ref).norm()) <= 2e-4 * float(ref.norm())
    zero = torch.zeros(130, 140, device=dev)
    assert not bool(K.orthogonalize([zero])[0].any())
    bad = u.clone()
    bad[3, 4] = math.nan
    good = _matrix(210, 220, "noise", 2)
    a, b = K.orthogonalize([bad.to(dev), good.to(dev)], dtype=BF)
    assert bool(torch.isnan(a).all())
    _near(b, good, BF, "beside a NaN")
    small = K.orthogonalize([(u * 1e-9).to(dev)], dtype=F4)[0]  # eps counts
    ref = _exact(u * 1e-9)
    assert float((small.cpu().double() - ref).norm()) <= 2e-4 * float(ref.norm())


def test_factors_are_near_orthogonal(dev):
    from zorse_amd import kernels as K
    o = K.orthogonalize([_matrix(256, 512, "noise", 3).to(dev)], dtype=F4)[0].cpu().double()
    sv = torch.linalg.svdvals(o)
    assert 0.6 < float(sv.min()) and float(sv.max()) < 1.25
    # other coefficients: the cubic iteration converges to 1
    o = K.orthogonalize([_matrix(96, 160, "noise", 3).to(dev)], steps=12, coefficients=(1.5, -0.5, 0.0),
                        dtype=F4)[0].cpu().double()
    ref = _exact(_matrix(96, 160, "noise", 3), 12, coef=(1.5, -0.5, 0.0))
    # X in 22 bits, each step's roundings grow 1.5 times: 12 steps
    assert float((o - ref).norm()) <= 1.5 ** 12 * 2.0 ** -20 * float(ref.norm())


def _plain_step(p, g, m, mu, lr, wd, nesterov, adjust):
    p, g, m = p.double(), g.double(), m.double()
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    f = 0.2 * math.sqrt(max(p.shape)) if adjust == "match_rms_adamw" else \
        math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
    return p * (1 - lr * wd), m, u, lr * f


@pytest.mark.parametrize("nesterov,adjust,dt", [(True, "original", BF), (False, "match_rms_adamw", F4),
                                                (True, "match_rms_adamw", FP)])
def test_step_of_a_list(dev, nesterov, adjust, dt):
    from zorse_amd import kernels as K
    shapes = [(300, 200), (64, 300), (257, 513), (7, 3)]
    ps = [_matrix(m, n, "noise", i) * 20 for i, (m, n) in enumerate(shapes)]
    gs = [_matrix(m, n, "strong", 9 + i, dt) for i, (m, n) in enumerate(shapes)]
    ms = [_matrix(m, n, "noise", 30 + i) * 0.3 for i, (m, n) in enumerate(shapes)]
    dp, dg, dm = ([t.to(dev) for t in ts] for ts in (ps, gs, ms))
    lows = None if dt == F4 else [p.to(dt) if i != 1 else None for i, p in enumerate(dp)]
    kw = dict(lr=0.02, momentum=0.9, weight_decay=0.1)
    K.muon_multi(dp, dg, dm, lowp_outs=lows, nesterov=nesterov, adjust=adjust, **kw)
    for i, (p, g, m) in enumerate(zip(ps, gs, ms)):
        keep, m2, u, rate = _plain_step(p, g, m, 0.9, 0.02, 0.1, nesterov, adjust)
        # two products and a sum in fp32
        assert bool(((dm[i].cpu().double() - m2).abs() <= 2.0 ** -22 * (m.abs() + g.abs().float())).all())
        ref = _exact(u)
        two = min(u.shape) <= 128
        fmt = float((_rounded(u, two) - ref).norm())
        # u itself is off by 2^-22 of its size, which grows as the small
        # singular values do, by 3.4445^5 at most
        bound = (8 if two else 1.5) * fmt + (A ** 5 * 2.0 ** -22 + math.sqrt(max(u.shape)) * 2.0 ** -22) * float(ref.norm())
        off = float((dp[i].cpu().double() - (keep - rate * ref)).norm())
        assert off <= rate * bound + 2.0 ** -23 * float(p.norm()), i
        if lows is not None and lows[i] is not None:
            assert torch.equal(lows[i], dp[i].to(dt))


def test_captured_and_on_another_stream(dev):
    from zorse_amd import kernels as K
    shapes = [(200, 300), (64, 64), (300, 140)]
    ps, gs, ms = ([torch.randn(s, device=dev) * 0.02 for s in shapes] for _ in range(3))

    def step():
        K.muon_multi(ps, gs, ms, lr=0.01, momentum=0.95, weight_decay=0.01)
        return K.orthogonalize(gs, dtype=BF)

    side = torch.cuda.Stream()
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
        start = [[torch.randn_like(t) * 0.02 for t in ts] for ts in (ps, gs, ms)]
        for ts, xs in zip((ps, gs, ms), start):
            for t, x in zip(ts, xs):
                t.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*ps, *ms, *out)]
        for ts, xs in zip((ps, gs, ms), start):
            for t, x in zip(ts, xs):
                t.copy_(x)
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (*ps, *ms, *want)))


def test_refusals_on_the_gpu(dev):
    from zorse_amd import kernels as K
    a, b = torch.zeros(40, 30, device=dev), torch.zeros(40, 30, device=dev)
    kw = dict(lr=0.1, momentum=0.9, weight_decay=0.0)
    with pytest.raises(ValueError, match="twice"):
        K.muon_multi([a, a], [b, b], [torch.zeros_like(a), torch.zeros_like(a)], **kw)
    with pytest.raises(ValueError, match="overlaps"):
        K.muon_multi([a], [a], [b], **kw)
    with pytest.raises(ValueError, match="overlaps"):
        K.orthogonalize([a], outs=[a])
    with pytest.raises(ValueError, match="column stride"):
        K.orthogonalize([a.t()])
    with pytest.raises(ValueError, match="rows that do not overlap"):
        K.orthogonalize([a[0].expand(40, 30)])
    with pytest.raises(ValueError, match="matrix"):
        K.orthogonalize([a[None]])
    with pytest.raises(ValueError, match="fp32"):
        K.muon_multi([a.half()], [b.half()], [b], **kw)
    with pytest.raises(ValueError, match="shape"):
        K.muon_multi([a], [b[:3]], [torch.zeros_like(a)], **kw)
    with pytest.raises(RuntimeError, match="grows beyond"):
        K.orthogonalize([a], coefficients=(9.0, 0.0, 0.0))
    with pytest.raises(ValueError, match="differ in length"):
        K.muon_multi([a], [], [b], **kw)


def _in_fp32_sums(p, q, run):
    """p q^T of operands in two numbers as the kernels add them: hi hi, hi lo and lo
    hi one after another into fp32 sums, each rounded after every `run` products."""
    acc = torch.zeros(p[0].shape[0], q[0].shape[0], dtype=torch.float64, device=p[0].device)
    for i, j in ((0, 0), (0, 1), (1, 0)):
        for k in range(0, p[0].shape[1], run):
            acc = (acc + p[i][:, k:k + run] @ q[j][:, k:k + run].T.contiguous()).float().double()
    return acc


def _near_on_gpu(got, u, dt, what):
    """_near for large sizes, the references on the GPU.  With an fp32 result the fp32
    sums weigh more than the two numbers (for a few strong directions over noise,
    whose small values grow 400 times over the steps), so the steps are taken with
    them: an instruction adds 32 products to a sum; it is allowed to round it after
    every four, and the norm of the error may be 1.5 times that of such steps.  X is
    scaled by 2^15, G and P by S and R."""
    got, u = got.double(), u.double()
    ref = _exact(u)
    norm = float(ref.norm())
    if dt == F4:
        sx, tall = 2.0 ** 15, u.shape[0] > u.shape[1]
        x = u * float(torch.tensor(sx / (float(u.norm()) + 1e-7), dtype=F4))
        hi, lo = _two((x.T if tall else x).contiguous())
        for _ in range(5):
            g = _two(_in_fp32_sums((hi, lo), (hi, lo), 4) * (S / sx) ** 2)
            p = _two(C * R / S ** 4 * _in_fp32_sums(g, g, 4) + B * R / S ** 2 * (g[0] + g[1]))
            px = _in_fp32_sums(p, (hi.T.contiguous(), lo.T.contiguous()), 4)
            hi, lo = _two((A * (hi + lo) + px / R).float().double())
        fmt = (hi + lo) / sx
        fmt = fmt.T if tall else fmt
    else:
        fmt = _rounded(u, False)
    bound = 1.5 * float((fmt - ref).norm()) + torch.finfo(dt).eps / 2 * norm
    off = float((got - ref).norm())
    assert off <= bound, f"{what}: {off / norm:.2e} off, {bound / norm:.2e} allowed"
    assert float((got - ref).abs().max()) <= 40 * bound / math.sqrt(ref.numel()) + \
        torch.finfo(dt).eps * float(ref.abs().max())


@pytest.mark.parametrize("m,n", [(2048, 2048), (2816, 1024)])
def test_fp32_results_of_large_matrices(dev, m, n):
    """Eight strong directions over noise."""
    from zorse_amd import kernels as K
    g = torch.Generator().manual_seed(m)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    u = (1e-3 * (mk(m, 8) @ mk(8, n) + 0.01 * mk(m, n))).float().to(dev)
    _near_on_gpu(K.orthogonalize([u])[0], u, F4, f"{m} x {n}")


@pytest.mark.parametrize("m,n", [(200, 230), (90, 60)])
def test_small_elements_keep_their_bits(dev, m, n):
    """One element in each row and column, so that no sum is rounded and each goes
    its own way: z <- a z + P z, P = b z^2 + c z^4.  A step rounds an element in two
    numbers (2^-23 of itself, where the second is a normal one: scaled by 2^15, from
    2^-18 on), P twice so (P and z^2: 2^-22 of it at most) and in fp32, the product and
    the sum (2^-24 of their magnitudes).  Relative to a z + P z that is below 2^-21 while
    P is small, and where |P| is up to 3.1, in the last two steps, (a + |P|) / (a + P) <
    6 times as much over two: 3 early steps and the scaling 4 2^-21, two late ones 6 2^-21."""
    from zorse_amd import kernels as K
    k = min(m, n)
    g = torch.Generator().manual_seed(k)
    z = torch.logspace(0, -4.5, k, dtype=torch.float64) * (1 - 2 * (torch.arange(k) % 2)) * 0.4
    rows, cols = torch.randperm(m, generator=g)[:k], torch.randperm(n, generator=g)[:k]
    u = torch.zeros(m, n)
    u[rows, cols] = z.float()
    got = K.orthogonalize([u.to(dev)])[0].cpu().double()
    ref = _exact(u)
    small = (u[rows, cols].double() / u.double().norm()).abs()
    small = (small < 0.002) & (small > 2.0 ** -18)
    assert int(small.sum()) > k // 3
    x, y = got[rows, cols][small], ref[rows, cols][small]
    assert float(((x - y) / y).abs().max()) <= 10 * 2.0 ** -21
    got[rows, cols] = 0
    assert not bool(got.any())


def test_tiny_matrices_without_eps(dev):
    """The scale of X over the norm leaves fp32's range."""
    from zorse_amd import kernels as K
    u = _matrix(200, 300, "noise", 1) * 1e-34
    got = K.orthogonalize([u.to(dev)], eps=0.0)[0].cpu().double()
    ref = _exact(u.double(), eps=0.0)
    assert float((got - ref).norm()) <= 2e-4 * float(ref.norm())


def test_symmetric_products_in_large_tiles(dev):
    """Sides of 2305 and more, in launches of over 512 tiles of 128 x 128 even for G
    and P: 256 x 256 tiles and their transposed copies, whole and padded."""
    from zorse_amd import kernels as K
    for m, n in ((2500, 2600), (2560, 2560)):
        us = [_matrix(m, n, "noise", 3 * m + i, BF).to(dev) for i in range(3)]
        for u, o in zip(us, K.orthogonalize(us, dtype=FP)):
            _near_on_gpu(o, u, FP, f"{m} x {n}")

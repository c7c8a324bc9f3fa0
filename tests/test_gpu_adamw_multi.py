"""AdamW over lists of tensors: with 32-bit moments the bits of a step for
each, with 8-bit moments the format's own arithmetic and the update's formula
in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32
H = dict(lr=2e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.05)
U = 2.0 ** -24
SIZES = [1, 3, 255, 256, 257, 1023, 1024, 1025, 70001, 0, 12]


def _lists(dev, sizes, gdt, ldt, seed=0, odd=True):
    """fp32 parameters, gradients, moments and copies; each tensor one element
    after a 256-byte boundary (``odd``), as views of flat shards lie."""
    g = torch.Generator().manual_seed(seed)

    def put(t, dt):
        room = torch.empty(t.numel() + 1, dtype=dt, device=dev)[int(odd):][:t.numel()]
        return room.copy_(t)

    p = [put(torch.randn(n, generator=g), F4) for n in sizes]
    gr = [put(torch.randn(n, generator=g) * 10 ** (-6 * torch.rand(n, generator=g)), gdt)
          for n in sizes]
    m = [put(torch.randn(n, generator=g) * 1e-3, F4) for n in sizes]
    v = [put(torch.rand(n, generator=g) * 1e-5, F4) for n in sizes]
    low = [put(torch.zeros(n), ldt) if ldt is not None and i % 4 else None
           for i, n in enumerate(sizes)]
    return p, gr, m, v, low


@pytest.mark.parametrize("gdt", [F4, BF, FP])
@pytest.mark.parametrize("ldt", [None, BF, FP, F4])
def test_bits_of_single_steps(dev, gdt, ldt):
    from zorse_amd import kernels
    sizes = SIZES * 11  # more than one launch
    p, gr, m, v, low = _lists(dev, sizes, gdt, ldt)
    steps = [1 + i % 5 for i in range(len(sizes))]
    want = [[None if t is None else t.clone() for t in ts] for ts in (p, m, v, low)]
    for i, t in enumerate(steps):
        if sizes[i]:
            kernels.adamw_step(want[0][i], gr[i].clone(), want[1][i], want[2][i],
                               lowp_out=want[3][i], step=t, **H)
    kernels.adamw_multi(p, gr, m, v, steps, lowp_outs=low, **H)
    for got, ref in zip((p, m, v, low), want):
        assert all(torch.equal(a, b) for a, b in zip(got, ref) if a is not None)


def test_mixed_types_and_neighbours_untouched(dev):
    """One launch of tensors whose gradients and copies differ in type, in one
    buffer with guards between them."""
    from zorse_amd import kernels
    buf = torch.full((4, 4000), 7.0, device=dev)
    cut = [(5, 700), (706, 1730), (1735, 3999)]
    p, g0, m, v = ([buf[r, a:b] for a, b in cut] for r in range(4))
    for t in (*p, *g0, *m, *v):
        t.copy_(torch.rand(t.numel(), device=dev))
    gr = [g0[0].bfloat16(), g0[1].half(), g0[2]]
    low = [torch.empty_like(p[0], dtype=FP), None, torch.empty_like(p[2], dtype=BF)]
    want = [(a.clone(), c.clone(), d.clone()) for a, c, d in zip(p, m, v)]
    kernels.adamw_multi(p, gr, m, v, [3, 3, 4], lowp_outs=low, **H)
    for i, (a, c, d) in enumerate(want):
        kernels.adamw_step(a, gr[i], c, d, step=[3, 3, 4][i], **H)
        assert torch.equal(a, p[i]) and torch.equal(c, m[i]) and torch.equal(d, v[i])
    assert torch.equal(low[0], p[0].half()) and torch.equal(low[2], p[2].bfloat16())
    for a, b in ((0, 5), (700, 706), (1730, 1735), (3999, 4000)):
        assert bool((buf[:, a:b] == 7.0).all())


# ------------------------------------------------------------ 8-bit moments --

def _values(codes, base, low):
    c = codes.astype(np.int64) & low
    b = np.repeat(base.astype(np.int64), 256)[:c.size]
    v = np.where(c > 0, (c + b) << 20, 0).astype(np.uint32).view(np.float32)
    return np.where(codes > low, -v, v) if low == 127 else v


def _codes(r, top, least):
    """(codes, base) of the integers r (-1: a moment of zero)."""
    n = r.size
    rows = np.concatenate((r, np.full(-n % 256, -1))).reshape(-1, 256)
    base = np.maximum(rows.max(1) - top, 0)
    c = np.maximum(rows - base[:, None], least)
    return np.where(rows < 0, 0, c).reshape(-1)[:n].astype(np.uint8), base.astype(np.int16)


def _random20(seed, n):
    with np.errstate(over="ignore"):
        x = np.arange(n, dtype=np.uint32) * np.uint32(0x9E3779B1) + np.uint32(seed)
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
        return ((x ^ (x >> np.uint32(16))) >> np.uint32(12)).astype(np.int64)


def _moments(m, v, g):
    """The update's moments with its roundings: fp32 operands, one rounding of
    each fused product and sum (exact in 64 bits up to 2^-53)."""
    f = np.float32
    w1, b2, w2 = f(1 - H["beta1"]), f(H["beta2"]), f(1 - H["beta2"])
    m2 = (np.float64(w1) * (g - m).astype(np.float64) + m).astype(f)
    v2 = (np.float64(w2) * (g * g).astype(np.float64) + (v * b2)).astype(f)
    return m2, v2


def _expected(codes_m, codes_v, base, g, seed):
    m, v = _moments(_values(codes_m, base[:, 0], 127), _values(codes_v, base[:, 1], 255), g)
    bits = (m.view(np.uint32) & 0x7FFFFFFF).astype(np.int64)
    cm, bm = _codes((bits + 0x7FFFF + (bits >> 20 & 1)) >> 20, 127, 0)
    cm = np.where((m < 0) & (cm > 0), cm | 128, cm).astype(np.uint8)
    bits = v.view(np.uint32).astype(np.int64)
    cv, bv = _codes(np.where(v > 0, (bits + _random20(seed, v.size)) >> 20, -1), 255, 1)
    return m, v, cm, cv, np.stack((bm, bv), 1)


def _state(dev, sizes):
    return ([torch.zeros(n, dtype=torch.uint8, device=dev) for n in sizes],
            [torch.zeros(n, dtype=torch.uint8, device=dev) for n in sizes],
            [torch.zeros(-(-n // 256), 2, dtype=torch.int16, device=dev) for n in sizes])


@pytest.mark.parametrize("gdt,ldt", [(F4, None), (BF, BF), (FP, FP), (BF, F4)])
def test_eight_bit_steps(dev, gdt, ldt):
    """Several steps of many tensors: codes and bases to the bit, parameters
    against the formula in 64 bits from the states held before the step."""
    from zorse_amd import kernels
    sizes = SIZES * 9
    p, gr, _, _, low = _lists(dev, sizes, gdt, ldt, seed=1)
    cm, cv, base = _state(dev, sizes)
    for step in (1, 2, 3):
        for i, t in enumerate(gr):
            t.mul_(0.5 if i % 2 else -1.7)
            t[:: 3 + step] = 0
        before = [[t.cpu() for t in ts] for ts in (p, cm, cv, base)]
        seeds = [1000 * step + 77 * i for i in range(len(sizes))]
        steps = [step + i % 3 for i in range(len(sizes))]
        kernels.adamw8_multi(p, gr, cm, cv, base, steps, seeds=seeds, lowp_outs=low, **H)
        ms, vs = kernels.adamw8_values(cm, cv, base)
        mb, _ = kernels.adamw8_values(cm, cv, base, dtype=BF)
        for i, n in enumerate(sizes):
            if not n:
                continue
            g = gr[i].float().cpu().numpy()
            p0, m0, v0, b0 = (before[k][i].numpy() for k in range(4))
            m, v, wm, wv, wb = _expected(m0, v0, b0, g, seeds[i])
            assert np.array_equal(cm[i].cpu().numpy(), wm)
            assert np.array_equal(cv[i].cpu().numpy(), wv)
            assert np.array_equal(base[i].cpu().numpy(), wb)
            assert np.array_equal(ms[i].cpu().numpy(), _values(wm, wb[:, 0], 127))
            assert np.array_equal(vs[i].cpu().numpy(), _values(wv, wb[:, 1], 255))
            assert torch.equal(mb[i].float(), ms[i])  # bf16 holds every value
            t = steps[i]
            g, mo = g.astype(np.float64), _values(m0, b0[:, 0], 127).astype(np.float64)
            vo = _values(v0, b0[:, 1], 255).astype(np.float64)
            m64 = H["beta1"] * mo + (1 - H["beta1"]) * g
            v64 = H["beta2"] * vo + (1 - H["beta2"]) * g * g
            den = np.sqrt(v64 / (1 - H["beta2"] ** t)) + H["eps"]
            size = H["lr"] / (1 - H["beta1"] ** t)
            ref = p0.astype(np.float64) * (1 - H["lr"] * H["weight_decay"]) - size * m64 / den
            # p: two roundings and the decay's; m: u of its two terms; the rest 8 u
            tol = U * (3 * np.abs(p0) + 16 * size * (np.abs(mo) + np.abs(g)) / den)
            assert bool((np.abs(p[i].cpu().numpy() - ref) <= tol).all())
            if low[i] is not None:
                assert torch.equal(low[i], p[i].to(low[i].dtype))


def test_second_moment_keeps_its_mean(dev):
    """A moment between two codes goes up with the fraction's probability: the
    mean of n draws is off by at most 6 sigma of a step, sigma^2 = f (1 - f) / n;
    to nearest it would be off by up to half a step."""
    from zorse_amd import kernels
    n = 1 << 18
    for f in (0.03, 0.5, 0.9):
        v = 8.0 + f  # between the codes of 8 and 9, a step of 1
        g = torch.full((n,), (v / (1 - H["beta2"])) ** 0.5, device=dev)
        cm, cv, base = _state(dev, [n])
        kernels.adamw8_multi([torch.zeros(n, device=dev)], [g], cm, cv, base, [1], seeds=[3], **H)
        vs = kernels.adamw8_values(cm, cv, base)[1][0].double()
        assert set(vs.unique().tolist()) == {8.0, 9.0}
        # 2^-20 of a step: the random bits; 1e-5: g, g^2 and the product in fp32
        assert abs(float(vs.mean()) - v) <= 6 * (f * (1 - f) / n) ** 0.5 + 2.0 ** -20 + 1e-5


def test_ranges_zeros_and_non_finite_gradients(dev):
    """Elements 2^20 and more apart share a block; one of zero stays zero; a
    moment below the block's range is held at its least, never at zero; NaN and
    infinity stay in their element."""
    from zorse_amd import kernels
    n = 512
    g = torch.full((n,), 1e-9)
    g[:4] = torch.tensor([1e3, 0.0, -1e-3, 2.0 ** -75])
    g[256:] = 1.0
    g[300], g[301] = float("nan"), float("inf")
    p = torch.ones(n, device=dev)
    cm, cv, base = _state(dev, [n])
    kernels.adamw8_multi([p], [g.to(dev)], cm, cv, base, [1], seeds=[0], **H)
    m, v = (t[0].cpu() for t in kernels.adamw8_values(cm, cv, base))
    # (2^-75)^2 = 2^-150, half of fp32's smallest number, is 0 in fp32 (to even)
    square = g * g
    assert float(square[3]) == 0 and int((square == 0).sum()) == 2
    assert float(m[1]) == 0 and float(v[1]) == 0 and bool((v[square != 0] > 0).all())
    want = (1 - H["beta1"]) * g.double()
    # half a step of 4 bits; the fp32 before it
    assert bool(((m[256:300].double() - want[256:300]).abs()
                 <= (2.0 ** -4 + 2.0 ** -20) * want[256:300].abs()).all())
    assert abs(float(m[0]) - float(want[0])) <= 2.0 ** -4 * float(want[0])
    assert float(m[2]) == 0 and float(m[4]) == 0  # 2^16 below the block's largest
    ok = torch.ones(n, dtype=torch.bool)
    ok[[300, 301]] = False
    assert bool(p.cpu()[ok].isfinite().all()) and not bool(p.cpu()[~ok].isfinite().any())
    # v4 is held above its own value, so its update is smaller than exact
    assert float(v[4]) >= (1 - H["beta2"]) * 1e-18


def test_tiny_moments_have_no_base(dev):
    """Moments at the bottom of fp32's range: codes counted from 0."""
    from zorse_amd import kernels
    g = (torch.rand(777) * 1e-18).numpy()
    g[::5] = 0
    cm, cv, base = _state(dev, [777])
    p = torch.zeros(777, device=dev)
    for seed in (1, 2):
        b = [t[0].cpu().numpy() for t in (cm, cv, base)]
        kernels.adamw8_multi([p], [torch.from_numpy(g).to(dev)], cm, cv, base, [seed],
                             seeds=[seed], **H)
        _, _, wm, wv, wb = _expected(b[0], b[1], b[2], g, seed)
        assert int(wb[:, 1].max()) == 0
        assert np.array_equal(cm[0].cpu().numpy(), wm)
        assert np.array_equal(cv[0].cpu().numpy(), wv)
        assert np.array_equal(base[0].cpu().numpy(), wb)


def test_refusals(dev):
    from zorse_amd import kernels
    p, gr, m, v, _ = _lists(dev, [8, 16], F4, None)
    with pytest.raises(ValueError, match="twice"):
        kernels.adamw_multi([p[0], p[0]], [gr[0]] * 2, [m[0]] * 2, [v[0]] * 2, [1, 1], **H)
    for bad in ((p, gr[::-1], m, v), (p, gr, m[::-1], v), (p, [gr[0], gr[1].double()], m, v),
                ([p[0], p[1].bfloat16()], gr, m, v), (p, gr, m, [v[0], v[1].cpu()])):
        with pytest.raises(ValueError):
            kernels.adamw_multi(*bad, [1, 1], **H)
    with pytest.raises(RuntimeError, match="step"):
        kernels.adamw_multi(p, gr, m, v, [1, 0], **H)
    cm, cv, base = _state(dev, [8, 16])
    with pytest.raises(ValueError):
        kernels.adamw8_multi(p, gr, m, v, base, [1, 1], seeds=[0, 0], **H)
    with pytest.raises(ValueError):
        kernels.adamw8_multi(p, gr, cm, cv, [base[0], base[1].repeat(2, 1)], [1, 1], seeds=[0, 0],
                             **H)


def test_optimizer_steps_lists(dev):
    """step() over several parameters has the bits of step_param on each, in
    both states; 8-bit states resume from a checkpoint with the same bits."""
    from zorse_amd.optim import FusedAdamW
    torch.manual_seed(0)
    shapes = [(33, 70), (5,), (1000,), (64, 8)]
    for bits in (32, 8):
        for dt in (F4, BF):
            a = [torch.nn.Parameter(torch.randn(s, device=dev).to(dt)) for s in shapes]
            b = [torch.nn.Parameter(t.detach().clone()) for t in a]
            fired = []
            oa, ob = (FusedAdamW(x, lr=1e-2, state_bits=bits) for x in (a, b))
            oa.add_step_hook(a[1], fired.append)
            for _ in range(2):
                ver = a[0]._version
                for x, y in zip(a, b):
                    x.grad = torch.randn_like(x)
                    y.grad = x.grad.clone()
                oa.step()
                for y in b:
                    ob.step_param(y)
                assert a[0]._version > ver
            assert len(fired) == 2 and fired[0] is a[1]
            for x, y in zip(a, b):
                assert torch.equal(x, y)
                assert all(torch.equal(s, t) for s, t in zip(oa.moments(x), ob.moments(y)))
            c = [torch.nn.Parameter(t.detach().clone()) for t in a]
            oc = FusedAdamW(c, state_bits=bits)
            oc.load_state_dict(oa.state_dict())
            for x, z in zip(a, c):
                x.grad = torch.randn_like(x)
                z.grad = x.grad.clone()
            oa.step()
            oc.step()
            assert all(torch.equal(x, z) for x, z in zip(a, c))


def test_large_tensors_among_small_ones(dev):
    """Tensors above the size that is launched alone, and elements past 2^31 of
    an 8-bit state, whose random bits go by the whole index."""
    from zorse_amd import kernels
    sizes = [(6 << 20) + 5, 7, 6 << 20]
    p, gr, m, v, low = _lists(dev, sizes, BF, BF)
    want = [[t.clone() for t in ts] for ts in (p, m, v)]
    for i in range(3):
        kernels.adamw_step(want[0][i], gr[i].clone(), want[1][i], want[2][i], step=2, **H)
    kernels.adamw_multi(p, gr, m, v, [2, 2, 2], lowp_outs=low, **H)
    for got, ref in zip((p, m, v), want):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    del p, gr, m, v, low, want
    n, tail = (1 << 31) + 700, 700
    p = torch.zeros(n, device=dev)
    g = torch.zeros(n, device=dev, dtype=BF)
    g[-tail:] = torch.linspace(-1, 1, tail)
    cm, cv, base = _state(dev, [n])
    kernels.adamw8_multi([p], [g], cm, cv, base, [1], seeds=[17], **H)
    gt = g[-tail:].float().cpu().numpy()
    z = np.zeros(tail, np.uint8)
    with np.errstate(over="ignore"):  # what 2^31 adds to the index's product
        seed = int(np.uint32(17) + np.uint32(1 << 31) * np.uint32(0x9E3779B1))
    _, _, wm, wv, wb = _expected(z, z, np.zeros((3, 2), np.int16), gt, seed)
    assert np.array_equal(cm[0][-tail:].cpu().numpy(), wm)
    assert np.array_equal(cv[0][-tail:].cpu().numpy(), wv)
    assert np.array_equal(base[0][-3:].cpu().numpy(), wb)
    assert not bool(cm[0][:-tail].any()) and not bool(cv[0][:-tail].any())
    assert not bool(p[:-tail].any()) and bool(p[-tail:].all())


def test_parameters_that_share_memory(dev):
    """Overlapping parameters: refused in a list, stepped one after another by
    the optimizer, as by steps of each; neighbours that only touch are a list.
    A list that is refused leaves the step counts."""
    from zorse_amd import kernels
    from zorse_amd.optim import FusedAdamW
    flat = torch.linspace(-1, 1, 64, device=dev)
    p, gr, m, v, _ = _lists(dev, [40, 40], F4, None)
    with pytest.raises(ValueError, match="overlap"):
        kernels.adamw_multi([flat[:40], flat[24:]], gr, m, v, [1, 1], **H)
    kernels.adamw_multi([flat[:24], flat[24:]], [gr[0][:24], gr[1]], [m[0][:24], m[1]],
                        [v[0][:24], v[1]], [1, 1], **H)
    for bits in (32, 8):
        got, want = flat.clone(), flat.clone()
        a, b = ([torch.nn.Parameter(t[:40]), torch.nn.Parameter(t[24:])] for t in (got, want))
        oa, ob = (FusedAdamW(x, lr=1e-2, state_bits=bits) for x in (a, b))
        for x, y in zip(a, b):
            assert x.data_ptr() in (got.data_ptr(), got[24:].data_ptr())
            x.grad = torch.randn_like(x)
            y.grad = x.grad.clone()
        oa.step()
        for y in b:
            ob.step_param(y)
        assert torch.equal(got, want)
        c = [torch.nn.Parameter(torch.zeros(8, device=dev)) for _ in range(2)]
        oc = FusedAdamW(c, state_bits=bits)
        for x in c:
            x.grad = torch.ones_like(x)
        oc.param_groups[0]["lr"] = float("nan")
        with pytest.raises(RuntimeError, match="range"):
            oc.step()
        assert [oc.state[x]["step"] for x in c] == [0, 0] and not bool(c[0].any())

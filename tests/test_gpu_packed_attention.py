"""Attention over packed sequences against the formulas in 64 bits.

With h half a step of the storage type, eps / 2, and u = 2^-24: a score is a sum
of d products and a scaling, off by (d + 3) u of the sum of its products'
magnitudes; its exponential adds 2^-21 of itself (exp2 of the hardware, the
reference maximum's and the scale's roundings), so a probability is off by
e = (d + 8) u max_j scale |q||k_j| + 2^-21 of itself, numerator and denominator:
twice that.  It is rounded to the type before it is summed with V (h), sums of n
terms cost n u of their magnitudes, the result is rounded once more (h):
  |dO| <= (h + 2e + n u) P|V| + h |O|.
delta is the sum of dO times the O that was stored: off by |dO| times that
bound, D in all, and by d u of its magnitudes.  dS is rounded once:
  |d dS| <= (h + 2e) |dS| + P (D + (d + 3) u |dO||V^T|),
and dQ, dK, dV carry h of the operands that are rounded, n u of their sums'
magnitudes and half a step of themselves.
Relative steps end where a type's normal range does: a probability below 2^-126
is 0 in fp32 (exp2 of the hardware gives no subnormals), one or a dS below 2^-14
in fp16 is off by up to 2^-24 (half a subnormal step, and another half for what
the conversion may cut), and in bf16 by up to 2^-126.  With w that
number, the sum of a row's weights relative to its reference maximum being at
least 1, P V is off by w of the magnitudes of V's rows that are seen, P^T dO by w
of dO's, dS by w (1 + |dP - delta|)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _half(dt):
    return 0.0 if dt == F4 else torch.finfo(dt).eps / 2


def _reference(q, k, v, do, offsets, causal, window, scale, dt):
    """[(value, bound)] of o, dq, dk, dv, and lse."""
    T, H, d = q.shape
    Hk = k.shape[1]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    h, step = _half(dt), torch.finfo(dt).eps / 2
    low = 2.0 ** -24 if dt == FP else 2.0 ** -126
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, k))
    bo, bq, bk, bv = (torch.zeros_like(t) for t in (q, q, k, k))
    lse = torch.full((H, T), -math.inf, dtype=torch.float64)
    for lo, hi in zip(offsets, offsets[1:]):
        n = hi - lo
        if n == 0:
            continue
        gap = torch.arange(n)[:, None] - torch.arange(n)[None]
        hidden = (gap < 0) if causal else torch.zeros(n, n, dtype=torch.bool)
        if window:
            hidden = hidden | (gap >= window)
        for x in range(H):
            g = x * Hk // H
            a, b, c, up = q[lo:hi, x], k[lo:hi, g], v[lo:hi, g], do[lo:hi, x]
            s = (a @ b.T * scale).masked_fill(hidden, -math.inf)
            lse[x, lo:hi] = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1)
            mag = (a.abs() @ b.abs().T * scale).masked_fill(hidden, 0)
            e = 2 * ((d + 8) * U * mag.amax(1, keepdim=True) + 2.0 ** -21)
            y = p @ c
            o[lo:hi, x] = y
            seen = (~hidden).double()
            by = (h + e + (n + 2) * U) * (p @ c.abs()) + step * y.abs() + low * (seen @ c.abs())
            bo[lo:hi, x] = by
            delta = (up * y).sum(1, keepdim=True)
            dp = up @ c.T
            ds = p * (dp - delta)
            off = (up.abs() * (by + d * U * y.abs())).sum(1, keepdim=True)
            bds = (h + e) * ds.abs() + p * (off + (d + 3) * U * (up.abs() @ c.abs().T))
            bds = bds + low * seen * (1 + (dp - delta).abs())
            # the roundings' sums, then the others'
            dq[lo:hi, x] = ds @ b * scale
            bq[lo:hi, x] += ((bds + n * U * ds.abs()) @ b.abs()) * scale
            dk[lo:hi, g] += ds.T @ a * scale
            m = n * H // Hk
            bk[lo:hi, g] += ((bds + m * U * ds.abs()).T @ a.abs()) * scale
            dv[lo:hi, g] += p.T @ up
            bv[lo:hi, g] += ((h + e + m * U) * p + low * seen).T @ up.abs()
    out = []
    for t, bound in ((o, bo), (dq, bq + step * dq.abs()), (dk, bk + step * dk.abs()),
                     (dv, bv + step * dv.abs())):
        out.append((t, bound * (1 + 2 * step) + torch.finfo(dt).tiny))
    return out, lse


def _inputs(T, H, Hk, d, dt, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: (torch.randn(*s, generator=g) * std).to(dt)  # noqa: E731
    return mk(T, H, d), mk(T, Hk, d), mk(T, Hk, d), mk(T, H, d)


def _run(dev, q, k, v, do, offsets, causal, window, scale=None):
    from zorse_amd import functional as F
    q, k, v = (t.detach().to(dev).requires_grad_() for t in (q, k, v))
    seqs = F.PackedSequences(torch.tensor(offsets, dtype=torch.int32).to(dev), q.shape[0])
    o = F.packed_attention(q, k, v, seqs, causal=causal, window=window, scale=scale)
    grads = torch.autograd.grad(o, (q, k, v), do.to(dev))
    return [o.detach(), *grads]


def _near(got, want, what, rows=slice(None)):
    for name, x, (ref, bound) in zip(("o", "dq", "dk", "dv"), got, want):
        x, ref, bound = x.cpu().double()[rows], ref[rows], bound[rows]
        bad = ~((x - ref).abs() <= bound)
        assert not bool(bad.any()), (
            f"{what} {name}: {int(bad.sum())} of {bad.numel()}, "
            f"worst {float(((x - ref).abs() / bound).max()):.2f} of the bound")


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


CASES = [
    # lengths, padding, heads, key heads, d, causal, window, type
    ((1,), 0, 1, 1, 64, True, 0, BF),
    ((1, 1, 0, 1), 0, 2, 1, 128, True, 0, FP),
    ((0, 0), 5, 2, 2, 64, True, 0, BF),
    ((3, 17, 45), 1, 4, 2, 64, True, 0, BF),
    ((31, 1, 32, 33, 0, 63), 3, 3, 3, 128, True, 0, BF),
    ((129, 255, 257, 64), 0, 8, 8, 128, True, 0, FP),
    ((700, 5, 300), 19, 16, 8, 128, True, 0, BF),
    ((513, 1, 1, 1, 1, 511), 0, 5, 1, 64, False, 0, BF),
    ((400, 37), 0, 4, 2, 128, False, 0, FP),
    ((900, 100), 11, 4, 4, 64, True, 100, FP),
    ((640, 321), 0, 6, 2, 128, True, 1, BF),
    ((640, 321), 0, 6, 2, 128, True, 65, BF),
    ((300, 300), 7, 2, 2, 100, True, 0, BF),
    ((129, 333), 2, 4, 1, 80, False, 0, FP),
    ((65, 130), 0, 3, 1, 2, True, 0, BF),
    ((65, 130), 9, 3, 3, 18, True, 40, FP),
    ((200, 61), 0, 2, 1, 34, False, 0, BF),
    ((200, 61), 0, 4, 2, 62, True, 0, FP),
    ((150, 90), 4, 2, 2, 126, True, 0, BF),
    ((37, 200), 4, 4, 2, 64, True, 0, F4),
    ((300, 1, 0, 70), 4, 2, 1, 128, False, 0, F4),
    ((129, 64), 0, 3, 1, 99, True, 50, F4),
    ((5,) * 100, 12, 2, 2, 64, True, 0, BF),
]


@pytest.mark.parametrize("lengths,pad,H,Hk,d,causal,window,dt", CASES)
def test_against_64_bits(dev, lengths, pad, H, Hk, d, causal, window, dt):
    offsets = _offsets(lengths)
    T = offsets[-1] + pad
    q, k, v, do = _inputs(T, H, Hk, d, dt, T + d)
    want, lse = _reference(q, k, v, do, offsets, causal, window, 1 / math.sqrt(d), dt)
    got = _run(dev, q, k, v, do, offsets, causal, window)
    _near(got, want, "packed")
    for x in got:
        assert not bool(x[offsets[-1]:].any())  # padding: zeros
    from zorse_amd import functional as F, kernels as K
    seqs = F.PackedSequences(offsets, T, device=dev)
    o, l = K.attn_packed_fwd(q.to(dev), k.to(dev), v.to(dev), seqs.plan, causal=causal, window=window)
    assert torch.equal(o, got[0])
    l = l.cpu().double()
    fine = torch.isfinite(lse)
    assert torch.equal(fine, torch.isfinite(l))
    # scores up to |q||k| / sqrt(d), about sqrt(d), summed in fp32
    assert bool(((l - lse)[fine].abs() <= (d + 16) * U * 8 * (d + lse[fine].abs())).all())
    assert torch.equal(seqs.positions.cpu(), torch.tensor(
        [i for n in lengths for i in range(n)] + [0] * pad))


# more blocks than the chip holds at once, where a block is one group of waves
MANY = [
    ((600, 1, 370), 40, 32, 32, 64, True, 0, BF),
    ((600, 1, 370), 40, 32, 8, 128, True, 0, FP),
    ((700, 300), 3, 32, 8, 64, True, 200, FP),
    ((700, 300), 3, 96, 24, 64, True, 200, BF),  # two query heads a sum
    ((333, 600), 3, 32, 32, 100, False, 0, BF),
    ((555, 401), 3, 34, 34, 64, True, 0, F4),
    ((555, 401), 3, 36, 36, 99, True, 300, F4),
]


@pytest.mark.parametrize("lengths,pad,H,Hk,d,causal,window,dt", MANY)
def test_launches_of_many_blocks(dev, lengths, pad, H, Hk, d, causal, window, dt):
    test_against_64_bits(dev, lengths, pad, H, Hk, d, causal, window, dt)


@pytest.mark.parametrize("dt,d", [(BF, 128), (FP, 64), (BF, 72), (F4, 64)])
@pytest.mark.parametrize("scale", [0.02, 1.5])
def test_scales_and_large_scores(dev, dt, d, scale):
    offsets = [0, 90, 260]
    q, k, v, do = _inputs(260, 2, 1, d, dt, 5, 2.0)
    want, _ = _reference(q, k, v, do, offsets, True, 0, scale, dt)
    _near(_run(dev, q, k, v, do, offsets, True, 0, scale), want, f"scale {scale}")


@pytest.mark.parametrize("dt,d", [(BF, 128), (FP, 64), (BF, 100), (F4, 64)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_odd_values_stay_in_their_rows(dev, dt, d, value):
    """Other sequences, later tokens and padding hold NaN or infinities."""
    offsets, T = [0, 70, 150, 200], 230
    q, k, v, do = _inputs(T, 4, 2, d, dt, 11)
    want, _ = _reference(q, k, v, do, offsets, True, 0, 1 / math.sqrt(d), dt)
    for t in (q, k, v, do):
        t[70:150] = value  # the middle sequence
        t[200:] = value    # padding
    got = _run(dev, q, k, v, do, offsets, True, 0)
    keep = torch.tensor([*range(70), *range(150, 200)])
    _near(got, want, "neighbours", keep)
    for x in got:
        assert not bool(x[200:].any())
    assert not bool(torch.isfinite(got[0][70:150]).any())
    # a later token's key and value reach no earlier query
    q, k, v, do = _inputs(T, 4, 2, d, dt, 12)
    want, _ = _reference(q, k, v, do, offsets, True, 0, 1 / math.sqrt(d), dt)
    k[60:70] = value
    v[60:70] = value
    got = _run(dev, q, k, v, do, offsets, True, 0)
    _near(got[:2], want[:2], "earlier queries", torch.tensor([*range(60), *range(70, 200)]))
    # a query's own infinities reach no key that it does not see
    q, k, v, do = _inputs(T, 4, 2, d, dt, 13)
    want, _ = _reference(q, k, v, do, offsets, True, 0, 1 / math.sqrt(d), dt)
    q[3] = value
    do[3] = value
    got = _run(dev, q, k, v, do, offsets, True, 0)
    _near(got, want, "later keys", torch.tensor([*range(4, 200)]))


@pytest.mark.parametrize("dt,H,d", [(BF, 4, 128), (FP, 4, 64), (BF, 4, 100), (FP, 32, 64), (F4, 48, 64)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_odd_values_in_long_runs(dev, dt, H, d, value):
    """The same where blocks are taken in two groups of waves, and where they are many."""
    offsets, T = [0, 300, 420, 800], 870
    q, k, v, do = _inputs(T, H, H // 2, d, dt, 14)
    want, _ = _reference(q, k, v, do, offsets, True, 0, 1 / math.sqrt(d), dt)
    for t in (q, k, v, do):
        t[300:420] = value
        t[800:] = value
    got = _run(dev, q, k, v, do, offsets, True, 0)
    _near(got, want, "neighbours", torch.tensor([*range(300), *range(420, 800)]))
    for x in got:
        assert not bool(x[800:].any())
    assert not bool(torch.isfinite(got[0][300:420]).any())


def test_no_weight_is_nan(dev):
    """Every visible score -inf: the softmax has no value."""
    q, k, v, do = _inputs(40, 1, 1, 64, BF, 1)
    q[:] = 1.0
    k[:] = -math.inf
    got = _run(dev, q, k, v, do, [0, 40], True, 0)
    assert bool(torch.isnan(got[0]).all())


def test_views_of_one_buffer_and_kept_rows(dev):
    from zorse_amd import functional as F, kernels as K
    offsets, T, H, Hk, d = [0, 33, 300], 310, 4, 2, 128
    buf = torch.randn(T, (H + 2 * Hk) * d, device=dev).to(BF)
    q = buf[:, :H * d].unflatten(1, (H, d))
    k = buf[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
    v = buf[:, (H + Hk) * d:].unflatten(1, (Hk, d))
    seqs = F.PackedSequences(offsets, T, device=dev)
    o, lse = K.attn_packed_fwd(q, k, v, seqs.plan)
    o2, lse2 = K.attn_packed_fwd(q.contiguous(), k.contiguous(), v.contiguous(), seqs.plan)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    mine = torch.full_like(o, 7.0)
    K.attn_packed_fwd(q, k, v, seqs.plan, out=mine)
    assert torch.equal(mine[:300], o[:300]) and bool((mine[300:] == 7).all())
    do = torch.randn_like(o)
    grads = K.attn_packed_bwd(q, k, v, o, do, lse, seqs.plan)
    dbuf = torch.full_like(buf, 7.0)
    dq = dbuf[:, :H * d].unflatten(1, (H, d))
    dk = dbuf[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
    dv = dbuf[:, (H + Hk) * d:].unflatten(1, (Hk, d))
    K.attn_packed_bwd(q, k, v, o, do, lse, seqs.plan, dq=dq, dk=dk, dv=dv)
    for a, b in zip((dq, dk, dv), grads):
        assert torch.equal(a[:300], b[:300]) and bool((a[300:] == 7).all())
    # heads at 4-byte addresses, odd views, broadcast heads
    odd = torch.randn(T, H, d + 2, device=dev).to(BF)[:, :, 2:]
    a = F.packed_attention(odd, k, v, seqs)
    assert torch.allclose(a.float(), F.packed_attention(odd.contiguous(), k, v, seqs).float(), atol=2e-2)
    odd = torch.randn(T, H, d + 1, device=dev).to(BF)[:, :, 1:]
    assert torch.equal(F.packed_attention(odd, k, v, seqs),
                       F.packed_attention(odd.contiguous(), k, v, seqs))
    one = k[:, :1].clone().requires_grad_()
    b = F.packed_attention(q, one.expand(T, Hk, d), v, seqs)
    assert torch.equal(b, F.packed_attention(q, one.expand(T, Hk, d).contiguous(), v, seqs))
    two = one.detach().expand(T, Hk, d).contiguous().requires_grad_()
    c = F.packed_attention(q, two, v, seqs)
    dk2 = torch.autograd.grad(c, two, do)[0]
    assert torch.allclose(torch.autograd.grad(b, one, do)[0].float(),
                          dk2.float().sum(1, keepdim=True), rtol=2 ** -7, atol=1e-6)


def test_equal_calls_equal_bits_and_other_streams(dev):
    offsets = [0, 500, 501, 1300]
    q, k, v, do = _inputs(1300, 8, 2, 64, BF, 2)
    one = _run(dev, q, k, v, do, offsets, True, 0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        two = _run(dev, q, k, v, do, offsets, True, 0)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_offsets_that_make_no_sense_stay_in_bounds(dev):
    """Offsets on the GPU are not checked: the plan refers to the run's tokens."""
    from zorse_amd import functional as F
    q, k, v, _ = _inputs(300, 2, 1, 64, BF, 3)
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    for offs in ([0, 900], [0, -5], [0, 250, 100, 300], [7, 100, 300], [0, 2 ** 40, 300], [300],
                 [-9, 5, 5, 4000]):
        seqs = F.PackedSequences(torch.tensor(offs, device=dev), 300)
        start, end = seqs.plan[16:316], seqs.plan[316:616]
        n, at = int(seqs.plan[0]), torch.arange(300, device=dev)
        assert 0 <= n <= 300
        own = at < n
        assert bool(((start >= 0) & (start <= at)).all())
        assert bool((~own | ((end > at) & (end <= n))).all()) and bool((own | (end == at)).all())
        assert F.packed_attention(q, k, v, seqs).shape == q.shape


@pytest.mark.parametrize("T", [1, 127, 128, 129, 5000, 70000])
def test_orders_list_every_block(dev, T):
    from zorse_amd import functional as F
    g = torch.Generator().manual_seed(T)
    cuts = sorted(torch.randint(0, T + 1, (9,), generator=g).tolist())
    seqs = F.PackedSequences(torch.tensor([0, *cuts], device=dev), T)
    plan, at = seqs.plan.cpu(), 16 + 2 * T
    for rows in (128, 128):
        n = -(-T // rows)
        assert sorted(plan[at:at + n].tolist()) == list(range(n))
        at += n
    assert at == plan.numel()


def test_gradients_against_differences(dev):
    offsets = [0, 40, 41, 130]
    q, k, v, do = _inputs(130, 2, 1, 64, F4, 4)
    got = _run(dev, q, k, v, do, offsets, True, 30)
    from zorse_amd import functional as F
    seqs = F.PackedSequences(offsets, device=dev)

    def loss(q, k, v):
        o = F.packed_attention(q.to(dev), k.to(dev), v.to(dev), seqs, window=30)
        return float((o.double() * do.to(dev).double()).sum())

    g = torch.Generator().manual_seed(9)
    for i, grad in enumerate(got[1:]):
        way = torch.randn((q, k, v)[i].shape, generator=g)
        way /= way.norm()
        step = 2.0 ** -5
        at = [[t + (s * step * way if i == j else 0) for j, t in enumerate((q, k, v))] for s in (1, -1)]
        slope = (loss(*at[0]) - loss(*at[1])) / (2 * step)
        want = float((grad.cpu().double() * way.double()).sum())
        # the central difference is off by step^2 / 6 third derivatives (of order
        # the gradient's size) and by the roundings of o over 2 step
        size = float(grad.double().norm())
        assert abs(slope - want) <= step ** 2 * size + 2.0 ** -20 * float(do.norm()) * 20 / step


def test_captured_and_updated(dev):
    """A captured pass replays with other inputs and other sequences."""
    from zorse_amd import functional as F
    T, H, Hk, d = 700, 4, 2, 128
    q, k, v, do = (t.to(dev) for t in _inputs(T, H, Hk, d, BF, 0))
    offs = torch.tensor([0, 300, 650], device=dev)
    seqs = F.PackedSequences(offs, T)

    def step():
        seqs.update(offs)
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = F.packed_attention(*leaves, seqs)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, cut in ((1, (0, 300, 650)), (2, (0, 1, 700)), (3, (0, 699, 699))):
        for t, x in zip((q, k, v, do), _inputs(T, H, Hk, d, BF, seed)):
            t.copy_(x)
        offs.copy_(torch.tensor(cut))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = _run(dev, q.cpu(), k.cpu(), v.cpu(), do.cpu(), list(cut), True, 0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_of_gradients(dev):
    from zorse_amd import functional as F
    q, k, v, do = (t.to(dev) for t in _inputs(20, 1, 1, 64, BF, 0))
    seqs = F.PackedSequences([0, 20], device=dev)
    q.requires_grad_()
    o = F.packed_attention(q, k, v, seqs)
    g = torch.autograd.grad(o, q, do, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
    o = F.packed_attention(q, k, v, seqs)
    seqs.update([0, 10, 20])  # the plan of a pass that is not over
    with pytest.raises(RuntimeError, match="modified"):
        o.backward(do)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            F.packed_attention(fwAD.make_dual(q.detach(), do), k, v, seqs)

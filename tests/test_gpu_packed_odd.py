"""Infinities and NaN in packed attention, element by element and in time: they stay
with the rows and columns that the formulas give them to, and a pass that is full of
them is not much slower than another.  The finite elements' bounds are those of
test_gpu_packed_attention."""
import math

import pytest
import torch

from tests.test_gpu_packed_attention import _inputs, _near, _reference, _run

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32
OFFSETS = [0, 70, 150, 200]


def _column_sums(x, rows_of, n):
    """For each of n rows the sum of the odd elements of x's rows rows_of(i) (any
    positive weights), 0 where there are none."""
    odd = torch.where(torch.isfinite(x), torch.zeros_like(x), x).float()
    return torch.stack([odd[rows_of(i)].sum(0) for i in range(n)])


def _agree(got, want, odd, what):
    """got is odd where `odd` is, in the same way, and within want's bound elsewhere."""
    ref, bound = want
    got, fine = got.cpu().double(), odd == 0
    assert torch.equal(torch.isnan(got), torch.isnan(odd)), what
    assert torch.equal(torch.where(torch.isinf(got), got, 0.0), torch.where(torch.isinf(odd), odd.double(), 0.0)), what
    assert bool(((got - ref).abs() <= bound)[fine].all()), what


@pytest.mark.parametrize("dt,H,d", [(BF, 4, 128), (FP, 4, 64), (BF, 4, 100), (FP, 34, 128), (F4, 4, 64)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_columns_of_rows_that_see_an_odd_element(dev, dt, H, d, value):
    """v (and, for dv, dO) holds single odd elements that are seen, beside whole odd
    rows that are not, in the same tiles."""
    T, Hk = 210, H // 2
    q, k, v, do = _inputs(T, H, Hk, d, dt, 21)
    for t in (v, do):
        t[10, :, 3] = math.inf
        t[30, :, 3] = -math.inf
        t[15, :, 7] = math.nan
        t[160, :, 5] = -math.inf
        t[190, :, d - 1] = math.inf
    clean = [torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (q, k, v, do)]
    want, _ = _reference(*clean, OFFSETS, True, 0, 1 / math.sqrt(d), dt)
    for t in (q, k, v, do):
        t[70:150] = value
        t[200:] = value
    got = _run(dev, q, k, v, do, OFFSETS, True, 0)
    start = lambda i: max(a for a in OFFSETS if a <= i)  # noqa: E731
    end = lambda i: min(a for a in OFFSETS if a > i)  # noqa: E731
    rep = H // Hk
    odd_o = _column_sums(v, lambda i: slice(start(i), i + 1), 200).repeat_interleave(rep, 1)
    # rows that see an odd v have no finite delta, and dv takes only their P and dO
    odd_dv = _column_sums(do, lambda j: slice(j, end(j)), 200).reshape(200, Hk, rep, d).sum(2)
    for rows in (slice(0, 70), slice(150, 200)):
        _agree(got[0][rows], [t[rows] for t in want[0]], odd_o[rows], "o")
        _agree(got[3][rows], [t[rows] for t in want[3]], odd_dv[rows], "dv")


@pytest.mark.parametrize("d,H", [(128, 4), (64, 34), (100, 4)])
def test_large_finite_values_of_others(dev, d, H):
    """Products with a neighbour's keys and gradients leave fp32's range."""
    T = 230
    q, k, v, do = _inputs(T, H, H // 2, d, BF, 22)
    want, _ = _reference(q, k, v, do, OFFSETS, True, 0, 1 / math.sqrt(d), BF)
    g = torch.Generator().manual_seed(1)
    for t in (q, k, v, do):
        t[70:150] = 3e38 * torch.sign(torch.randn(80, *t.shape[1:], generator=g)).to(BF)
        t[200:] = 3e38
    got = _run(dev, q, k, v, do, OFFSETS, True, 0)
    _near(got, want, "neighbours", torch.tensor([*range(70), *range(150, 200)]))


@pytest.mark.parametrize("dt,H,d", [(BF, 4, 128), (FP, 34, 64), (FP, 4, 72), (BF, 34, 100), (F4, 4, 64)])
@pytest.mark.parametrize("causal,window", [(True, 50), (True, 200), (False, 0)])
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_odd_rows_outside_a_window_and_of_whole_sequences(dev, dt, H, d, causal, window, value):
    """Odd tokens at both ends of a long sequence, those of a neighbour among its
    blocks, and single ones: rows that see none of them are as without them."""
    T, offsets = 420, [0, 301, 310, 400]
    q, k, v, do = _inputs(T, H, H // 2, d, dt, 24)
    want, _ = _reference(q, k, v, do, offsets, causal, window, 1 / math.sqrt(d), dt)
    odd = [*range(3), 299, 300, *range(301, 310), *range(400, T)]
    if not causal:  # a whole sequence sees its own
        odd = [*range(301, 310), *range(400, T)]
    for t in (q, k, v, do):
        t[odd] = value
    got = _run(dev, q, k, v, do, offsets, causal, window)
    sees = [i for i in range(400) if not any(
        (a <= j < b and a <= i < b) and (not causal or (j <= i and (not window or i - j < window)))
        for j in odd for a, b in zip(offsets, offsets[1:]))]
    seen = [j for j in range(400) if not any(
        (a <= j < b and a <= i < b) and (not causal or (j <= i and (not window or i - j < window)))
        for i in odd for a, b in zip(offsets, offsets[1:]))]
    rows = torch.tensor(sees)
    _near(got[:2], want[:2], "rows", rows)
    # a key's gradients take the rows that see it: of those that see an odd token too, its
    # own dv has their P, which is not a number, so keys beside no odd row or key
    clean = [j for j in seen if all(i in set(sees) for i in range(400) if any(
        a <= j < b and a <= i < b for a, b in zip(offsets, offsets[1:])) and
        (not causal or (j <= i and (not window or i - j < window))))]
    assert len(sees) > 80 and len(clean) > 40
    for n in (2, 3):
        _near(got[n:n + 1], want[n:n + 1], "keys", torch.tensor(clean))
    for x in got:
        assert not bool(x[400:].any())


def _time(fn):
    fn()
    best = math.inf
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fn()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("dt,d", [(BF, 128), (FP, 64), (BF, 100)])
@pytest.mark.parametrize("offsets", [[0, 2048], [0, 1000, 1016, 1030, 2048]])
def test_a_pass_of_nan_takes_little_longer(dev, dt, d, offsets):
    """One odd element, one odd row, rows of a short neighbour, or all of them: each
    within forty passes, where rows taken one token at a time are thousands."""
    from zorse_amd import functional as F, kernels as K
    T, H, Hk = 2048, 16, 8
    q, k, v, do = (t.to(dev) for t in _inputs(T, H, Hk, d, dt, 23))
    seqs = F.PackedSequences(offsets, device=dev)

    def passes(q, k, v, do):
        def fn():
            o, lse = K.attn_packed_fwd(q, k, v, seqs.plan)
            return K.attn_packed_bwd(q, k, v, o, do, lse, seqs.plan)
        return fn

    plain = _time(passes(q, k, v, do))
    nan = math.nan
    for what, rows, value in (("one row", slice(T - 1, T), nan), ("first row", slice(0, 1), nan),
                              ("some", slice(1000, 1030), math.inf), ("all", slice(0, T), nan),
                              ("all", slice(0, T), math.inf)):
        for which in range(4):
            ts = [q, k, v, do]
            ts[which] = ts[which].clone()
            ts[which][rows] = value
            t = _time(passes(*ts))
            assert t <= 40 * plain, f"{what} of {'q k v dO'.split()[which]} {value}: {t / plain:.0f} passes"
    one = do.clone()
    one[T - 1, 0, 0] = nan
    assert _time(passes(q, k, v, one)) <= 40 * plain

"""Packed attention's fp16 gradients where dO is far from 1, against the formulas in
64 bits.

P and dS are rounded to fp16 as operands.  P is at most 1 and is scaled by 2^15, so it
is off by half a step h = 2^-11 of itself or by 2^-25 / 2^15; dS is scaled by a power
of two of its row (of dQ, or of dK), by which the row's largest dS so far is at least
2^7: it is off by h of itself or by 2^-25 / 2^7 of that largest.  A rounding is spread
evenly over its step: its variance is a third of its square.  delta carries the
roundings of O, and of P in the forward, which is at least one relative to the row's
maximum.  The roundings of different elements are independent, so that the norm of
the error is the root of the variances' sum, to a few per cent for a hundred thousand
elements; fp32 sums, exponentials and what an element of less than average size has
less are covered by the factor 1.5."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP = torch.float16
H2 = 2.0 ** -22 / 3  # of a rounding, relative to the square


def _with_variances(q, k, v, do, offsets, causal, scale):
    """[(value, variance of its error)] of dq, dk, dv."""
    T, H, d = q.shape
    Hk = k.shape[1]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    out = [torch.zeros_like(t) for t in (q, k, k)]
    var = [torch.zeros_like(t) for t in (q, k, k)]
    for lo, hi in zip(offsets, offsets[1:]):
        gap = torch.arange(hi - lo)[:, None] - torch.arange(hi - lo)[None]
        hidden = gap < 0 if causal else torch.zeros_like(gap, dtype=torch.bool)
        seen = (~hidden).double()
        for x in range(H):
            g = x * Hk // H
            a, b, c, up = q[lo:hi, x], k[lo:hi, g], v[lo:hi, g], do[lo:hi, x]
            p = torch.softmax((a @ b.T * scale).masked_fill(hidden, -math.inf), 1)
            y = p @ c
            v_y = H2 * (y ** 2 + p ** 2 @ c ** 2) + (2.0 ** -24) ** 2 / 3 * (seen @ c ** 2)
            v_delta = (up ** 2 * v_y).sum(1, keepdim=True)
            ds = p * (up @ c.T - (up * y).sum(1, keepdim=True))
            least = (2.0 ** -31) ** 2 * seen
            v_ds = H2 * ds ** 2
            out[0][lo:hi, x] = ds @ b * scale
            var[0][lo:hi, x] = ((v_ds + least * ds.abs().amax(1, keepdim=True) ** 2) @ b ** 2
                                + v_delta * (p @ b) ** 2) * scale ** 2
            out[1][lo:hi, g] += ds.T @ a * scale
            var[1][lo:hi, g] += (v_ds + least * ds.abs().amax(0, keepdim=True) ** 2
                                 + v_delta * p ** 2).T @ a ** 2 * scale ** 2
            out[2][lo:hi, g] += p.T @ up
            var[2][lo:hi, g] += (H2 * p ** 2 + (2.0 ** -40) ** 2 / 3 * seen).T @ up ** 2
    return [(t, s + H2 * t ** 2 + (2.0 ** -25) ** 2 / 3) for t, s in zip(out, var)]


def _grads(dev, q, k, v, do, offsets, causal):
    from zorse_amd import functional as F
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    seqs = F.PackedSequences(offsets, q.shape[0], device=dev)
    o = F.packed_attention(*leaves, seqs, causal=causal)
    return [t.cpu().double() for t in torch.autograd.grad(o, leaves, do.to(dev))]


CASES = [
    # lengths, heads, key heads, d, causal, sizes of q, k, v, dO
    ((2048,), 2, 1, 128, True, 1 / 16, 16, 1, 1e-3),   # dq's own size stays in fp16's range
    ((2048,), 2, 1, 128, True, 16, 1 / 16, 1, 1e-3),   # dk's
    ((1500, 300), 2, 2, 64, False, 1 / 32, 32, 1, 1e-4),
    ((1500, 300), 32, 16, 64, True, 32, 1 / 32, 1, 1e-4),
    ((900, 100), 2, 2, 100, True, 1 / 16, 16, 1, 1e-3),
    ((1000,), 2, 1, 128, True, 1, 1, 1, 1),
    # dS up to 5e5, and the gradients within fp16's range
    ((300, 40), 2, 1, 128, True, 0.01, 0.01, 200, 300),
    ((300, 40), 34, 34, 64, False, 0.01, 0.01, 200, 600),
]


@pytest.mark.parametrize("lengths,H,Hk,d,causal,sq,sk,sv,so", CASES)
def test_norms_of_errors(dev, lengths, H, Hk, d, causal, sq, sk, sv, so):
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    T = offsets[-1]
    g = torch.Generator().manual_seed(T + d + H)
    q, k, v, do = ((torch.randn(T, h, d, generator=g) * s).to(FP)
                   for h, s in ((H, sq), (Hk, sk), (Hk, sv), (H, so)))
    want = _with_variances(q, k, v, do, offsets, causal, 1 / math.sqrt(d))
    got = _grads(dev, q, k, v, do, offsets, causal)
    for name, x, (ref, var) in zip(("dq", "dk", "dv"), got, want):
        off, allowed = float((x - ref).norm()), 1.5 * math.sqrt(float(var.sum()))
        assert off <= allowed, f"{name}: {off:.3e} off, {allowed:.3e} allowed, of {float(ref.norm()):.3e}"

"""Token embedding and its gradient against plain sums in 64 bits.

A gradient row is a sum of n terms in fp32 in some order, scaled and rounded
once: it is off by at most (n + 2) 2^-24 of the sum of their absolute values,
and by half a step of its type (and of the type's smallest number)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32
TINY = {BF: 2.0 ** -134, FP: 2.0 ** -25, F4: 2.0 ** -150}


def _bound(ref, terms, dt):
    """Half a step of a value next to ref, plus what comes before rounding."""
    half = torch.finfo(dt).eps / 2
    return terms * (1 + half) + half * ref.abs() + TINY[dt]


def _ids(kind, shape, V, g):
    if kind == "uniform":
        return torch.randint(0, V, shape, generator=g)
    if kind == "one":
        return torch.full(shape, V - 1)
    if kind == "zipf":
        u = torch.rand(shape, generator=g, dtype=torch.float64)
        return ((V + 1.0) ** u - 1).long().clamp_(0, V - 1)
    if kind == "runs":  # ids that fill whole blocks of 64 grouped tokens, and one more
        n = 1
        for s in shape:
            n *= s
        return (torch.arange(n) // 64 % V).view(shape)
    bad = torch.randint(-3, V + 3, shape, generator=g)  # some outside the table
    return bad


def _reference(ids, dy, V, scale, pad, old=None):
    """(gradient, what its sums may be off by) in 64 bits."""
    ids, dy = ids.reshape(-1), dy.double().reshape(ids.numel(), -1)
    ok = (ids >= 0) & (ids < V)
    if pad is not None:
        ok &= ids != pad
    ref = torch.zeros(V, dy.shape[1], dtype=torch.float64)
    mag, n = ref.clone(), torch.zeros(V, 1, dtype=torch.float64)
    ref.index_add_(0, ids[ok], dy[ok])
    mag.index_add_(0, ids[ok], dy[ok].abs())
    n.index_add_(0, ids[ok], torch.ones(int(ok.sum()), 1, dtype=torch.float64))
    ref, terms = ref * scale, (n + 2) * 2.0 ** -24 * mag * abs(scale)
    if old is not None:
        ref, terms = ref + old.double(), terms + 2.0 ** -24 * old.double().abs()
    return ref, terms, n[:, 0] > 0


CASES = [
    # tokens, hidden, vocab, ids, table, activations, scale, pad
    ((1,), 1, 1, "one", F4, F4, 1.0, None),
    ((1, 1), 8, 300, "uniform", BF, BF, 1.0, None),
    ((64,), 512, 7, "one", BF, BF, 1.0, None),
    ((65,), 520, 3, "one", FP, FP, 0.5, None),
    ((5, 77), 100, 257, "uniform", F4, F4, 10.0, None),
    ((128,), 1030, 61, "zipf", F4, FP, 3.0, None),  # the most that one launch takes
    ((100,), 24, 5, "outside", FP, FP, 1.0, 4),
    ((129,), 7, 1000, "zipf", BF, F4, 1.0, 0),
    ((3, 43), 1033, 50, "zipf", F4, BF, -2.0, 49),
    ((4097,), 264, 128, "runs", BF, BF, 1.0, None),
    ((2, 3000), 2056, 33000, "zipf", BF, BF, 1.0, None),
    ((700,), 130, 140000, "uniform", FP, F4, 1.0, 5),
    ((20011,), 24, 4, "uniform", F4, F4, 1.0, None),
    ((9, 31), 64, 40, "outside", BF, FP, 1.0, 1),
]


@pytest.mark.parametrize("shape,h,V,kind,wdt,adt,scale,pad", CASES)
@pytest.mark.parametrize("idt", [torch.int64, torch.int32])
def test_lookup_and_gradient(dev, shape, h, V, kind, wdt, adt, scale, pad, idt):
    from zorse_amd import functional
    g = torch.Generator().manual_seed(h + V)
    ids = _ids(kind, shape, V, g)
    w = torch.randn(V, h, generator=g).to(wdt)
    dy = torch.randn(*shape, h, generator=g).to(adt)
    wd = w.to(dev).requires_grad_()
    y = functional.embedding(ids.to(dev, idt), wd, scale=scale, padding_idx=pad, dtype=adt)
    y.backward(dy.to(dev))
    inside = (ids >= 0) & (ids < V)
    ref = w.double()[ids.clamp(0, V - 1)] * scale
    got = y.detach().cpu()
    assert got.dtype == adt and got.shape == ref.shape
    assert bool(got[~inside].isnan().all())
    off = (got.double() - ref).abs()[inside]
    assert bool((off <= _bound(ref[inside], 2.0 ** -24 * ref[inside].abs(), adt)).all())
    if scale == 1.0 and adt == wdt:
        assert torch.equal(got[inside], w[ids[inside]])
    ref, terms, _ = _reference(ids, dy, V, scale, pad)
    assert wd.grad.dtype == wdt
    assert bool(((wd.grad.cpu().double() - ref).abs() <= _bound(ref, terms, wdt)).all())


@pytest.mark.parametrize("shape,h,V,kind,wdt,adt,scale,pad", CASES)
def test_accumulated_gradient(dev, shape, h, V, kind, wdt, adt, scale, pad):
    """Added to what is there; rows that no token names keep their bits."""
    from zorse_amd import kernels
    g = torch.Generator().manual_seed(h * V)
    ids = _ids(kind, shape, V, g)
    dy = torch.randn(*shape, h, generator=g).to(adt)
    old = torch.randn(V, h, generator=g).to(wdt)
    dw = old.to(dev)
    out = kernels.embedding_bwd(ids.to(dev), dy.to(dev), V, scale=scale, padding_idx=pad, dw=dw,
                                accumulate=True)
    assert out is dw
    ref, terms, named = _reference(ids, dy, V, scale, pad, old)
    got = dw.cpu()
    assert torch.equal(got[~named], old[~named])
    assert bool(((got.double() - ref).abs() <= _bound(ref, terms, wdt)).all())


def test_equal_calls_give_equal_bits(dev):
    """Also with other calls in between, and on another stream."""
    from zorse_amd import kernels
    g = torch.Generator().manual_seed(3)
    ids = _ids("zipf", (9001,), 5000, g).to(dev)
    dy = torch.randn(9001, 96, generator=g).to(dev)
    first = kernels.embedding_bwd(ids, dy, 5000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = kernels.embedding_bwd(ids, dy, 5000)
    kernels.embedding_bwd(ids.flip(0), dy, 5000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)


def test_strided_inputs_and_empty_batches(dev):
    from zorse_amd import functional, kernels
    g = torch.Generator().manual_seed(4)
    w = torch.randn(30, 10, generator=g).to(dev).requires_grad_()
    ids = torch.randint(0, 30, (6, 8), generator=g).to(dev)
    y = functional.embedding(ids.t(), w)
    assert torch.equal(y, w[ids.t()])
    y.sum().backward()  # a gradient with strides of zero
    want = torch.bincount(ids.flatten(), minlength=30).float()[:, None].expand(30, 10)
    assert torch.equal(w.grad, want)
    none = functional.embedding(ids[:0], w)
    assert none.shape == (0, 8, 10)
    grad, = torch.autograd.grad(none, w, torch.empty_like(none))
    assert not bool(grad.any())
    keep = torch.ones(30, 10, device=dev)
    kernels.embedding_bwd(ids[:0], none.detach(), 30, dw=keep, accumulate=True)
    assert bool((keep == 1).all())
    with pytest.raises(ValueError):
        kernels.embedding_bwd(ids, torch.zeros(6, 9, 10, device=dev), 30)
    with pytest.raises(ValueError):
        kernels.embedding_bwd(ids, torch.zeros(6, 8, 10, device=dev), 30, accumulate=True)
    with pytest.raises(ValueError):
        kernels.embedding_fwd(ids.float(), w.detach())


def test_non_finite_rows_stay_where_they_are(dev):
    from zorse_amd import functional
    w = torch.zeros(4, 16, device=dev)
    w[1], w[2] = float("inf"), float("nan")
    w.requires_grad_()
    ids = torch.tensor([0, 1, 2, 3, 0], device=dev)
    y = functional.embedding(ids, w)
    assert bool((y[[0, 3, 4]] == 0).all()) and bool((y[1] == float("inf")).all())
    dy = torch.ones_like(y)
    dy[1] = float("nan")
    y.backward(dy)
    assert bool(w.grad[1].isnan().all())
    assert torch.equal(w.grad[[0, 2, 3]], torch.tensor([2.0, 1.0, 1.0], device=dev)[:, None]
                       .expand(3, 16))


def test_captured_pass_replays_with_new_tokens(dev):
    """Forward and gradient in a graph, replayed between eager calls."""
    from zorse_amd import kernels
    g = torch.Generator().manual_seed(5)
    V, h, n = 700, 72, 1500
    w = torch.randn(V, h, generator=g).to(dev)
    dy = torch.randn(n, h, generator=g).to(dev)
    ids = torch.zeros(n, dtype=torch.int64, device=dev)
    kernels.embedding_bwd(ids, dy, V)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kernels.embedding_fwd(ids, w)
        dw = kernels.embedding_bwd(ids, dy, V)
    for seed in range(3):
        ids.copy_(_ids("zipf", (n,), V, torch.Generator().manual_seed(seed)))
        want = kernels.embedding_bwd(ids, dy, V)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w[ids]) and torch.equal(dw, want)


def test_model_embedding_module(dev):
    """The models' table: lookup bits of nn.Embedding, its gradient."""
    from zorse_amd.llama_simple import TokenEmbedding
    torch.manual_seed(1)
    m = TokenEmbedding(64, 40, padding_idx=3).to(dev)
    ids = torch.randint(0, 64, (3, 17), device=dev)
    ids[0, :5] = 3
    y = m(ids)
    assert torch.equal(y, torch.nn.functional.embedding(ids, m.weight, 3))
    dy = torch.randn_like(y)
    y.backward(dy)
    ref, terms, _ = _reference(ids.cpu(), dy.cpu(), 64, 1.0, 3)
    assert bool(((m.weight.grad.cpu().double() - ref).abs() <= _bound(ref, terms, F4)).all())


def test_gradient_is_differentiable(dev):
    """A second differentiation (create_graph): the table's gradient is linear
    in dy, its own gradient the lookup, and zero for tokens without one."""
    from zorse_amd import functional
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-2, 14, (5, 40), generator=g).to(dev)
    w = torch.randn(12, 24, generator=g).to(dev).requires_grad_()
    dy = torch.randn(5, 40, 24, generator=g).to(dev).requires_grad_()
    a = torch.randn(12, 24, generator=g).to(dev).requires_grad_()
    for scale, pad in ((1.0, None), (0.5, 4)):
        y = functional.embedding(ids, w, scale=scale, padding_idx=pad)
        plain, = torch.autograd.grad(y, w, dy.detach(), retain_graph=True)
        dw, = torch.autograd.grad(y, w, dy, create_graph=True)
        assert torch.equal(dw, plain)
        ddy, = torch.autograd.grad(dw, dy, a, create_graph=True)
        ok = (ids >= 0) & (ids < 12)
        if pad is not None:
            ok &= ids != pad
        want = torch.where(ok.unsqueeze(-1), scale * a[ids.clamp(0, 11)], 0.0)
        assert torch.equal(ddy, want)
        da, = torch.autograd.grad(ddy, a, dy.detach())  # linear in a: dw again
        assert torch.equal(da, plain)

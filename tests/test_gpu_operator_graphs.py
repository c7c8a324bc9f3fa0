"""The operators' training passes captured into a graph, through their autograd
nodes: replays with other inputs against eager passes.

As torch's own: the pass is warmed up on the capturing stream, and no eager
graph of the captured leaves is alive."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _captured(step, fill, leaves):
    """(graph, its outputs) of step(leaves), after a pass on a side stream."""
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
    return graph, out


def _check(step, fill, leaves):
    graph, out = _captured(step, fill, leaves)
    for seed in (1, 2, 3):
        fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        # other leaves with the same values: an eager graph of their own
        twins = [t.detach().clone().requires_grad_() for t in leaves]
        want = step(twins)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("tokens", [100, 3000])
def test_embedding_pass(dev, tokens):
    from zorse_amd import functional
    V, h = 900, 136
    w = torch.randn(V, h, device=dev, dtype=torch.bfloat16).requires_grad_()
    ids = torch.zeros(2, tokens // 2, dtype=torch.int64, device=dev)
    dy = torch.zeros(2, tokens // 2, h, device=dev, dtype=torch.bfloat16)

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        ids.copy_(torch.randint(0, V, ids.shape, generator=g) // (1 + seed % 2 * 20))
        dy.copy_(torch.randn(dy.shape, generator=g))

    def step(leaves):
        y = functional.embedding(ids, leaves[0], scale=2.0, padding_idx=3)
        return y.detach(), *torch.autograd.grad(y, leaves, dy)

    _check(step, fill, [w])


def test_head_norm_pass(dev):
    from zorse_amd import functional
    q, k, dq, dk = (torch.zeros(2, 150, h, 64, device=dev, dtype=torch.bfloat16)
                    for h in (6, 2, 6, 2))
    leaves = [q.requires_grad_(), k.requires_grad_(),
              *(torch.ones(64, device=dev).requires_grad_() for _ in range(2))]
    ang = torch.arange(150)[:, None] * 1e4 ** (-torch.arange(0, 64, 2) / 64)
    cos, sin = ang.cos().to(dev), ang.sin().to(dev)

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            for t in (*leaves, dq, dk):
                t.copy_(torch.randn(t.shape, generator=g))

    def step(x):
        y = functional.qk_norm_rope(x[0], x[1], x[2], x[3], cos, sin)
        return *(t.detach() for t in y), *torch.autograd.grad(y, x, (dq, dk))

    _check(step, fill, leaves)


def test_list_step(dev):
    """The step over lists with 32-bit moments; a replay repeats its count."""
    from zorse_amd import kernels
    sizes = [700, 33, 5000] * 25  # two launches
    state = [[torch.randn(n, device=dev) * 1e-2 for n in sizes] for _ in range(3)]
    state.append([torch.rand(n, device=dev) * 1e-4 for n in sizes])
    low = [torch.zeros(n, device=dev, dtype=torch.bfloat16) for n in sizes]
    twin = [[t.clone() for t in ts] for ts in (*state, low)]

    def step(p, g, m, v, copies):
        kernels.adamw_multi(p, g, m, v, [7] * len(p), lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8,
                            weight_decay=0.1, lowp_outs=copies)

    step(*state, low)
    step(*twin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*state, low)
    for _ in range(3):
        for a, b in zip(state[1], twin[1]):
            a.mul_(-0.7)
            b.mul_(-0.7)
        graph.replay()
        step(*twin)
        torch.cuda.synchronize()
        for ts, us in zip((*state, low), twin):
            assert all(torch.equal(a, b) for a, b in zip(ts, us))

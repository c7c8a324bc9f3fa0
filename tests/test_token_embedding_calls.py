"""The models' token table in calls that no kernel can serve: nn.Embedding's
own operations, as before the kernels."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from zorse_amd.llama_simple import TokenEmbedding


def test_fake_tensors():
    """Shapes of a model on a GPU, worked out without one (CPU)."""
    with FakeTensorMode():
        m = TokenEmbedding(11, 6, padding_idx=2, device="cuda", dtype=torch.bfloat16)
        y = m(torch.zeros(3, 4, dtype=torch.long, device="cuda"))
        assert y.shape == (3, 4, 6) and y.dtype == torch.bfloat16 and y.device.type == "cuda"


class _Wrapped(torch.Tensor):
    """A subclass without memory, as distributed tensors are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device="cuda")

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        out = func(*(a.inner if isinstance(a, _Wrapped) else a for a in args), **(kwargs or {}))
        return _Wrapped(out) if func is torch.ops.aten.detach.default else out


def test_tensors_without_memory():
    """The operation reaches the subclass (CPU: the inner tensors are here)."""
    table = torch.arange(12.0).view(6, 2)
    m = TokenEmbedding(6, 2)
    m.weight = torch.nn.Parameter(_Wrapped(table), requires_grad=False)
    assert m.weight.is_cuda
    ids = torch.tensor([5, 0])
    assert torch.equal(m(_Wrapped(ids)), table[ids])


@pytest.fixture
def both(dev):
    torch.manual_seed(2)
    ours = TokenEmbedding(13, 8, padding_idx=1, device=dev)
    theirs = torch.nn.Embedding(13, 8, padding_idx=1, device=dev)
    theirs.load_state_dict(ours.state_dict())
    return ours, theirs, torch.randint(0, 13, (4, 9), device=dev)


@pytest.mark.gpu
def test_function_transforms(both):
    *modules, ids = both
    t = torch.randn(13, 8, device=ids.device)
    got = []
    for m in modules:
        def f(w, i=ids):
            return torch.func.functional_call(m, {"weight": w}, (i,))
        w = m.weight.detach()
        tables = torch.stack((w, t))
        got.append((torch.func.vmap(f)(tables, torch.stack((ids, ids.flip(0)))),
                    torch.func.vmap(lambda i: f(w, i))(ids), *torch.func.jvp(f, (w,), (t,)),
                    torch.func.grad(lambda x: f(x).square().sum())(w)))
    for a, b in zip(*(g[:4] for g in got)):
        assert torch.equal(a, b)
    # sums of up to 36 equal terms 2 w: 36 roundings of 2^-24 of the sum
    assert float((got[0][4] - got[1][4]).abs().max()) <= 72 * 2.0 ** -24 * float(got[1][4].abs().max())


@pytest.mark.gpu
def test_recorded_calls(both):
    """A trace holds the lookup, not one call's rows."""
    ours, theirs, ids = both
    traced = torch.jit.trace(ours, (ids,))
    other = ids.flip(1).contiguous()
    assert torch.equal(traced(other), theirs(other))


@pytest.mark.gpu
def test_compiled_call_has_one_graph(both):
    """As nn.Embedding's: nothing that would cut the recorded graph."""
    ours, theirs, ids = both
    torch._dynamo.reset()
    compiled = torch.compile(ours, backend="eager", fullgraph=True)
    for i in (ids, ids.flip(0)):
        y = compiled(i)
        assert torch.equal(y, theirs(i))
    grad, = torch.autograd.grad(y.sum(), ours.weight)
    want, = torch.autograd.grad(theirs(ids).sum(), theirs.weight)
    assert torch.equal(grad, want)  # sums of ones

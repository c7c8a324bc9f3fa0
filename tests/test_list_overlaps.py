"""Lists of tensors whose memory overlaps: refused where one that is written
meets another, before any launch (CPU: tensors that have addresses alone)."""
import numpy as np
import pytest
import torch

from zorse_amd import kernels


class _At(torch.Tensor):
    """n elements of a type at an address of the GPU, without memory."""

    @staticmethod
    def __new__(cls, address, n, dtype):
        size = torch.empty(0, dtype=dtype).element_size()
        return torch.Tensor._make_wrapper_subclass(cls, (n,), (1,), address // size, dtype=dtype,
                                                   device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} on an address")


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    """Nothing is launched on these addresses, whatever a check lets through."""
    def launched():
        raise AssertionError("launched")
    monkeypatch.setattr(kernels, "lib", launched)


F4, BF, U8, I16 = torch.float32, torch.bfloat16, torch.uint8, torch.int16
N = 300


def _lists(n=3):
    """Columns of tensors apart from each other: p, g, m, v, low."""
    def column(c, dt):
        return [_At((c * n + i + 1) << 14, N, dt) for i in range(n)]
    return [column(c, dt) for c, dt in enumerate((F4, BF, F4, F4, BF))]


def _table(p, g, m, v, low):
    states = (("exp_avg", m, kernels._F32, kernels._SAME, kernels._WRITTEN),
              ("exp_avg_sq", v, kernels._F32, kernels._SAME, kernels._WRITTEN))
    return kernels._step_table("adamw_multi", states, p, g, [1] * len(p), low)


def test_lists_apart_are_taken():
    cols = _lists()
    index, table = _table(*cols)
    assert index == 0 and len(table) == 3 * 9 * 8
    rows = np.frombuffer(table, dtype=np.int64).reshape(3, 9)
    for c in range(5):
        assert rows[:, c].tolist() == [(c * 3 + i + 1) << 14 for i in range(3)]
    for order in ([4, 1, 0, 3, 2], [2, 3, 1, 4, 0]):  # columns anywhere in memory
        moved = [[_At((order[c] * 3 + 2 - i + 1) << 14, N, t.dtype) for i, t in enumerate(ts)]
                 for c, ts in enumerate(cols)]
        _table(*moved)
    inter = [[_At((i * 5 + c + 1) << 14, N, t.dtype) for i, t in enumerate(ts)]
             for c, ts in enumerate(cols)]
    _table(*inter)
    # neighbours, gradients that are shared, a copy that is the parameter or the gradient
    p, g, m, v, low = cols
    _table(p, g, [_At((1 << 20) + i * 4 * N, N, F4) for i in range(3)], v, low)
    _table(p, [g[0]] * 3, m, v, low)
    _table(p, g, m, v, [None, p[1], g[2]])
    _table(p[:1], g[:1], m[:1], v[:1], [None])


@pytest.mark.parametrize("column", [0, 2, 3, 4])
@pytest.mark.parametrize("apart", [0, 4, 4 * N - 4])
def test_written_tensors_that_meet(column, apart):
    """The same one twice, or one that begins inside another."""
    cols = _lists()
    dt = cols[column][0].dtype
    at = (column * 3 + 1) << 14
    if dt == BF:
        apart //= 2
    cols[column][2] = _At(at + apart, N, dt)
    with pytest.raises(ValueError, match="twice, or overlaps"):
        kernels.adamw_multi(*cols[:4], [1] * 3, lowp_outs=cols[4], lr=1e-3, beta1=0.9, beta2=0.99,
                            eps=1e-8, weight_decay=0.0)


@pytest.mark.parametrize("a,b", [(a, b) for a in range(5) for b in (0, 2, 3, 4) if a != b])
def test_columns_that_meet(a, b):
    """A tensor that is written in the place of another parameter's."""
    cols = _lists()
    cols[a][0] = _At((b * 3 + 3) << 14, N, cols[a][0].dtype)
    with pytest.raises(ValueError, match="twice, or overlaps"):
        _table(*cols)


def test_one_tensors_columns_that_meet_shifted():
    p, g, m, v, low = _lists(1)
    for col, dt in ((m, F4), (g, BF), (g, F4), (low, BF)):
        old = col[0]
        col[0] = _At((1 << 14) + 8, N, dt)
        with pytest.raises(ValueError, match="twice, or overlaps"):
            _table(p, g, m, v, low)
        col[0] = old
    low[0] = _At(1 << 14, N, BF)  # a 16-bit copy over the fp32 parameter
    with pytest.raises(ValueError, match="twice, or overlaps"):
        _table(p, g, m, v, low)


def test_eight_bit_lists_that_meet():
    def column(c, dt, n=N):
        return [_At((c * 2 + i + 1) << 14, n, dt) for i in range(2)]
    h = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, seeds=[1, 2])
    for twice in (0, 2, 3, 4):
        cols = [column(0, F4), column(1, BF), column(2, U8), column(3, U8),
                [_At((8 + i + 1) << 14, 4, I16) for i in range(2)]]
        cols[twice][1] = cols[twice][0]
        with pytest.raises(ValueError, match="twice, or overlaps"):
            kernels.adamw8_multi(*cols, [1, 1], **h)
    codes = (column(2, U8), column(3, U8), [_At((8 + i + 1) << 14, 4, I16) for i in range(2)])
    first, second = column(5, F4), column(6, F4)
    for outs in (([first[0]] * 2, second), (first, [first[1], second[1]])):
        with pytest.raises(ValueError, match="twice, or overlaps"):
            kernels.adamw8_values(*codes, outs=outs)

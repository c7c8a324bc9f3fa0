"""The operators around the layers as a training step uses them together:
token table -> projection -> norm of query and key heads with the rotation ->
attention -> head and loss, backward, and an AdamW step of every tensor, against
the same step in 64 bits on the CPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

B, S, V, H, HK, D = 2, 65, 90, 4, 2, 64
HID = H * D


def _weights(g):
    shapes = {"table": (V, HID), "qkv": ((H + 2 * HK) * D, HID), "q_norm": (D,), "k_norm": (D,),
              "o": (HID, HID), "norm": (HID,), "head": (V, HID)}
    return {k: (1 + 0.1 * torch.randn(s, generator=g)) if k.endswith("norm")
            else torch.randn(s, generator=g) / math.sqrt(HID) for k, s in shapes.items()}


def _batch(g):
    ids = torch.randint(1, V, (B, S), generator=g)
    ids[1, 40:] = 0  # padding
    labels = torch.where(ids == 0, -100, torch.randint(0, V, (B, S), generator=g))
    return ids, labels


def _tables():
    inv = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(S, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _plain(w, ids, labels, cos, sin, scale):
    """The loss in the weights' own precision, elementary operations."""
    def norm(x, wt):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * wt

    def turn(x):
        a, b = x.chunk(2, -1)
        c, s = cos[:, None], sin[:, None]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    x = w["table"][ids] * scale
    x = torch.where((ids == 0)[..., None], x.detach(), x)  # no gradient into the padding row
    qkv = x @ w["qkv"].t()
    q, k, v = qkv.split([H * D, HK * D, HK * D], -1)
    q = turn(norm(q.unflatten(-1, (H, D)), w["q_norm"])).transpose(1, 2)
    k = turn(norm(k.unflatten(-1, (HK, D)), w["k_norm"])).transpose(1, 2)
    v = v.unflatten(-1, (HK, D)).transpose(1, 2)
    k, v = (t.repeat_interleave(H // HK, 1) for t in (k, v))
    att = (q @ k.transpose(-1, -2)) / math.sqrt(D)
    mask = torch.ones(S, S, dtype=torch.bool).tril()
    att = att.masked_fill(~mask, float("-inf")).softmax(-1) @ v
    h = x + att.transpose(1, 2).flatten(-2) @ w["o"].t()
    logits = norm(h, w["norm"]) @ w["head"].t()
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), labels.flatten())


def _ours(p, ids, labels, cos, sin, scale, dt):
    from zorse_amd import functional as F
    from zorse_amd.lm_head import lm_head_cross_entropy
    lin = torch.nn.functional.linear
    x = F.embedding(ids, p["table"], scale=scale, padding_idx=0, dtype=dt)
    qkv = lin(x, p["qkv"])
    q = qkv[..., :H * D].unflatten(-1, (H, D))
    k = qkv[..., H * D:(H + HK) * D].unflatten(-1, (HK, D))
    v = qkv[..., (H + HK) * D:].unflatten(-1, (HK, D))
    q, k = F.qk_norm_rope(q, k, p["q_norm"], p["k_norm"], cos, sin)
    o = F.flash_attention(q, k, v)
    h = x + lin(o.flatten(-2), p["o"])
    return lm_head_cross_entropy(F.rms_norm(h, p["norm"]), p["head"], labels)


@pytest.mark.parametrize("dt,bits", [(torch.float32, 32), (torch.float32, 8),
                                     (torch.bfloat16, 32), (torch.bfloat16, 8)])
def test_step_against_64_bits(dev, dt, bits):
    from zorse_amd.optim import FusedAdamW
    g = torch.Generator().manual_seed(21)
    w = {k: t.to(dt) for k, t in _weights(g).items()}
    ids, labels = _batch(g)
    cos, sin = _tables()
    scale = 4.0
    ref = {k: t.double().requires_grad_() for k, t in w.items()}
    loss_ref = _plain(ref, ids, labels, cos.double(), sin.double(), scale)
    loss_ref.backward()
    p = {k: torch.nn.Parameter(t.to(dev)) for k, t in w.items()}
    opt = FusedAdamW(list(p.values()), lr=1e-2, weight_decay=0.1, state_bits=bits)
    loss = _ours(p, ids.to(dev), labels.to(dev), cos.to(dev), sin.to(dev), scale, dt)
    loss.backward()
    # Normwise, a chain of 8 stages each of whose sums (fp32: up to 256 terms,
    # 2^-24 sqrt(256) of their norm) and roundings (half a step) adds up:
    # fp32 8 * 17 * 2^-24 = 8e-6, bf16 8 * 2^-8 = 3e-2; twice that for the
    # backward, which runs through the forward's errors as well
    tol = {torch.float32: 2e-5, torch.bfloat16: 6.3e-2}[dt]
    assert abs(loss.item() - loss_ref.item()) <= tol * loss_ref.item()
    for k, t in ref.items():
        got = p[k].grad.double().cpu()
        assert float((got - t.grad).norm()) <= tol * float(t.grad.norm()), k
    assert not bool(p["table"].grad[0].any())
    before = {k: t.detach().clone() for k, t in p.items()}
    opt.step()
    for k, t in p.items():
        # the first step is lr g / (|g| + eps) after the decay, by the tensor's own gradient
        g0, old = t.grad.double(), before[k].double()
        want = old * (1 - 1e-3) - 1e-2 * g0 / (g0.abs() + 1e-8)
        half = torch.finfo(dt).eps / 2
        # fp32 update: 16 roundings of a step of 1e-2 and 3 of the parameter
        bound = 2.0 ** -24 * (3 * old.abs() + 16e-2) + half * want.abs()
        # near eps the bias corrections' rounding moves the quotient by 2^-22 more
        assert bool(((t.double() - want).abs() <= bound + 2.0 ** -22 * 1e-2).all()), k
        m, v = opt.moments(t)
        step = 2.0 ** -4 if bits == 8 else 2.0 ** -23
        below = g0.abs().max() * 0.1 * (2.0 ** -15 if bits == 8 else 0.0)
        assert bool(((m.view_as(g0).double() - 0.1 * g0).abs()
                     <= step * (1 + 2.0 ** -10) * 0.1 * g0.abs() + below).all()), k


def test_steps_repeat_bit_for_bit(dev):
    """Three steps from the same start, with 8-bit states, twice."""
    from zorse_amd.optim import FusedAdamW
    ends = []
    for _ in range(2):
        g = torch.Generator().manual_seed(5)
        p = {k: torch.nn.Parameter(t.to(dev)) for k, t in _weights(g).items()}
        opt = FusedAdamW(list(p.values()), lr=1e-3, state_bits=8)
        cos, sin = (t.to(dev) for t in _tables())
        for _ in range(3):
            ids, labels = _batch(g)
            opt.zero_grad()
            _ours(p, ids.to(dev), labels.to(dev), cos, sin, 1.0, torch.float32).backward()
            # what the operators here give; library products may not repeat
            for k in ("qkv", "o"):
                p[k].grad = None
            opt.step()
        ends.append(p)
    for k in ends[0]:
        assert torch.equal(ends[0][k], ends[1][k]), k


def test_stage_with_eight_bit_states(dev):
    """StageRunner(state_bits=8): every layer is stepped in the backward."""
    from zorse_amd import llama_simple as L
    from zorse_amd.stage import StageRunner
    cfg = L.llama_config(hidden_size=256, num_attention_heads=2, intermediate_size=512)
    layers = [L.Block(cfg, i, init_std=0.02, param_dtype=torch.bfloat16).to(dev) for i in range(2)]
    stage = StageRunner(layers, state_bits=8)
    before = [b.block.flat_param.detach().clone() for b in layers]
    x = torch.randn(1, 96, 256, device=dev).bfloat16().requires_grad_()
    stage.step(x, torch.randn_like(x))
    torch.cuda.synchronize()
    for b, old, opt in zip(layers, before, stage.optimizers):
        flat = b.block.flat_param
        st = opt.state[flat]
        assert st["exp_avg"].dtype == torch.uint8 and st["step"] == 1
        assert not torch.equal(flat, old) and torch.equal(flat, opt.master_param(flat).bfloat16())


def test_captured_update(dev):
    """Loss, gradients and the step of lists in a graph: replays repeat the
    eager calls on the same inputs."""
    from zorse_amd import kernels
    g = torch.Generator().manual_seed(9)
    sizes = [700, 33, 5000]
    args = [[torch.randn(n, generator=g).to(dev) for n in sizes] for _ in range(2)]
    cm, cv = ([torch.zeros(n, dtype=torch.uint8, device=dev) for n in sizes] for _ in range(2))
    base = [torch.zeros(-(-n // 256), 2, dtype=torch.int16, device=dev) for n in sizes]
    hyper = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0)

    def step(p, gr, a, b, c):
        kernels.adamw8_multi(p, gr, a, b, c, [4] * 3, seeds=[1, 2, 3], **hyper)

    state = (args[0], args[1], cm, cv, base)
    twin = [[t.clone() for t in ts] for ts in state]
    step(*state)
    step(*twin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*state)
    for _ in range(3):
        for a, b in zip(state[1], twin[1]):
            a.mul_(-0.7)
            b.mul_(-0.7)
        graph.replay()
        step(*twin)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(state, twin) for a, b in zip(x, y))

"""A training step over packed sequences with the operators together: rotation
by several axes, attention within the sequences, and Muon's step, as a model of
one's own has them; and decoder layers whose stage steps with Muon.

Gradients are compared with the same model in 64 bits on the same 16-bit
weights and inputs, beside the error of the same model in elementary torch
operations in 16 bits: at most 1.5 times that and a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _plain(x, w, offsets, cos, sin, positions, axes, H, Hk, d):
    """out [T, h]: q|k|v, rotation, attention, output product."""
    dt = x.dtype
    T = x.shape[0]
    qkv = x @ w["qkv"].t()
    q = qkv[:, :H * d].view(T, H, d)
    k = qkv[:, H * d:(H + Hk) * d].view(T, Hk, d)
    v = qkv[:, (H + Hk) * d:].view(T, Hk, d)
    pair = torch.arange(d // 2)
    at = positions[list(axes)].t()
    c, s = (t.to(dt if dt == torch.float64 else torch.float32)[at, pair][:, None] for t in (cos, sin))

    def turn(t):
        a, b = t.to(c.dtype).chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1).to(dt)

    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    outs = []
    for lo, hi in zip(offsets, offsets[1:]):
        n = hi - lo
        a, b, e = (t[lo:hi].transpose(0, 1).to(c.dtype) for t in (q, k, v))
        sc = (a @ b.transpose(1, 2).contiguous()) / math.sqrt(d)
        sc = sc.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
        outs.append((torch.softmax(sc, -1).to(dt).to(c.dtype) @ e).transpose(0, 1).to(dt))
    outs.append(torch.zeros(T - offsets[-1], H, d, dtype=dt))
    return torch.cat(outs).reshape(T, H * d) @ w["o"].t()


def test_a_step_of_the_operators_together(dev):
    from zorse_amd import functional as F, kernels as K, optim
    T, h, H, Hk, d, offsets = 400, 256, 4, 2, 64, [0, 150, 151, 151, 380]
    g = torch.Generator().manual_seed(3)
    mk = lambda *s: (torch.randn(*s, generator=g)).to(BF)  # noqa: E731
    x, up = mk(T, h), mk(T, h)
    x[380:] = 0
    w = {"qkv": (mk((H + 2 * Hk) * d, h) * 0.06).to(BF), "o": (mk(h, H * d) * 0.06).to(BF)}
    axes = F.pair_axes_of((12, 10, 10))
    cos, sin = F.rope_tables(400, d, 1e4, torch.float32, torch.device("cpu"))
    seqs = F.PackedSequences(offsets, T, device=dev)
    own = seqs.positions.cpu()
    positions = torch.stack((own, own // 7, own % 7))

    def grads(dt):
        ws = {k: t.to(dt).requires_grad_() for k, t in w.items()}
        y = _plain(x.to(dt), ws, offsets, cos, sin, positions, axes, H, Hk, d)
        y.backward(up.to(dt))
        return y.detach().double(), {k: t.grad.double() for k, t in ws.items()}

    ref, gref = grads(torch.float64)
    low, glow = grads(BF)

    class Linear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a, b):
            ctx.save_for_backward(a, b)
            return K.gemm(a, b)

        @staticmethod
        def backward(ctx, dy):
            a, b = ctx.saved_tensors
            dy = dy.contiguous()
            return K.gemm(dy, b, b_kmajor=True), K.gemm(dy, a, a_kmajor=True, b_kmajor=True)

    params = {k: torch.nn.Parameter(t.to(dev)) for k, t in w.items()}
    opt = optim.Muon(params.values(), lr=0.02)
    dcos, dsin, dpos = cos.to(dev), sin.to(dev), positions.to(dev)
    xs = x.to(dev).requires_grad_()
    for step in range(2):
        qkv = Linear.apply(xs, params["qkv"])
        q = qkv[:, :H * d].unflatten(1, (H, d))
        k = qkv[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d))
        v = qkv[:, (H + Hk) * d:].unflatten(1, (Hk, d))
        q, k = F.rope_axes(q, k, dcos, dsin, dpos, axes)
        o = F.packed_attention(q, k, v, seqs)
        y = Linear.apply(o.flatten(1), params["o"])
        y.backward(up.to(dev))
        if step == 0:
            for name, got, want, other in [("out", y.detach(), ref, low)] + [
                    (k, params[k].grad, gref[k], glow[k]) for k in params]:
                off = float((got.cpu().double() - want).norm())
                bound = 1.5 * float((other - want).norm()) + 2 ** -8 * float(want.norm())
                assert off <= bound, f"{name}: {off:.3e} > {bound:.3e}"
            assert not bool(xs.grad[380:].any())
        before = [p.detach().clone() for p in params.values()]
        opt.step()
        opt.zero_grad()
        for p, b in zip(params.values(), before):
            assert bool(torch.isfinite(p).all()) and not torch.equal(p, b)


@pytest.mark.parametrize("dt", [torch.float32, BF])
def test_muon_over_a_model(dev, dt):
    """Matrices, vectors and a flat layer, against the kernels' own calls."""
    from zorse_amd import kernels as K, llama_simple, optim
    cfg = llama_simple.llama_config(hidden_size=128, num_attention_heads=2, num_key_value_heads=1,
                                    intermediate_size=256, rope_theta=1e4)
    layer = llama_simple.LlamaDecoderLayer(cfg, 0, param_dtype=dt).to(dev)
    w, b = (torch.nn.Parameter(torch.randn(s, device=dev).to(dt)) for s in ((160, 200), (200,)))
    mats = optim.flat_matrices(layer)
    opt = optim.Muon([{"params": [w, b]}, {"params": [layer.flat_param], "matrices": mats, "lr": 3e-3,
                                           "adam_lr": 1e-3}], lr=0.01, adjust="match_rms_adamw")
    params = [w, b, layer.flat_param]
    for p in params:
        p.grad = torch.randn_like(p) * 0.01
    start = [p.detach().float().clone() for p in params]
    versions = [p._version for p in params]
    seen = []
    opt.add_step_hook(w, seen.append)
    for _ in range(2):
        opt.step()
    assert all(p._version >= v + 2 for p, v in zip(params, versions)) and len(seen) == 2
    kw = dict(momentum=0.95, weight_decay=0.1, adjust="match_rms_adamw")
    # the same by hand
    m, mine = torch.zeros(160, 200, device=dev), start[0].clone()
    low = None if dt == torch.float32 else [torch.empty_like(w)]
    for _ in range(2):
        K.muon_multi([mine], [w.grad], [m], lr=0.01, lowp_outs=low, **kw)
    assert torch.equal(opt.master_param(w).view(160, 200), mine) and torch.equal(w.detach().float(), mine.to(dt).float())
    assert torch.equal(opt.moments(w), m.view(-1))
    flat, grad = start[2].clone(), layer.flat_param.grad
    ps = [flat[a:a + r * c].view(r, c) for a, r, c in mats]
    ms = [torch.zeros(r, c, device=dev) for _, r, c in mats]
    gs = [grad[a:a + r * c].view(r, c) for a, r, c in mats]
    rest = slice(mats[-1][0] + 128 * 256, None)
    v1, v2 = torch.zeros(256, device=dev), torch.zeros(256, device=dev)
    for t in (1, 2):
        K.muon_multi(ps, gs, ms, lr=3e-3, **kw)
        K.adamw_step(flat[rest], grad[rest], v1, v2, step=t, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
                     weight_decay=0.1)
    assert torch.equal(opt.master_param(layer.flat_param), flat)
    assert torch.equal(layer.flat_param.detach(), flat.to(dt))


def test_resumed_runs_repeat(dev):
    import copy
    from zorse_amd import optim
    torch.manual_seed(0)
    w = torch.nn.Parameter(torch.randn(140, 150, device=dev).to(BF))
    b = torch.nn.Parameter(torch.randn(33, device=dev).to(BF))
    opt = optim.Muon([w, b])
    for p in (w, b):
        p.grad = torch.randn_like(p)
    opt.step()
    saved, at = copy.deepcopy(opt.state_dict()), [w.detach().clone(), b.detach().clone()]
    opt.step()
    end = [w.detach().clone(), b.detach().clone()]
    with torch.no_grad():
        w.copy_(at[0])
        b.copy_(at[1])
    other = optim.Muon([w, b], lr=7.0)
    other.load_state_dict(saved)
    other.step()
    assert torch.equal(w.detach(), end[0]) and torch.equal(b.detach(), end[1])


def test_a_stage_steps_with_muon(dev):
    from zorse_amd import llama_simple, optim
    from zorse_amd.stage import StageRunner
    cfg = llama_simple.llama_config(hidden_size=256, num_attention_heads=2, num_key_value_heads=1,
                                    intermediate_size=512, rope_theta=1e4)

    def build():
        g = torch.Generator().manual_seed(0)
        return [llama_simple.LlamaDecoderLayer(cfg, i, init_std=0.02, generator=g, param_dtype=BF).to(dev)
                for i in range(2)]

    x = torch.randn(1, 128, 256, device=dev).to(BF)
    dout = torch.randn(1, 128, 256, device=dev).to(BF)
    layers = build()
    stage = StageRunner(layers, optimizer=lambda layer, params: optim.Muon(
        params, lr=0.01, matrices=optim.flat_matrices(layer)))
    stage.step(x, dout)
    torch.cuda.synchronize()
    twins = build()
    y = x.clone().requires_grad_()
    h = y
    for layer in twins:
        h = layer(h)[0]
    h.backward(dout)
    for layer, twin in zip(layers, twins):
        opt = optim.Muon([twin.flat_param], lr=0.01, matrices=optim.flat_matrices(twin))
        opt.step()
        assert torch.equal(layer.flat_param, twin.flat_param)

"""Performance cases of a training step over packed sequences.

Each case is one pass through an operator as a training program calls it:
  attention  functional.packed_attention: softmax attention within each of the
             sequences that lie one after another in one run of tokens (causal,
             with or without a sliding window, or over the whole sequence), with
             grouped heads; forward only or with all gradients;
  rope       functional.rope_axes: the rotation of query and key heads by
             positions of several axes (time, height, width); forward only or
             with both gradients;
  muon       kernels.orthogonalize: the orthogonal factors of a list of
             gradient matrices by Newton-Schulz products, or kernels.muon_multi:
             the momentum, the factors and the step of the weights.

``listed`` names the workloads, ``draw`` takes others from the same ranges.
Where ``own`` is false, ``run`` computes the same in elementary torch
operations.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # three short prompts of the smallest test model in one call: latency
        {"name": "attn_short_prompts", "op": "attention", "mode": "forward", "tokens": 64,
         "pad": 1, "shortest": 1, "longest": 45, "lengths": 3, "heads": 4, "kv_heads": 2,
         "dim": 64, "causal": True, "window": 0, "dtype": "bf16"},
        # the 7B layer's micro-batch of 4096 tokens filled with documents
        {"name": "attn_7b_documents_train", "op": "attention", "mode": "train", "tokens": 4096,
         "pad": 0, "shortest": 30, "longest": 2500, "lengths": 1, "heads": 32, "kv_heads": 32,
         "dim": 128, "causal": True, "window": 0, "dtype": "bf16"},
        # a whole prompt of 8192 tokens with grouped heads: the most work a call has
        {"name": "attn_gqa_long_train", "op": "attention", "mode": "train", "tokens": 8192,
         "pad": 0, "shortest": 8192, "longest": 8192, "lengths": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "window": 0, "dtype": "bf16"},
        # sliding window over long and short texts, the batch not filled
        {"name": "attn_window_train", "op": "attention", "mode": "train", "tokens": 8000,
         "pad": 77, "shortest": 100, "longest": 6000, "lengths": 2, "heads": 32, "kv_heads": 8,
         "dim": 64, "causal": True, "window": 1024, "dtype": "fp16"},
        # images of different sizes, every patch sees its whole image; head dim 100
        {"name": "attn_images_train", "op": "attention", "mode": "train", "tokens": 5001,
         "pad": 13, "shortest": 64, "longest": 1100, "lengths": 4, "heads": 16, "kv_heads": 16,
         "dim": 100, "causal": False, "window": 0, "dtype": "bf16"},
        # an fp32 layer's packed sequences
        {"name": "attn_fp32_train", "op": "attention", "mode": "train", "tokens": 1111, "pad": 0,
         "shortest": 5, "longest": 500, "lengths": 5, "heads": 8, "kv_heads": 4, "dim": 64,
         "causal": True, "window": 0, "dtype": "fp32"},
        # one new token for each of three sequences: latency
        {"name": "rope_single_tokens", "op": "rope", "mode": "forward", "tokens": 3, "heads": 32,
         "kv_heads": 8, "dim": 128, "axes": 3, "turns": False, "interleaved": False,
         "dtype": "bf16"},
        # a packed batch of text and video frames, grouped heads of 128
        {"name": "rope_video_train", "op": "rope", "mode": "train", "tokens": 16384, "heads": 32,
         "kv_heads": 8, "dim": 128, "axes": 3, "turns": False, "interleaved": False,
         "dtype": "bf16"},
        # image patches with height and width, the axes in turn, head dim 100, fp32
        {"name": "rope_images_train", "op": "rope", "mode": "train", "tokens": 5001, "heads": 16,
         "kv_heads": 16, "dim": 100, "axes": 2, "turns": True, "interleaved": True,
         "dtype": "fp32"},
        # the few small matrices of a test model: launches
        {"name": "muon_small_factors", "op": "muon", "mode": "factors", "matrices": 4, "rows": 256,
         "cols": 256, "tall": 2, "ragged": False, "seed": 1, "dtype": "fp32"},
        # matrices of odd shapes, wide and tall
        {"name": "muon_odd_factors", "op": "muon", "mode": "factors", "matrices": 5, "rows": 1000,
         "cols": 2753, "tall": 2, "ragged": True, "seed": 2, "dtype": "fp16"},
        # a decoder layer of the 7B model: q, k, v, o, gate, up and down
        {"name": "muon_7b_layer_step", "op": "muon", "mode": "step", "matrices": 7, "rows": 4096,
         "cols": 11008, "tall": 3, "ragged": False, "seed": 7, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above: 1 to 8192 tokens in sequences from one
    token on, up to 32 heads of even dims up to 128; 1 to 16384 tokens with up
    to 4 axes; 1 to 8 matrices of 16 to 11008 rows."""
    while True:
        case = _draw(rng)
        w = work(case)
        if case["op"] == "attention":
            fits = case["tokens"] ** 2 * case["heads"] <= 8192 ** 2 * 32 and w["flops"] <= 1.9e12
        else:
            fits = w["bytes"] <= 1.5e9 if case["op"] == "rope" else w["flops"] <= 1.4e13
        if fits:
            return case


def _draw(rng):
    op = rng.choice(["attention", "attention", "rope", "muon"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    mode = rng.choice(["forward", "train", "train"])
    if op == "muon":
        rows, cols = _log(rng, 16, 11008), _log(rng, 16, 11008)
        n = rng.randint(1, 8)
        return {"op": op, "mode": rng.choice(["factors", "step"]), "matrices": n, "rows": rows,
                "cols": cols, "tall": rng.randint(0, n), "ragged": rng.random() < 0.5,
                "seed": rng.randint(0, 999), "dtype": dtype}
    kv = _log(rng, 1, 16)
    heads = kv * rng.choice([g for g in (1, 2, 4, 5, 8) if kv * g <= 32])
    if op == "rope":
        axes = rng.choice([1, 2, 3, 3, 4])
        return {"op": op, "mode": mode, "tokens": _log(rng, 1, 16384), "heads": heads,
                "kv_heads": kv, "dim": rng.choice([64, 128, 128, 2 * rng.randint(4, 128)]),
                "axes": axes, "turns": rng.random() < 0.4, "interleaved": rng.random() < 0.3,
                "dtype": dtype}
    tokens = _log(rng, 1, 2000 if dtype == "fp32" else 8192)
    pad = rng.choice([0, 0, rng.randint(0, tokens // 10)])
    longest = _log(rng, 1, tokens - pad) if tokens > pad else 1
    causal = rng.random() < 0.75
    return {"op": op, "mode": mode, "tokens": tokens, "pad": pad,
            "shortest": _log(rng, 1, longest), "longest": longest, "lengths": rng.randint(0, 999),
            "heads": heads, "kv_heads": kv,
            "dim": rng.choice([64, 128, 128, 2 * rng.randint(8, 64)]), "causal": causal,
            "window": _log(rng, 1, tokens) if causal and rng.random() < 0.3 else 0,
            "dtype": dtype}


def _lengths(case):
    """The sequences' lengths, log-uniform from the shortest to the longest, the
    last cut to fit; now and then a sequence without a token."""
    r, left, out = random.Random(case["lengths"]), case["tokens"] - case["pad"], []
    while left > 0:
        n = min(left, _log(r, case["shortest"], case["longest"]))
        out.append(n)
        left -= n
        if r.random() < 0.1:
            out.append(0)
    return out


def _pairs(n, case):
    """(query, key) pairs of a sequence of n tokens that see each other."""
    if not case["causal"]:
        return n * n
    w = case["window"] if 0 < case["window"] < n else n
    return w * (w + 1) // 2 + (n - w) * w


def _shapes(case):
    """The matrices: the last ``tall`` of rows x cols have cols rows (a layer's
    first ones are square); ragged ones vary from a half to the whole."""
    r, out = random.Random(case["seed"]), []
    for i in range(case["matrices"]):
        m, n = case["rows"], case["cols"]
        if case["ragged"]:
            m, n = r.randint((m + 1) // 2, m), r.randint((n + 1) // 2, n)
        elif i < case["matrices"] - case["tall"]:
            n = m
        out.append((n, m) if i >= case["matrices"] - case["tall"] else (m, n))
    return out


def work(case):
    """Bytes: every input once and every output once.  Operations: two for each
    product of a matrix product that cannot be left out (products whose result
    is symmetric count half), one for each of an elementwise formula."""
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        T, H, Hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        pairs = sum(_pairs(n, case) for n in _lengths(case)) * H
        if case["mode"] == "forward":
            return {"bytes": T * d * (2 * H + 2 * Hk) * e, "flops": 4 * d * pairs}
        return {"bytes": T * d * (4 * H + 4 * Hk) * e, "flops": 14 * d * pairs}
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 1 if case["mode"] == "forward" else 2
        return {"bytes": passes * (2 * n * e + 8 * case["axes"] * case["tokens"]),
                "flops": passes * 3 * n}
    flops = elements = 0
    for m, n in _shapes(case):
        s, t = min(m, n), max(m, n)
        flops += STEPS * (s * s * t + s * s * s + 2 * s * s * t)
        elements += m * n
    per = 2 * e if case["mode"] == "factors" else e + 16
    return {"bytes": per * elements, "flops": flops}


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 41)


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    dt = DTYPES[case["dtype"]]
    if case["op"] == "muon":
        return _prepare_muon(st, case, g, dt)
    T, H, Hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    train = case["mode"] == "train"
    # q | k | v as one projection writes them
    qkv = _randn(g, (T, (H + 2 * Hk) * d), dt)
    st["q"] = qkv[:, :H * d].unflatten(1, (H, d)).requires_grad_(train)
    st["k"] = qkv[:, H * d:(H + Hk) * d].unflatten(1, (Hk, d)).requires_grad_(train)
    if case["op"] == "rope":
        if train:
            st["dq"], st["dk"] = _randn(g, (T, H, d), dt), _randn(g, (T, Hk, d), dt)
        return _prepare_rope(st, case, seed)
    st["v"] = qkv[:, (H + Hk) * d:].unflatten(1, (Hk, d)).requires_grad_(train)
    if train:
        st["do"] = _randn(g, (T, H, d), dt)
    lengths = _lengths(case)
    random.Random(seed).shuffle(lengths)
    ends = torch.tensor([0] + lengths).cumsum(0)
    st["offsets"] = ends.to("cuda", torch.int32)
    if own:  # laid out once a batch, for every layer
        from zorse_amd import functional
        st["sequences"] = functional.PackedSequences(st["offsets"], T)
    return st


def _prepare_rope(st, case, seed):
    T, d, A = case["tokens"], case["dim"], case["axes"]
    # text advances on every axis at once, an image or a clip by its own rows
    # and columns
    r, rows, at = random.Random(seed), [], 3 * seed % 17
    while sum(x.shape[1] for x in rows) < T:
        if r.random() < 0.4:
            n = r.randint(1, 300)
            rows.append((at + torch.arange(n)).expand(A, n))
            at += n
        else:
            grid = [r.randint(1, 24) for _ in range(A)]
            axes = torch.meshgrid(*(torch.arange(n) for n in grid), indexing="ij")
            rows.append(at + torch.stack([x.reshape(-1) for x in axes])[:, :4000])
            at += max(grid)
    st["positions"] = torch.cat(rows, 1)[:, :T].contiguous().to("cuda")
    at = int(st["positions"].max()) + 1
    half = d // 2
    if case["turns"]:
        st["pair_axes"] = [i % A for i in range(half)]
    else:
        st["pair_axes"] = sorted(i % A for i in range(half))
    inv = 1e4 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    ang = torch.arange(at, device="cuda", dtype=torch.float64)[:, None] * inv
    st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    return st


def _prepare_muon(st, case, g, dt):
    st["grads"], shapes = [], _shapes(case)
    for m, n in shapes:
        # a few strong directions over noise, as gradients of a batch have
        k = max(1, min(m, n) // 16)
        strong = torch.randn(m, k, generator=g, device="cuda") * torch.rand(
            k, generator=g, device="cuda").square() * (4.0 / math.sqrt(k))
        x = strong @ torch.randn(k, n, generator=g, device="cuda")
        st["grads"].append(((x + torch.randn(m, n, generator=g, device="cuda")) * 1e-3).to(dt))
    if case["mode"] == "step":
        st["params"] = [_randn(g, s, torch.float32, 0.02) for s in shapes]
        st["momenta"] = [_randn(g, s, torch.float32, 5e-4) for s in shapes]
        st["lows"] = None if dt == torch.float32 else [p.to(dt) for p in st["params"]]
    return st


STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
HYPER = {"lr": 1e-3, "momentum": 0.95, "weight_decay": 0.1, "nesterov": True}


# ------------------------------------------------------------------ passes --

def run(st):
    case = st["case"]
    if case["op"] == "attention":
        return _run_attention(st, case)
    if case["op"] == "rope":
        return _run_rope(st, case)
    return _run_muon(st, case)


def _run_attention(st, case):
    if own:
        from zorse_amd import functional
        o = functional.packed_attention(st["q"], st["k"], st["v"], st["sequences"],
                                        causal=case["causal"], window=case["window"])
        if case["mode"] == "forward":
            return o
        return o.detach(), *torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"])
    T, H, Hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    dt = DTYPES[case["dtype"]]
    # heads first; each key head serves H / Hk query heads, one after another
    q, k, v = (st[x].detach().float().transpose(0, 1).contiguous() for x in "qkv")
    q = q.view(Hk, H // Hk * T, d)
    at = torch.arange(T, device="cuda")
    # rows behind the last sequence belong to none
    which = (at[:, None] >= st["offsets"][None].long()).sum(1)
    seen = (which[:, None] == which[None]) & (at < st["offsets"][-1])
    if case["causal"]:
        seen &= at[None] <= at[:, None]
    if case["window"] > 0:
        seen &= at[None] > at[:, None] - case["window"]
    scale = 1.0 / math.sqrt(d)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(scale).view(Hk, H // Hk, T, T)
    s = s.masked_fill_(~seen, -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    p = s.div_(s.sum(-1, keepdim=True).clamp_(min=1e-30)).view(Hk, H // Hk * T, T)
    o = torch.bmm(p, v)
    out = o.view(H, T, d).transpose(0, 1).to(dt)
    if case["mode"] == "forward":
        return out
    do = st["do"].float().transpose(0, 1).contiguous().view(Hk, H // Hk * T, d)
    pt = p.transpose(1, 2).contiguous()
    dv = torch.bmm(pt, do)
    del pt
    ds = torch.bmm(do, v.transpose(1, 2).contiguous()).sub_((do * o).sum(-1, keepdim=True))
    ds = ds.mul_(p).mul_(scale)
    dq = torch.bmm(ds, k)
    del p, s
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q)
    return (out, dq.view(H, T, d).transpose(0, 1).to(dt), dk.transpose(0, 1).to(dt),
            dv.transpose(0, 1).to(dt))


def _rotate(x, cos, sin, interleaved):
    """x [T, H, d] with the pairs' angles [T, 1, d/2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _run_rope(st, case):
    if own:
        from zorse_amd import functional
        y = functional.rope_axes(st["q"], st["k"], st["cos"], st["sin"], st["positions"],
                                 st["pair_axes"], interleaved=case["interleaved"])
        if case["mode"] == "forward":
            return y
        grads = torch.autograd.grad(y, (st["q"], st["k"]), (st["dq"], st["dk"]))
        return y[0].detach(), y[1].detach(), *grads
    dt = DTYPES[case["dtype"]]
    pair = torch.arange(case["dim"] // 2, device="cuda")
    pos = st["positions"][st["pair_axes"]].t()  # [T, d/2]
    cos, sin = st["cos"][pos, pair][:, None], st["sin"][pos, pair][:, None]
    outs = [_rotate(st[x].detach().float(), cos, sin, case["interleaved"]).to(dt) for x in "qk"]
    if case["mode"] == "train":  # the transpose: the opposite angle
        outs += [_rotate(st[x].float(), cos, -sin, case["interleaved"]).to(dt)
                 for x in ("dq", "dk")]
    return tuple(outs)


def _factor(x):
    """The orthogonal factor of x by Newton-Schulz products, in fp32."""
    x = x.float()
    x = x / (x.square().sum(dtype=torch.float64).sqrt().float() + EPS)
    a, b, c = COEFFICIENTS
    if x.shape[0] > x.shape[1]:
        x = x.t().contiguous()
        turned = True
    else:
        turned = False
    for _ in range(STEPS):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if turned else x


def _run_muon(st, case):
    dt = DTYPES[case["dtype"]]
    if own:
        from zorse_amd import kernels
        if case["mode"] == "factors":
            return kernels.orthogonalize(st["grads"], steps=STEPS, coefficients=COEFFICIENTS,
                                         eps=EPS, dtype=_factor_type(case))
        kernels.muon_multi(st["params"], st["grads"], st["momenta"], lowp_outs=st["lows"],
                           steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, **HYPER)
        return _step_outputs(st)
    if case["mode"] == "factors":
        return [_factor(g).to(_factor_type(case)).contiguous() for g in st["grads"]]
    mu, lr = HYPER["momentum"], HYPER["lr"]
    for i, (p, g, m) in enumerate(zip(st["params"], st["grads"], st["momenta"])):
        g = g.float()
        m.mul_(mu).add_(g, alpha=1 - mu)
        o = _factor(g * (1 - mu) + m * mu)
        p.mul_(1 - lr * HYPER["weight_decay"]).sub_(
            o * (lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))))
        if st["lows"] is not None:
            st["lows"][i].copy_(p)
    return _step_outputs(st)


def _factor_type(case):
    """The factors of fp32 gradients are bf16: their singular values lie
    anywhere from 0.7 to 1.2."""
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _step_outputs(st):
    outs = {"params": st["params"], "momenta": st["momenta"]}
    if st["lows"] is not None:
        outs["lows"] = st["lows"]
    return outs


# ------------------------------------------------------- the definitions ----

def exact(case, seed):
    """What ``run`` returns for these inputs, from the definitions in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(st, case)
    if case["op"] == "rope":
        return _exact_rope(st, case)
    return _exact_muon(st, case)


def _exact_attention(st, case):
    """Sequence by sequence and head by head, the gradients by the softmax's
    Jacobian."""
    T, H, Hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    train = case["mode"] == "train"
    q, k, v = (st[x].detach().double() for x in "qkv")
    o, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    ends = st["offsets"].tolist()
    for lo, hi in zip(ends, ends[1:]):
        n = hi - lo
        i = torch.arange(n, device="cuda")
        gap = i[:, None] - i[None]
        hidden = torch.zeros(n, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden = gap < 0
        if case["window"] > 0:
            hidden = hidden | (gap >= case["window"])
        for h in range(H if n else 0):
            g = h * Hk // H
            a, b, c = q[lo:hi, h], k[lo:hi, g], v[lo:hi, g]
            p = torch.softmax((a @ b.t() / math.sqrt(d)).masked_fill(hidden, -math.inf), 1)
            o[lo:hi, h] = p @ c
            if train:
                up = st["do"][lo:hi, h].double()
                dp = up @ c.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dv[lo:hi, g] += p.t() @ up
                dq[lo:hi, h] = ds @ b
                dk[lo:hi, g] += ds.t() @ a
    return (o, dq, dk, dv) if train else o


def _exact_rope(st, case):
    """The pairs as complex numbers, times the unit number of their angle."""
    axis = torch.tensor(st["pair_axes"], device="cuda")
    turn = torch.complex(st["cos"].double(), st["sin"].double())
    index = st["positions"].index_select(0, axis)  # [d/2, T]
    turn = torch.gather(turn.t(), 1, index).t()[:, None]
    res = []
    for name, back in (("q", False), ("k", False), ("dq", True), ("dk", True)):
        if name not in st:
            continue
        x = st[name].detach().double()
        half = x.shape[-1] // 2
        if case["interleaved"]:
            z = torch.view_as_complex(x.contiguous().unflatten(-1, (half, 2)))
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())
        z = z * (turn.conj() if back else turn)
        parts = (z.real, z.imag)
        res.append(torch.stack(parts, -1).flatten(-2) if case["interleaved"]
                   else torch.cat(parts, -1))
    return tuple(res)


def _exact_factor(x):
    """The same polynomials through the smaller Gram matrix: with S the product
    of the steps' q(G) = a + b G + c G G, the factor is S x (or x S)."""
    x = x / (torch.linalg.vector_norm(x) + EPS)
    tall = x.shape[0] > x.shape[1]
    a, b, c = COEFFICIENTS
    one = torch.eye(min(x.shape), dtype=torch.float64, device="cuda")
    for _ in range(STEPS):
        gram = x.mT @ x if tall else x @ x.mT
        poly = a * one + gram @ (b * one + c * gram)
        x = x @ poly if tall else poly @ x
    return x


def _exact_muon(st, case):
    if case["mode"] == "factors":
        return [_exact_factor(g.double()) for g in st["grads"]]
    mu, lr, wd = HYPER["momentum"], HYPER["lr"], HYPER["weight_decay"]
    outs = {"params": [], "momenta": []}
    for p, g, m in zip(st["params"], st["grads"], st["momenta"]):
        m = mu * m.double() + (1 - mu) * g.double()
        o = _exact_factor((1 - mu) * g.double() + mu * m)
        wide = max(1.0, p.shape[0] / p.shape[1])
        outs["params"].append(p.double() - lr * (wd * p.double() + math.sqrt(wide) * o))
        outs["momenta"].append(m)
    if st["lows"] is not None:
        outs["lows"] = outs["params"]
    return outs

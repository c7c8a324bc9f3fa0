"""Performance cases of the operators around a decoder stack's layers.

Each case is one pass through an operator as a training program calls it:
  embedding  functional.embedding: rows of a token table, scaled; forward only
             or with the table's gradient; or kernels.embedding_bwd adding a
             micro-batch's gradient to a buffer that holds the earlier ones';
  qk         functional.qk_norm_rope: RMS norm of every query and key head with
             the position rotation in the same pass; forward only or with all
             gradients;
  adamw      one AdamW step over a list of tensors, with both moments in 32
             bits (kernels.adamw_multi) or in 8 (kernels.adamw8_multi, after
             which kernels.adamw8_values reads the moments back as the
             values that their codes stand for, as a checkpoint does).

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
BLOCK = 256  # elements that share the offset of their 8-bit codes


def listed():
    return [
        # a short prompt's lookup in the smallest test model: a launch
        {"name": "embed_toy_forward", "op": "embedding", "mode": "forward", "batch": 1,
         "seq": 37, "hidden": 256, "vocab": 320, "ids": "uniform", "pad": -1, "scale": 1.0,
         "dtype": "fp32", "out": "fp32"},
        # the first pipeline stage of the 7B model, micro-batch 1: text's own
        # distribution of tokens, the whole table's gradient
        {"name": "embed_7b_train", "op": "embedding", "mode": "train", "batch": 1, "seq": 4096,
         "hidden": 4096, "vocab": 49152, "ids": "zipf", "pad": -1, "scale": 1.0,
         "dtype": "bf16", "out": "bf16"},
        # a padded batch of odd lengths with embeddings scaled by sqrt(hidden):
        # nearly half the tokens are padding, which takes no gradient
        {"name": "embed_padded_scaled", "op": "embedding", "mode": "train", "batch": 8,
         "seq": 2039, "hidden": 2048, "vocab": 32000, "ids": "padded", "pad": 0,
         "scale": 45.25, "dtype": "fp16", "out": "fp16"},
        # the last micro-batch of a large batch: 16-bit gradients of 65536
        # tokens added to the fp32 gradient of the 13B model's table
        {"name": "embed_13b_accumulate", "op": "embedding", "mode": "accumulate", "batch": 16,
         "seq": 4096, "hidden": 5120, "vocab": 49152, "ids": "zipf", "pad": -1, "scale": 1.0,
         "dtype": "fp32", "out": "bf16"},
        # one token for each of three sequences at far positions (generating
        # samples between training steps): latency
        {"name": "qk_single_token", "op": "qk", "mode": "forward", "batch": 3, "seq": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "far": 8000, "rows": True,
         "interleaved": False, "dtype": "bf16"},
        # the 7B layer's heads at 4096 tokens
        {"name": "qk_7b_train", "op": "qk", "mode": "train", "batch": 1, "seq": 4096,
         "heads": 32, "kv_heads": 32, "dim": 128, "far": 0, "rows": False,
         "interleaved": False, "dtype": "bf16"},
        # grouped-query heads, several packed sequences of odd length with
        # positions of their own
        {"name": "qk_gqa_packed_train", "op": "qk", "mode": "train", "batch": 5, "seq": 6007,
         "heads": 32, "kv_heads": 8, "dim": 128, "far": 2000, "rows": True,
         "interleaved": False, "dtype": "bf16"},
        # the 3B model's head dim in fp32, interleaved pairs
        {"name": "qk_3b_fp32_train", "op": "qk", "mode": "train", "batch": 1, "seq": 2048,
         "heads": 32, "kv_heads": 32, "dim": 100, "far": 0, "rows": False,
         "interleaved": True, "dtype": "fp32"},
        # the norm weights of a 32-layer model held as tensors of their own
        {"name": "adamw_norms", "op": "adamw", "bits": 32, "set": "norms", "tensors": 65,
         "numel": 4096, "seed": 0, "step": 11,
         "packed": False, "dtype": "fp32"},
        # a two-layer stage of the tiny model with its table, norm and head
        {"name": "adamw_tiny_stage", "op": "adamw", "bits": 32, "set": "stage", "tensors": 5,
         "numel": 51384320, "seed": 2048, "step": 200,
         "packed": False, "dtype": "bf16"},
        # adapters and biases of all sizes, 8-bit moments
        {"name": "adamw8_mixed", "op": "adamw", "bits": 8, "set": "mixed", "tensors": 150,
         "numel": 300000, "seed": 5, "step": 3,
         "packed": True, "dtype": "fp32"},
        # a layer of the 7B model with the table and head of its stage, 8-bit
        # moments: the states that decide whether the model fits
        {"name": "adamw8_7b_stage", "op": "adamw", "bits": 8, "set": "stage", "tensors": 4,
         "numel": 202383360, "seed": 4096, "step": 1000,
         "packed": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above: 1 to 65536 tokens, tables of 100 to
    131072 rows; 1 to 40 heads of even dims up to 256; 1 to 200 tensors of 1 to
    2e8 elements."""
    while True:
        case = _draw(rng)
        if work(case)["bytes"] <= 6.5e9:
            return case


def _draw(rng):
    op = rng.choice(["embedding", "embedding", "qk", "qk", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embedding":
        hidden = _log(rng, 64, 5120)
        if rng.random() < 0.7:
            hidden = hidden // 8 * 8
        tokens = _log(rng, 1, 65536)
        batch = rng.choice([b for b in (1, 2, 3, 8) if b <= tokens])
        mode = rng.choice(["forward", "train", "train", "accumulate"])
        ids = rng.choice(["uniform", "zipf", "padded", "one"])
        return {"op": op, "mode": mode, "batch": batch, "seq": max(1, tokens // batch),
                "hidden": hidden, "vocab": _log(rng, 100, 131072), "ids": ids,
                "pad": 0 if ids == "padded" and rng.random() < 0.6 else -1,
                "scale": rng.choice([1.0, 1.0, round(math.sqrt(hidden), 2)]), "dtype": dtype,
                "out": rng.choice([dtype, dtype, "bf16"])}
    if op == "qk":
        kv = _log(rng, 1, 32)
        heads = kv * rng.choice([g for g in (1, 2, 4, 5, 8) if kv * g <= 40])
        dim = rng.choice([64, 128, 128, 256, 2 * rng.randint(1, 128)])
        tokens = _log(rng, 1, 32768)
        batch = rng.choice([b for b in (1, 2, 3, 5) if b <= tokens])
        return {"op": op, "mode": rng.choice(["forward", "train", "train"]), "batch": batch,
                "seq": max(1, tokens // batch), "heads": heads, "kv_heads": kv, "dim": dim,
                "far": rng.choice([0, 0, 10000]), "rows": rng.random() < 0.4,
                "interleaved": rng.random() < 0.4, "dtype": dtype}
    kind = rng.choice(["norms", "mixed", "stage"])
    if kind == "norms":
        tensors, numel = rng.randint(1, 200), _log(rng, 1, 8192)
    elif kind == "mixed":
        tensors, numel = rng.randint(1, 200), _log(rng, 10, 3000000)
    else:
        tensors, numel = rng.randint(3, 6), _log(rng, 100000, 202383360)
    return {"op": "adamw", "bits": rng.choice([8, 32]), "set": kind, "tensors": tensors,
            "numel": numel, "seed": rng.choice([512, 1024, 2048]) if kind == "stage"
            else rng.randint(0, 999), "step": _log(rng, 1, 100000),
            "packed": rng.random() < 0.3, "dtype": dtype}


def _sizes(case):
    """Elements of each tensor: equal vectors; log-uniform sizes up to numel;
    or a stage's flat layers of numel elements between a table, a norm and a
    head whose width is the case's seed."""
    n, numel, kind = case["tensors"], case["numel"], case["set"]
    if kind == "norms":
        return [numel] * n
    if kind == "mixed":
        r = random.Random(case["seed"])
        return [max(1, int(math.exp(r.uniform(0.0, math.log(numel))))) for _ in range(n)]
    h = case["seed"]
    table = min(49152, max(1, numel // h)) * h
    return [table] + [numel] * (n - 3) + [h, table]


def _arena(case, per, dtype):
    """(flat, views): one allocation for a list of tensors, as a program that
    saves or reduces them in one piece keeps them.  They start at multiples of
    256 elements, or each where the one before ends."""
    at, starts = 0, []
    for n in per:
        starts.append(at)
        at += n if case["packed"] else -(-n // 256) * 256
    flat = torch.zeros(at, device="cuda", dtype=dtype)
    return flat, [flat[a:a + n] for a, n in zip(starts, per)]


def _bytes(name):
    return 4 if name == "fp32" else 2


def work(case):
    """Bytes: every input once and every output once.  Operations: one for
    each sum, product, root and quotient of the formulas."""
    if case["op"] == "embedding":
        T, h, V = case["batch"] * case["seq"], case["hidden"], case["vocab"]
        w, y = _bytes(case["dtype"]), _bytes(case["out"])
        rows = min(V, T)  # at most: a text names fewer
        fwd = rows * h * w + T * h * y + 8 * T
        if case["mode"] == "forward":
            return {"bytes": fwd, "flops": T * h}
        if case["mode"] == "train":
            return {"bytes": fwd + T * h * y + V * h * w, "flops": 2 * T * h}
        # the rows that tokens name are read and written
        return {"bytes": T * h * y + 8 * T + 2 * rows * h * w, "flops": T * h}
    if case["op"] == "qk":
        n = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        e = _bytes(case["dtype"])
        if case["mode"] == "forward":
            return {"bytes": 2 * n * e, "flops": 7 * n}
        return {"bytes": 5 * n * e, "flops": 22 * n}
    n, g = sum(_sizes(case)), _bytes(case["dtype"])
    copy = 2 if case["dtype"] != "fp32" else 0
    if case["bits"] == 32:
        return {"bytes": n * (24 + g + copy), "flops": 14 * n}
    return {"bytes": n * (8 + g + copy + 4 + 4), "flops": 20 * n}


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _ids(case, g):
    B, S, V = case["batch"], case["seq"], case["vocab"]
    u = torch.rand(B, S, generator=g, device="cuda", dtype=torch.float64)
    if case["ids"] == "uniform":
        ids = (u * V).long()
    elif case["ids"] == "one":  # one token everywhere but for a few
        other = (torch.rand(B, S, generator=g, device="cuda") < 0.1) * (u * V).long()
        ids = other + (other == 0) * (V // 2)
    else:  # frequencies that fall as 1 / rank, as a text's do
        ids = (torch.exp(u * math.log(V + 1)) - 1.0).long()
    if case["ids"] == "padded":  # each sequence ends in token 0
        share = torch.rand(B, 1, generator=g, device="cuda")
        ids = ids * (torch.arange(S, device="cuda")[None] < share * S + 1)
    return ids.clamp_(0, V - 1)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    dt = DTYPES[case["dtype"]]
    if case["op"] == "embedding":
        out = DTYPES[case["out"]]
        B, S, h, V = case["batch"], case["seq"], case["hidden"], case["vocab"]
        st["ids"] = _ids(case, g)
        if case["mode"] == "accumulate":
            st["dw"] = _randn(g, (V, h), dt)
        else:
            st["weight"] = _randn(g, (V, h), dt, 0.02).requires_grad_(case["mode"] == "train")
        if case["mode"] != "forward":
            st["dy"] = _randn(g, (B, S, h), out)
        return st
    if case["op"] == "qk":
        B, S, Hq, Hk, d = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        train = case["mode"] == "train"
        # q | k | v as one projection writes them; v is not touched
        qkv = _randn(g, (B, S, (Hq + 2 * Hk) * d), dt)
        st["q"] = qkv[..., :Hq * d].unflatten(-1, (Hq, d)).requires_grad_(train)
        st["k"] = qkv[..., Hq * d:(Hq + Hk) * d].unflatten(-1, (Hk, d)).requires_grad_(train)
        for name in ("wq", "wk"):
            w = (1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
            st[name] = w.requires_grad_(train)
        start = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device="cuda")
        pos = start + torch.arange(S, device="cuda")[None]
        st["positions"] = pos.contiguous() if case["rows"] else None
        n_pos = S + (case["far"] if case["rows"] else 0)
        inv = 1e4 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        if train:
            st["dq"] = _randn(g, (B, S, Hq, d), dt)
            st["dk"] = _randn(g, (B, S, Hk, d), dt)
        return st
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    kinds = {"p": torch.float32, "g": dt, "low": dt, "m": torch.float32, "v": torch.float32}
    if case["bits"] == 8:  # the moments' values are kept in 16 bits, which hold every code's
        kinds |= {"m": torch.bfloat16, "v": torch.bfloat16, "m8": torch.uint8, "v8": torch.uint8}
        flat, views = _arena(case, [2 * b for b in blocks], torch.int16)
        st["base"] = [t.view(-1, 2) for t in views]
    for k, kind in kinds.items():
        st["flat_" + k], st[k] = _arena(case, sizes, kind)
    for i, n in enumerate(sizes):
        st["p"][i].copy_(_randn(g, (n,), torch.float32, 0.02))
        st["low"][i].copy_(st["p"][i])
        # gradients of very different sizes side by side, some rows untouched
        size = torch.exp(torch.randn((n + 63) // 64, generator=g, device="cuda") * 2.0 - 7.0)
        size = (size * (size < 0.01)).repeat_interleave(64)[:n]
        st["g"][i].copy_(torch.randn(n, generator=g, device="cuda") * size)
        m = torch.randn(n, generator=g, device="cuda") * size * 0.3
        v = (torch.rand(n, generator=g, device="cuda") + 0.5) * size * size
        if case["bits"] == 32:
            st["m"][i].copy_(m)
            st["v"][i].copy_(v)
            continue
        m8, mb = _pack(_nearest(m), 127)
        v8, vb = _pack(_nearest(v), 255)
        st["m8"][i].copy_(m8 | ((m < 0) & (m8 > 0)).to(torch.uint8) * 128)
        st["v8"][i].copy_(v8)
        st["base"][i].copy_(torch.stack((mb, vb), 1))
    if dt == torch.float32:
        st["low"] = None
    st["steps"] = [case["step"] + 7 * (i % 3) for i in range(len(sizes))]
    st["seeds"] = [(seed * 7919 + 104729 * i) % 2**32 for i in range(len(sizes))]
    return st


HYPER = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.1}


# ------------------------------------------------------------------ passes --

def run(st):
    case = st["case"]
    if case["op"] == "embedding":
        return _run_embedding(st, case)
    if case["op"] == "qk":
        return _run_qk(st, case)
    return _run_adamw(st, case)


def _run_embedding(st, case):
    pad = case["pad"] if case["pad"] >= 0 else None
    out = DTYPES[case["out"]]
    if own:
        from zorse_amd import functional, kernels
        if case["mode"] == "accumulate":
            return kernels.embedding_bwd(st["ids"], st["dy"], case["vocab"], scale=case["scale"],
                                         padding_idx=pad, dw=st["dw"], accumulate=True)
        y = functional.embedding(st["ids"], st["weight"], scale=case["scale"], padding_idx=pad,
                                 dtype=out)
        if case["mode"] == "forward":
            return y
        return y.detach(), torch.autograd.grad(y, st["weight"], st["dy"])[0]
    ids = st["ids"].reshape(-1)
    if case["mode"] != "accumulate":
        w = st["weight"].detach()
        y = (w[st["ids"]].float() * case["scale"]).to(out)
        if case["mode"] == "forward":
            return y
    dy = st["dy"].reshape(-1, case["hidden"]).float()
    if pad is not None:
        dy = dy * (ids != pad)[:, None]
    if case["mode"] == "train":
        dw = torch.zeros(case["vocab"], case["hidden"], device="cuda").index_add_(0, ids, dy)
        return y, (dw * case["scale"]).to(w.dtype)
    add = torch.zeros(case["vocab"], case["hidden"], device="cuda").index_add_(0, ids, dy)
    st["dw"].copy_(st["dw"].float() + add * case["scale"])
    return st["dw"]


def _rotate(x, cos, sin, interleaved):
    """x [B, S, H, d] with the pairs' angles [S or B S.., 1, d/2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _run_qk(st, case):
    if own:
        from zorse_amd import functional
        y = functional.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"],
                                    positions=st["positions"], eps=1e-6,
                                    interleaved=case["interleaved"])
        if case["mode"] == "forward":
            return y
        grads = torch.autograd.grad(y, (st["q"], st["k"], st["wq"], st["wk"]),
                                    (st["dq"], st["dk"]))
        return (y[0].detach(), y[1].detach(), *grads)
    pos = st["positions"]
    if pos is None:
        pos = torch.arange(case["seq"], device="cuda")
    cos, sin = st["cos"][pos].unsqueeze(-2), st["sin"][pos].unsqueeze(-2)
    outs, dxs, dws = [], [], []
    for x, w, dy in ((st["q"], st["wq"], st.get("dq")), (st["k"], st["wk"], st.get("dk"))):
        dt = x.dtype
        x, w = x.detach().float(), w.detach().float()
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        xh = x * rstd
        outs.append(_rotate(xh * w, cos, sin, case["interleaved"]).to(dt))
        if case["mode"] == "forward":
            continue
        dn = _rotate(dy.float(), cos, -sin, case["interleaved"])  # the transpose
        # a sum over every head of every token
        dws.append((dn * xh).double().sum((0, 1, 2)).to(dt))
        gw = dn * w
        dxs.append((rstd * (gw - xh * (gw * xh).mean(-1, keepdim=True))).to(dt))
    return (*outs, *dxs, *dws)


def _fma(a, b, c):
    """a b + c with one rounding: values next to a code's border."""
    return (a * b.double() + c.double()).float()


def _nearest(x):
    """The top 12 bits below the sign (8 of exponent, 3 of mantissa) of |x|,
    rounded to nearest, ties to even: an integer that grows with |x|."""
    b = x.view(torch.int32) & 0x7FFFFFFF
    return (b + 0x7FFFF + ((b >> 20) & 1)) >> 20


def _blocks(r):
    pad = -r.numel() % BLOCK
    return torch.cat((r, r.new_zeros(pad))).view(-1, BLOCK) if pad else r.view(-1, BLOCK)


def _pack(r, top):
    """(codes uint8 [n], base [blocks]): the block's largest r is code ``top``
    unless r itself fits; what lies ``top`` steps and more below it is 0."""
    rows = _blocks(r)
    base = (rows.amax(1) - top).clamp_(min=0)
    codes = (rows - base[:, None]).clamp_(min=0).view(-1)[:r.numel()]
    return codes.to(torch.uint8), base


def _value(code, base, low):
    """fp32 values of codes (bits ``low`` of them) with their blocks' bases."""
    c = (code & low).to(torch.int32)
    b = base.to(torch.int32).repeat_interleave(BLOCK)[:code.numel()]
    return (((c + b) << 20) * (c > 0)).view(torch.float32)


def _hash20(seed, n):
    """20 bits for each element of a tensor: index and seed mixed by
    products with the fractions of the roots of 2 and 3, in 32 bits."""
    i = torch.arange(n, device="cuda", dtype=torch.int64)
    x = ((i & 0xFFFFFFFF) * 0x9E3779B1 + (i >> 32) * 0x85157AF5 + seed) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return ((x ^ (x >> 16)) >> 12).to(torch.int32)


def _run_adamw(st, case):
    low = st["low"]
    outs = {k: st["flat_" + k] for k in ("p", "m", "v") + (("low",) if low is not None else ())}
    if own:
        from zorse_amd import kernels
        if case["bits"] == 32:
            kernels.adamw_multi(st["p"], st["g"], st["m"], st["v"], st["steps"], lowp_outs=low,
                                **HYPER)
        else:
            kernels.adamw8_multi(st["p"], st["g"], st["m8"], st["v8"], st["base"], st["steps"],
                                 seeds=st["seeds"], lowp_outs=low, **HYPER)
            kernels.adamw8_values(st["m8"], st["v8"], st["base"], outs=(st["m"], st["v"]))
        return outs
    b1, b2, lr = HYPER["beta1"], HYPER["beta2"], HYPER["lr"]
    f32 = {k: torch.tensor(x, dtype=torch.float32).item()
           for k, x in (("1-b1", 1 - b1), ("b2", b2), ("1-b2", 1 - b2))}
    for i, (p, g) in enumerate(zip(st["p"], st["g"])):
        g = g.float()
        if case["bits"] == 32:
            m, v = st["m"][i], st["v"][i]
        else:
            m, v = _values(st, i)
        m = _fma(f32["1-b1"], g - m, m)
        v = _fma(f32["1-b2"], g * g, v * f32["b2"])
        t = st["steps"][i]
        denom = v.sqrt() / math.sqrt(1 - b2 ** t) + HYPER["eps"]
        p.mul_(1 - lr * HYPER["weight_decay"]).sub_(m / denom * (lr / (1 - b1 ** t)))
        if low is not None:
            low[i].copy_(p)
        if case["bits"] == 8:
            codes, mb = _pack(_nearest(m), 127)
            st["m8"][i].copy_(codes | ((m < 0) & (codes > 0)).to(torch.uint8) * 128)
            # up to the next code with the probability of the fraction cut off;
            # a moment that is not zero never becomes zero
            r = (v.view(torch.int32) + _hash20(st["seeds"][i], v.numel())) >> 20
            codes, vb = _pack(r * (v > 0), 255)
            st["v8"][i].copy_(codes.clamp_(min=1) * (v > 0))
            st["base"][i].copy_(torch.stack((mb, vb), 1))
            m, v = _values(st, i)
        st["m"][i].copy_(m)
        st["v"][i].copy_(v)
    return outs


def _values(st, i):
    """Both moments of a tensor as the fp32 values of their codes."""
    c, base = st["m8"][i], st["base"][i]
    m = _value(c, base[:, 0], 127)
    return torch.where(c > 127, -m, m), _value(st["v8"][i], base[:, 1], 255)


# ------------------------------------------------------- the definitions ----

def exact(case, seed):
    """What ``run`` returns for these inputs, from the definitions in 64 bits."""
    if work(case)["bytes"] > 6e9:
        return None
    st = prepare(case, seed)
    if case["op"] == "embedding":
        return _exact_embedding(st, case)
    if case["op"] == "qk":
        return _exact_qk(st, case)
    outs, views = {}, {}
    for k in ("p", "m", "v") + (("low",) if st["low"] is not None else ()):
        outs[k], views[k] = _arena(case, _sizes(case), torch.float64)
    for i in range(len(st["p"])):
        for k, t in _exact_step(st, case, i).items():
            if k in views:
                views[k][i].copy_(t)
    return outs


def _exact_embedding(st, case):
    """The gradient as the ordered sums of each token's rows."""
    ids, V, s = st["ids"], case["vocab"], case["scale"]
    y = None
    if case["mode"] != "accumulate":
        rows = torch.index_select(st["weight"].detach().double(), 0, ids.flatten())
        y = (rows * s).view(*ids.shape, -1)
        if case["mode"] == "forward":
            return y
    dy = st["dy"].double().flatten(0, 1)
    order = torch.argsort(ids.flatten(), stable=True)
    count = torch.bincount(ids.flatten(), minlength=V)
    ends = count.cumsum(0)
    sums = torch.cat((dy.new_zeros(1, dy.shape[1]), dy[order].cumsum(0)))
    dw = s * (sums[ends] - sums[ends - count])
    if case["pad"] >= 0:
        dw[case["pad"]] = 0
    return dw + st["dw"].double() if case["mode"] == "accumulate" else (y, dw)


def _exact_qk(st, case):
    """Autograd of the norm and of the rotation as a complex product."""
    pos = st["positions"] if st["positions"] is not None else torch.arange(
        case["seq"], device="cuda")[None]
    turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, :, None]
    res, grads = [], []
    for x, w, dy in ((st["q"], st["wq"], st.get("dq")), (st["k"], st["wk"], st.get("dk"))):
        x, w = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        z = w * x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        d = z.shape[-1]
        pairs = z.unflatten(-1, (d // 2, 2) if case["interleaved"] else (2, d // 2))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        if not case["interleaved"]:
            turned = turned.transpose(-1, -2)
        y = turned.flatten(-2)
        res.append(y.detach())
        if case["mode"] == "train":
            grads.append(torch.autograd.grad(y, (x, w), dy.double()))
    if case["mode"] == "forward":
        return tuple(res)
    return (*res, grads[0][0], grads[1][0], grads[0][1], grads[1][1])


def _held(codes, base, top):
    """The signed values of codes below ``top`` (a set bit above them is a
    minus): eight steps an octave, without a leading one in the lowest."""
    index = torch.arange(codes.numel(), device="cuda") // BLOCK
    c = codes.long() % top
    r = c + base.long()[index]
    val = torch.where(r < 8, r % 8, 8 + r % 8) * torch.exp2((r // 8).clamp(min=1).double() - 130)
    return torch.where(c > 0, val, 0.0) * torch.where(codes.long() >= top, -1.0, 1.0)


def _on_grid(x, top, u=None):
    """x on its block's grid: to nearest, or down after u of a step was added
    (then at least one step, where x is not 0); what lies top steps and more
    below the block's largest is 0."""
    a = x.abs()
    octave = torch.frexp(a)[1].clamp(min=-125).long() - 1
    q = a * torch.exp2(3 - octave.double())
    q = torch.round(q) if u is None else torch.floor(q + u)
    r = torch.where(a > 0, (octave + 126) * 8 + q.long(), 0)
    index = torch.arange(x.numel(), device="cuda") // BLOCK
    most = torch.zeros(index[-1] + 1, dtype=torch.int64, device="cuda")
    most.scatter_reduce_(0, index, r, "amax")
    base = (most - top).clamp(min=0)[index]
    c = (r - base).clamp(min=0 if u is None else 1) * (a > 0)
    r = c + base
    val = torch.where(r < 8, r % 8, 8 + r % 8) * torch.exp2((r // 8).clamp(min=1).double() - 130)
    return torch.where(c > 0, val, 0.0) * torch.sign(x)


def _fractions(seed, n):
    """The 20 random bits of each element, as fractions of a step."""
    i = torch.arange(n, device="cuda", dtype=torch.int64)
    x = (i % 2 ** 32 * 2654435761 + i // 2 ** 32 * 2232777461 + seed) % 2 ** 32
    x = torch.bitwise_xor(x, x // 65536)
    x = x * 1779033703 % 2 ** 32
    x = torch.bitwise_xor(x, x // 32768)
    x = x * 3144134277 % 2 ** 32
    return (torch.bitwise_xor(x, x // 65536) // 4096).double() / 2 ** 20


def _exact_step(st, case, i):
    """One tensor's step; its 8-bit moments as multiples of their grid."""
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    p, g, t = st["p"][i].double(), st["g"][i].double(), st["steps"][i]
    if case["bits"] == 32:
        m, v = st["m"][i].double(), st["v"][i].double()
    else:
        m = _held(st["m8"][i], st["base"][i][:, 0], 128)
        v = _held(st["v8"][i], st["base"][i][:, 1], 256)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    root = torch.sqrt(v / (1 - b2 ** t)) + HYPER["eps"]
    p = p - HYPER["lr"] * (HYPER["weight_decay"] * p + m / (1 - b1 ** t) / root)
    if case["bits"] == 8:
        m, v = _on_grid(m, 127), _on_grid(v, 255, _fractions(st["seeds"][i], v.numel()))
    return {"p": p, "low": p, "m": m, "v": v}

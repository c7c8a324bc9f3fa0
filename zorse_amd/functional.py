"""Autograd functions over the HIP kernels (RMSNorm, RoPE + flash attention,
attention over packed sequences, the rotation by several axes, SwiGLU, token
embedding, the norm of query and key heads), usable on their own; the fused
decoder layer lives in ``layer.py``.

RoPE tables are built once per (S, d, theta, pairing, dtype, device) with the
reference's formula (models/llama_simple.py:75-81, 115-137: inv_freq and the
position product in fp32, cos/sin rounded to the activation dtype for the
half-split pairing; models/llama_v2.py:102-122 for the interleaved pairing,
which stays fp32) and handed to the kernel as fp32 [S, d/2] tables.
"""
from __future__ import annotations

import math
import threading

import torch

from . import kernels as K
from ._abi import nodes


# ------------------------------------------------------------- RoPE tables --

_rope_cache: dict = {}
_rope_lock = threading.Lock()


def rope_tables(seq: int, head_dim: int, theta: float, dtype: torch.dtype,
                device: torch.device, interleaved: bool = False):
    """fp32 cos / sin tables [seq, head_dim/2] holding exactly the values the
    reference multiplies by (rounded to ``dtype`` for the half-split form)."""
    key = (seq, head_dim, float(theta), dtype, device, interleaved)
    with _rope_lock:
        hit = _rope_cache.get(key)
    if hit is not None:
        return hit
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.int64).float() / head_dim))
    pos = torch.arange(seq, dtype=torch.int64).float()
    freqs = torch.outer(pos, inv_freq)  # fp32 on the host: deterministic tables
    cos, sin = freqs.cos(), freqs.sin()
    if not interleaved and dtype != torch.float32:
        cos, sin = cos.to(dtype).float(), sin.to(dtype).float()
    tab = (cos.contiguous().to(device), sin.contiguous().to(device))
    with _rope_lock:
        _rope_cache[key] = tab
    return tab


# ---------------------------------------------------------------- RMSNorm --

class RMSNormFunction(torch.autograd.Function):
    """y = w * round(x * rsqrt(mean(x^2) + eps)) -- HF LlamaRMSNorm.forward
    (imported at models/llama_simple.py:9)."""

    @staticmethod
    def forward(ctx, x, weight, eps):
        shape = x.shape
        x2 = x.contiguous().view(-1, shape[-1])
        y, rstd, _ = K.rmsnorm_fwd(x2, weight.contiguous(), eps)
        ctx.save_for_backward(x2, weight, rstd)
        out_dtype = torch.promote_types(x.dtype, weight.dtype)
        y = y.view(shape)
        return y if out_dtype == y.dtype else y.to(out_dtype)

    @staticmethod
    def backward(ctx, dy):
        x2, weight, rstd = ctx.saved_tensors
        dy2 = dy.to(x2.dtype).contiguous().view_as(x2)
        dx, dw = K.rmsnorm_bwd(dy2, x2, weight.contiguous(), rstd,
                               dw_dtype=weight.dtype)
        return dx.view(dy.shape), dw, None


def rms_norm(x, weight, eps=1e-6):
    return RMSNormFunction.apply(x, weight, eps)


# ----------------------------------------------------------------- SwiGLU --

class SwiGLUFunction(torch.autograd.Function):
    """z = silu(g) * u on [T, F] (HF LlamaMLP's activation, models/
    llama_simple.py:418)."""

    @staticmethod
    def forward(ctx, g, u):
        g2 = g.contiguous().view(-1, g.shape[-1])
        u2 = u.contiguous().view(-1, u.shape[-1])
        z = K.swiglu_fwd(g2, u2)
        ctx.save_for_backward(g2, u2)
        return z.view(g.shape)

    @staticmethod
    def backward(ctx, dz):
        g2, u2 = ctx.saved_tensors
        dz2 = dz.contiguous().view_as(g2)
        dg, du = torch.empty_like(g2), torch.empty_like(u2)
        K.swiglu_bwd(dz2, g2, u2, dg, du)
        return dg.view(dz.shape), du.view(dz.shape)


def swiglu(g, u):
    return SwiGLUFunction.apply(g, u)


# -------------------------------------------------------- Token embedding --

def embedding(ids, weight, *, scale=1.0, padding_idx=None, dtype=None):
    """Rows of a token table: scale * weight[ids] as [*ids.shape, hidden] in
    ``dtype`` (default the table's).  ids int32 / int64; an id outside
    [0, vocab) gives a row of NaN and no gradient (nothing is read back to the
    host to check it).  ``padding_idx`` (negative: from the end, as nn.Embedding
    takes it): the row whose tokens have no gradient.  Linear in the table: it can
    be differentiated twice, and forward-mode tangents go through it."""
    return nodes().embedding(ids, weight, scale, padding_idx, dtype)


# ----------------------------------------- Norm of q and k heads, rotation --

def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, *, positions=None, eps=1e-6,
                 interleaved=False):
    """(q', k') for attention without rope_theta: RMS norm of every head of q
    [B,S,Hq,d] and k [B,S,Hkv,d] over its d elements with the weights [d], then
    the rotation, in one pass with one rounding.  cos / sin: fp32 [n_pos, d/2]
    tables (rope_tables(..., torch.float32, ...)); ``positions`` int64 [S] or
    [B, S], default 0 .. S-1; a position outside the tables gives NaN.  Any even
    d up to 1024; q and k may be views of one q|k|v buffer.  It can be
    differentiated once, backward."""
    return nodes().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)


# -------------------------------------------------------------- Attention --

class FlashAttentionFunction(torch.autograd.Function):
    """Causal / sliding-window GQA attention with RoPE applied to Q and K
    first; [B, S, H, d] in and out.  The attention core replaces
    models/llama_simple.py:320-342 (and the FA2 / SDPA classes chosen at
    :376-416); RoPE replaces apply_rotary_pos_emb (:34-58)."""

    @staticmethod
    def forward(ctx, q, k, v, causal, window, scale, rope_theta, interleaved):
        B, S, Hq, d = q.shape
        if rope_theta is not None:
            cos, sin = rope_tables(S, d, rope_theta, q.dtype, q.device, interleaved)
            q, k = K.rope_copy(q, k, cos, sin, interleaved=interleaved)
        o, lse = K.attn_fwd(q, k, v, causal=causal, window=window, scale=scale)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.cfg = (causal, window, scale, rope_theta, interleaved)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        causal, window, scale, rope_theta, interleaved = ctx.cfg
        do = do.contiguous()
        if do.stride() != o.stride():
            do = do.view(o.shape)
        rope = None
        if rope_theta is not None:
            B, S, Hq, d = q.shape
            cos, sin = rope_tables(S, d, rope_theta, q.dtype, q.device, interleaved)
            rope = (cos, sin, None, interleaved)
        # with RoPE the kernels also apply the rotation's transpose to dq / dk
        dq, dk, dv = K.attn_bwd(q, k, v, o, do, lse, causal=causal, window=window,
                                scale=scale, rope=rope)
        return dq, dk, dv, None, None, None, None, None


def flash_attention(q, k, v, *, causal=True, window=0, scale=None, rope_theta=None,
                    interleaved=False):
    """Autograd entry: q [B,S,Hq,d], k / v [B,S,Hkv,d] (bf16 / fp16 / fp32)."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return FlashAttentionFunction.apply(q, k, v, bool(causal), int(window or 0),
                                        float(scale), rope_theta, bool(interleaved))


# ------------------------------------------- Packed sequences, their attention --

class PackedSequences:
    """Sequences that lie one after another in one run of ``tokens`` tokens:
    sequence s is the tokens offsets[s] .. offsets[s + 1] - 1.  It is made once
    a batch and serves every layer, forward and backward.

    ``offsets``: sequences + 1 ascending token counts from 0 on, int32 / int64.
    On the GPU they are not read back to the host to check them, and ``tokens``
    is needed; a list or a CPU tensor is checked, moved to ``device`` (default
    the current GPU) and gives ``tokens`` (default the last offset).  Tokens
    behind the last sequence are padding.

    ``plan`` holds the kernels' tables, ``positions`` (int64 [tokens]) every
    token's place in its sequence, for the rotations."""

    def __init__(self, offsets, tokens=None, *, device=None):
        offsets = self._offsets(offsets, tokens, device)
        if tokens is None:
            if self._last is None:
                raise ValueError("PackedSequences: tokens is needed for offsets on the GPU")
            tokens = self._last
        self.tokens = int(tokens)
        self.plan = torch.empty(K.packed_plan_words(self.tokens), device=offsets.device,
                                dtype=torch.int32)
        self.positions = torch.empty(self.tokens, device=offsets.device, dtype=torch.int64)
        self._make(offsets)

    def update(self, offsets) -> "PackedSequences":
        """Other sequences of the same run of tokens, in the same tables: what a
        captured graph that uses them replays with."""
        self._make(self._offsets(offsets, self.tokens, self.plan.device))
        torch.autograd.graph.increment_version((self.plan, self.positions))
        return self

    def _offsets(self, offsets, tokens, device):
        self._last = None
        if torch.is_tensor(offsets) and offsets.is_cuda:
            return offsets.contiguous()
        offsets = torch.as_tensor(offsets)
        if offsets.dim() != 1 or offsets.numel() == 0 or offsets.is_floating_point():
            raise ValueError("PackedSequences: offsets are [sequences + 1] integers")
        steps = offsets.tolist()
        if steps[0] != 0 or any(b < a for a, b in zip(steps, steps[1:])):
            raise ValueError("PackedSequences: offsets start at 0 and ascend")
        if tokens is not None and steps[-1] > tokens:
            raise ValueError(f"PackedSequences: the sequences have {steps[-1]} tokens, "
                             f"more than {tokens}")
        self._last = steps[-1]
        return offsets.to(device="cuda" if device is None else device, dtype=torch.int64)

    def _make(self, offsets) -> None:
        K.packed_plan(offsets, self.tokens, self.plan, self.positions)


def packed_attention(q, k, v, sequences, *, causal=True, window=0, scale=None):
    """Attention within each of the ``sequences`` (PackedSequences): q
    [tokens, Hq, d], k / v [tokens, Hkv, d], Hq a multiple of Hkv, d up to 128
    (even in bf16 / fp16) -> [tokens, Hq, d].  ``causal``: a token sees those up
    to itself, with ``window`` > 0 the last ``window`` of them; otherwise its
    whole sequence.  Padding rows of the result and of the gradients are zeros,
    and nothing of a token that a row does not see reaches it, be it infinite or
    NaN.  It can be differentiated once, backward; rotate q and k before
    (``sequences.positions``)."""
    return nodes().packed_attention(q, k, v, sequences.plan, causal, window or 0, scale)


# ------------------------------------------------ Rotation by several axes --

def rope_axes(q, k, cos, sin, positions, pair_axes, *, interleaved=False):
    """(q', k'): the rotation of q [tokens, Hq, d] and k [tokens, Hkv, d] (or
    [B, S, H, d]; k may be None) by positions of several axes.  ``positions``
    int64 [axes, tokens] (or [axes, B, S]); ``pair_axes``: the axis of each of
    the d/2 pairs (pair_axes_of); cos / sin: fp32 [n_pos, d/2] tables
    (rope_tables(..., torch.float32, ...)), pair i of a token turned by their row
    positions[pair_axes[i], token].  fp32 with one rounding; a position outside
    the tables gives NaN in its axis' pairs.  Any even d up to 512; q and k may
    be views of one q|k|v buffer.  Linear in q and k: it can be differentiated
    any number of times, backward."""
    return nodes().rope_axes(q, k, cos, sin, positions, bytes(pair_axes), interleaved)


def pair_axes_of(sections, *, turns=False):
    """The axis of each pair, for ``sections[a]`` pairs of axis a: one axis' pairs
    after another's, or, with ``turns``, the axes in turn as long as each has
    pairs left."""
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0 or len(sections) > 256:
        raise ValueError(f"pair_axes_of: numbers of pairs are needed (got {sections})")
    if not turns:
        return bytes(a for a, n in enumerate(sections) for _ in range(n))
    return bytes(a for i in range(max(sections)) for a, n in enumerate(sections) if i < n)

"""Fused AdamW on flat parameter shards and on lists of tensors.

Replaces ``torch.optim.Adam(fused=True)`` as the reference builds it for each
FSDP module's flat shard (zorse_utils/pipeline.py:150-181) and steps it from
the reduce-grad callback (utils/patch.py:76-154).  The grad cast of
utils/patch.py:115-119 (reduce dtype -> fp32) is folded into the kernel: the
gradient is read in whatever float dtype it has.

Mixed precision: when a parameter is bf16 / fp16 (the compute copy the layer
runs on), the optimizer keeps an fp32 master copy in its state, updates the
master, m and v, and writes the rounded parameter back -- all in the same
pass.  With an fp32 parameter the update is in place.

``step()`` steps all of a group's parameters on a GPU in one launch (for every
56), ``step_param`` one of them.  ``state_bits=8`` holds both moments in 8 bits
a value (kernels.adamw8_multi): 2 bytes an element of state beside the master
where 32 bits take 8.  ``seed`` sets the random bits of their rounding apart
from those of other optimizers (a model with one for each layer); it is one of
the groups' options and saved with them.

``weight_decay`` is decoupled (AdamW); ``FusedAdam`` is the same optimizer
with weight decay fixed at 0, which is exactly ``torch.optim.Adam`` with its
defaults -- the reference's optimizer.
"""
from __future__ import annotations

import itertools
import operator

import torch

from . import kernels as K


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 state_bits=32, seed=0):
        if lr < 0 or eps < 0 or weight_decay < 0:
            raise ValueError("lr, eps and weight_decay must be non-negative")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"invalid betas {betas}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32 (got {state_bits})")
        self.state_bits = state_bits
        random = {"seed": operator.index(seed)} if state_bits == 8 else {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, **random))
        self._step_hooks = {}   # param -> [callable(param)]

    def add_step_hook(self, p: torch.Tensor, fn) -> None:
        """``fn(p)`` runs after every step of ``p`` (after its version bump)."""
        self._step_hooks.setdefault(p, []).append(fn)

    def _init_state(self, p: torch.Tensor) -> dict:
        st = self.state[p]
        if not st:
            n, kw = p.numel(), {"device": p.device}
            st["step"] = 0
            moment = torch.uint8 if self.state_bits == 8 else torch.float32
            st["exp_avg"] = torch.zeros(n, dtype=moment, **kw)
            st["exp_avg_sq"] = torch.zeros(n, dtype=moment, **kw)
            if self.state_bits == 8:
                st["exp_base"] = torch.zeros(-(-n // K.ADAMW8_BLOCK), 2, dtype=torch.int16, **kw)
            if p.dtype != torch.float32:
                st["master"] = p.detach().reshape(-1).to(torch.float32)
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is not None:
                    by_device.setdefault(p.device, []).append(p)
            for dev, params in by_device.items():
                if dev.type == "cuda":
                    self._step_list(group, params)
                else:
                    for p in params:
                        self._step_one(group, p)
        return loss

    @torch.no_grad()
    def step_param(self, p: torch.Tensor) -> None:
        """Step ``p`` alone (the other parameters of this optimizer are left
        as they are, whatever their gradients): the per-parameter step of an
        optimizer-in-backward hook, which fires once per parameter as its
        gradient completes.  No-op when ``p.grad`` is None."""
        for group in self.param_groups:
            for q in group["params"]:
                if q is p:
                    if p.grad is not None:
                        self._step_one(group, p)
                    return
        raise ValueError("step_param: the tensor is not a parameter of this optimizer")

    def _checked(self, p: torch.Tensor) -> dict:
        """p's state, on p's device, after the checks of p and its gradient."""
        if p.grad.is_sparse:
            raise RuntimeError("FusedAdamW does not support sparse gradients")
        if not p.is_contiguous() or not p.grad.is_contiguous():
            raise ValueError("FusedAdamW needs contiguous parameters and gradients")
        st = self._init_state(p)
        if st["exp_avg"].device != p.device:
            for k in ("exp_avg", "exp_avg_sq", "exp_base", "master"):
                if k in st:
                    st[k] = st[k].to(p.device)
        return st

    def _stepped(self, p: torch.Tensor) -> None:
        # the kernel wrote p through a raw pointer: advance its version
        # counter as an in-place torch op would, so caches keyed on it
        # (compute-dtype weight copies, attention caches) see the update
        torch.autograd.graph.increment_version(p)
        for fn in self._step_hooks.get(p, ()):
            fn(p)

    @staticmethod
    def _hyper(group: dict) -> dict:
        b1, b2 = group["betas"]
        return dict(lr=group["lr"], beta1=b1, beta2=b2, eps=group["eps"],
                    weight_decay=group["weight_decay"])

    def _seeds(self, group: dict, params: list, steps: list) -> list:
        """Of the random bits of each second moment at its step: from the group's
        seed (0 in checkpoints without one), the parameter's place in the
        optimizer and the step, so that a resumed run repeats them."""
        place = {id(p): i for i, p in enumerate(itertools.chain.from_iterable(
            g["params"] for g in self.param_groups))}
        own = group.get("seed", 0) * 0x165667B1
        counts = {t: int(t) * 0xC2B2AE3D + own for t in set(steps)}
        return [(counts[t] + place[id(p)] * 0x27D4EB2F) & 0xFFFFFFFF
                for p, t in zip(params, steps)]

    def _step_one(self, group: dict, p: torch.Tensor) -> None:
        if self.state_bits == 8:
            self._step_list(group, [p])
            return
        st = self._checked(p)
        st["step"] += 1
        master = st.get("master")
        K.adamw_step(master if master is not None else p.view(-1),
                     p.grad.view(-1), st["exp_avg"], st["exp_avg_sq"],
                     lowp_out=p.view(-1) if master is not None else None,
                     step=st["step"], **self._hyper(group))
        self._stepped(p)

    def _step_list(self, group: dict, params: list) -> None:
        # one parameter, or parameters that share memory: one by one
        shared = len(params) > 1 and K.spans_meet(
            [p.data_ptr() for p in params], [p.nbytes for p in params], 1)
        if (len(params) == 1 or shared) and self.state_bits == 32:
            for p in params:
                self._step_one(group, p)
            return
        if shared:
            for p in params:
                self._step_list(group, [p])
            return
        states = [self._checked(p) for p in params]
        masters = [st.get("master") for st in states]
        args = ([p if m is None else m for p, m in zip(params, masters)],
                [p.grad for p in params], [st["exp_avg"] for st in states],
                [st["exp_avg_sq"] for st in states])
        steps = [st["step"] + 1 for st in states]
        lows = [None if m is None else p for p, m in zip(params, masters)]
        if self.state_bits == 8:
            K.adamw8_multi(*args, [st["exp_base"] for st in states], steps, lowp_outs=lows,
                           seeds=self._seeds(group, params, steps), **self._hyper(group))
        else:
            K.adamw_multi(*args, steps, lowp_outs=lows, **self._hyper(group))
        for st, t in zip(states, steps):  # a refused list has not been stepped
            st["step"] = t
        for p in params:
            self._stepped(p)

    def load_state_dict(self, state_dict) -> None:
        """As torch.optim.Optimizer's, but a state tensor's type does not follow
        the parameter's: masters and 32-bit moments are fp32 whatever type they
        were saved in, 8-bit codes and others keep their own."""
        # between the caller's hooks: what those before the load leave is loaded,
        # and those after it find the state as it stays
        saved = {}
        before = self.register_load_state_dict_pre_hook(
            lambda _, sd: self._check_loaded(sd, saved))
        after = self.register_load_state_dict_post_hook(
            lambda _: self._keep_types(saved), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            before.remove()
            after.remove()

    def _check_loaded(self, state_dict, saved: dict) -> None:
        for st in state_dict["state"].values():
            if "exp_avg" not in st:
                continue
            dt = st["exp_avg"].dtype
            if not (dt == torch.uint8 if self.state_bits == 8 else dt.is_floating_point):
                raise ValueError(f"the saved moments are {dt}, not those of "
                                 f"state_bits={self.state_bits}")
        saved.update(state_dict)

    def _keep_types(self, saved: dict) -> None:
        keys = itertools.chain.from_iterable(g["params"] for g in saved["param_groups"])
        params = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for key, p in zip(keys, params):
            for name, t in saved["state"].get(key, {}).items():
                if torch.is_tensor(t) and name != "step":
                    held = name in ("exp_avg", "exp_avg_sq", "master") and t.is_floating_point()
                    self.state[p][name] = t.detach().to(
                        device=p.device, dtype=torch.float32 if held else t.dtype, copy=True)

    def master_param(self, p: torch.Tensor) -> torch.Tensor:
        """fp32 master of ``p`` (``p`` itself when it is fp32)."""
        st = self._init_state(p)
        return st.get("master", p.view(-1))

    def moments(self, p: torch.Tensor):
        """(exp_avg, exp_avg_sq) of ``p`` as fp32 values [numel] (of 8-bit
        states: new tensors with the values that the codes stand for)."""
        st = self._init_state(p)
        if self.state_bits == 32:
            return st["exp_avg"], st["exp_avg_sq"]
        m, v = K.adamw8_values([st["exp_avg"]], [st["exp_avg_sq"]], [st["exp_base"]])
        return m[0], v[0]


class FusedAdam(FusedAdamW):
    """torch.optim.Adam's defaults (lr 1e-3, betas (0.9, 0.999), eps 1e-8,
    no weight decay) -- the optimizer the reference builds per flat shard."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0,
                 state_bits=32, seed=0):
        if weight_decay != 0:
            raise ValueError("FusedAdam applies no weight decay; use FusedAdamW for "
                             "decoupled weight decay")
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=0.0,
                         state_bits=state_bits, seed=seed)

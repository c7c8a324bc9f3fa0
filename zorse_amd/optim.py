"""Fused AdamW on flat parameter shards and on lists of tensors, and Muon.

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

    _HELD = ("exp_avg", "exp_avg_sq", "master")  # in fp32, whatever they were saved in

    def _keep_types(self, saved: dict) -> None:
        keys = itertools.chain.from_iterable(g["params"] for g in saved["param_groups"])
        params = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for key, p in zip(keys, params):
            for name, t in saved["state"].get(key, {}).items():
                if torch.is_tensor(t) and name != "step":
                    held = name in self._HELD and t.is_floating_point()
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


def flat_matrices(module) -> list:
    """The matrices of a decoder layer's (or a Block's) flat parameter, as Muon's
    ``matrices``: (offset, rows, cols) of its projections (the norms' weights are
    none)."""
    specs = [m.spec for m in module.modules() if hasattr(m, "flat_param")]
    if len(specs) != 1:
        raise ValueError(f"flat_matrices: a module with one flat parameter is needed (got {len(specs)})")
    shapes = specs[0].shapes()
    return [(a, *shapes[k]) for k, (a, _) in specs[0].offsets().items() if len(shapes[k]) == 2]


class Muon(FusedAdamW):
    """Matrices stepped by the orthogonal factor of their momentum
    (kernels.muon_multi), all of a group's in the same launches; everything else
    by AdamW.

    A group's ``matrices``: None, every 2-D parameter is a matrix; or a list of
    (offset, rows, cols) that each of its parameters holds in its elements
    (flat_matrices(layer) for a decoder layer's flat parameter; [] for none, as
    for embeddings and heads).  What lies in none of them (norm weights, biases)
    takes AdamW's step with ``adam_lr`` (default lr), ``adam_betas`` and
    ``adam_eps``, with the same weight decay.

    ``adjust``: "original" multiplies a factor by sqrt(max(1, rows / cols)),
    "match_rms_adamw" by 0.2 sqrt(max(rows, cols)), so that one learning rate
    suits both steps.  bf16 / fp16 parameters keep an fp32 master."""

    def __init__(self, params, lr=1e-3, momentum=0.95, weight_decay=0.1, nesterov=True, ns_steps=5,
                 ns_coefficients=K.MUON_COEFFICIENTS, eps=1e-7, adjust="original", matrices=None,
                 adam_lr=None, adam_betas=(0.9, 0.999), adam_eps=1e-8):
        if lr < 0 or eps < 0 or weight_decay < 0 or adam_eps < 0 or (adam_lr or 0) < 0:
            raise ValueError("lr, eps and weight_decay must be non-negative")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"invalid momentum {momentum}")
        if not (0.0 <= adam_betas[0] < 1.0 and 0.0 <= adam_betas[1] < 1.0):
            raise ValueError(f"invalid betas {adam_betas}")
        if adjust not in ("original", "match_rms_adamw"):
            raise ValueError(f"adjust is 'original' or 'match_rms_adamw' (got {adjust!r})")
        self.state_bits = 32
        torch.optim.Optimizer.__init__(self, params, dict(
            lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov,
            ns_steps=operator.index(ns_steps), ns_coefficients=tuple(ns_coefficients), eps=eps,
            adjust=adjust, matrices=matrices, adam_lr=adam_lr, adam_betas=tuple(adam_betas),
            adam_eps=adam_eps))
        self._step_hooks = {}

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            for p in group["params"]:
                self._layout(group, p)
        except ValueError:
            self.param_groups.pop()
            raise

    @staticmethod
    def _layout(group: dict, p: torch.Tensor):
        """(matrices, rest) of p: (offset, rows, cols) and (offset, elements)."""
        n = p.numel()
        if group["matrices"] is None:
            mats = [(0, *p.shape)] if p.dim() == 2 else []
        else:
            mats = sorted((int(a), int(r), int(c)) for a, r, c in group["matrices"])
        mats = [m for m in mats if m[1] * m[2] != 0]
        rest, at = [], 0
        for a, r, c in mats:
            if a < at or min(r, c) < 0 or a + r * c > n:
                raise ValueError(f"matrices of a parameter of {n} elements overlap or leave it: "
                                 f"{r} x {c} at {a}")
            if a > at:
                rest.append((at, a - at))
            at = a + r * c
        if at < n:
            rest.append((at, n - at))
        return mats, rest

    def _init_state(self, p: torch.Tensor) -> dict:
        st = self.state[p]
        if not st:
            group = next(g for g in self.param_groups if any(q is p for q in g["params"]))
            mats, rest = self._layout(group, p)
            kw = {"dtype": torch.float32, "device": p.device}
            st["step"] = 0
            st["momentum_buffer"] = torch.zeros(sum(r * c for _, r, c in mats), **kw)
            if rest:
                n = sum(k for _, k in rest)
                st["exp_avg"], st["exp_avg_sq"] = torch.zeros(n, **kw), torch.zeros(n, **kw)
            if p.dtype != torch.float32:
                st["master"] = p.detach().reshape(-1).to(torch.float32)
        return st

    def _checked(self, p: torch.Tensor) -> dict:
        if p.grad.is_sparse:
            raise RuntimeError("Muon does not support sparse gradients")
        if not p.is_contiguous() or not p.grad.is_contiguous():
            raise ValueError("Muon needs contiguous parameters and gradients")
        st = self._init_state(p)
        if st["momentum_buffer"].device != p.device:
            for k, t in st.items():
                if torch.is_tensor(t) and k != "step":
                    st[k] = t.to(p.device)
        return st

    @staticmethod
    def _check_sizes(where: list, p: torch.Tensor, st: dict) -> None:
        """A loaded state may be of other matrices or another parameter."""
        n = sum(r * c for _, r, c in where)
        for name, want in (("momentum_buffer", n), ("exp_avg", p.numel() - n), ("exp_avg_sq", p.numel() - n)):
            if (st[name].numel() if name in st else 0) != want:
                raise ValueError(f"Muon: a state's {name} does not have its parameter's {want} elements")
        if "master" in st and st["master"].numel() != p.numel():
            raise ValueError(f"Muon: a state's master does not have its parameter's {p.numel()} elements")

    def _step_one(self, group: dict, p: torch.Tensor) -> None:
        self._step_list(group, [p])

    def _step_list(self, group: dict, params: list) -> None:
        if len(params) > 1 and K.spans_meet([p.data_ptr() for p in params],
                                            [p.nbytes for p in params], 1):
            for p in params:
                self._step_list(group, [p])
            return
        states = [self._checked(p) for p in params]
        mats = ([], [], [], [])   # params, grads, momenta, rounded copies
        rest = ([], [], [], [], [])  # params, grads, moments, rounded copies
        steps = []
        for p, st in zip(params, states):
            master, grad, low = st.get("master"), p.grad.view(-1), None
            flat = p.detach().view(-1)
            if master is not None:
                flat, low = master, flat
            where, others = self._layout(group, p)
            self._check_sizes(where, p, st)
            at = 0
            for a, r, c in where:
                cut = slice(a, a + r * c)
                mats[0].append(flat[cut].view(r, c))
                mats[1].append(grad[cut].view(r, c))
                mats[2].append(st["momentum_buffer"][at:at + r * c].view(r, c))
                mats[3].append(None if low is None else low[cut].view(r, c))
                at += r * c
            at = 0
            for a, n in others:
                rest[0].append(flat[a:a + n])
                rest[1].append(grad[a:a + n])
                rest[2].append(st["exp_avg"][at:at + n])
                rest[3].append(st["exp_avg_sq"][at:at + n])
                rest[4].append(None if low is None else low[a:a + n])
                steps.append(st["step"] + 1)
                at += n
        # a refused list has not been stepped: both are checked before either is
        muon = None
        if mats[0]:
            muon = K.muon_step(*mats[:3], lowp_outs=mats[3], lr=group["lr"], momentum=group["momentum"],
                               weight_decay=group["weight_decay"], nesterov=group["nesterov"],
                               adjust=group["adjust"], steps=group["ns_steps"],
                               coefficients=group["ns_coefficients"], eps=group["eps"])
        if rest[0]:
            lr = group["lr"] if group["adam_lr"] is None else group["adam_lr"]
            b1, b2 = group["adam_betas"]
            K.adamw_multi(*rest[:4], steps, lowp_outs=rest[4], lr=lr, beta1=b1, beta2=b2,
                          eps=group["adam_eps"], weight_decay=group["weight_decay"])
        if muon is not None:
            muon.run()
        for st in states:
            st["step"] = st["step"] + 1
        for p in params:
            self._stepped(p)

    def _check_loaded(self, state_dict, saved: dict) -> None:
        for st in state_dict["state"].values():
            if "momentum_buffer" not in st:
                raise ValueError("the saved state is not Muon's")
        saved.update(state_dict)

    _HELD = ("momentum_buffer", "exp_avg", "exp_avg_sq", "master")

    def moments(self, p: torch.Tensor):
        """The momentum of p's matrices, fp32, one matrix after another."""
        return self._init_state(p)["momentum_buffer"]

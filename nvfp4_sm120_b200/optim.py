"""AdamW over all parameters of a model in one launch (csrc/adamw.cu), with moments in 32 bits or in 8, and the norm of
the gradients that clips them.

The reference steps torch.optim.AdamW after clip_grad_norm_ (nvfp4_train.py:159-185): a pass that reads the gradients, one
that scales them in place and one that reads them again, and 8 bytes of moments for each parameter.  Here the scaling
is part of the step, and the moments take 8 bytes or 2."""
from __future__ import annotations

import torch

from . import _lib

BLOCK = 256            # elements of a moment tensor that share a scale when it is held in 8 bits
_M64 = 2 ** 64 - 1
_NAMES = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale")}


def _dtype8(name):
    return torch.float8_e8m0fnu if name.endswith("_scale") else torch.float8_e4m3fn


def _same_order(strides, p):
    """Are `strides` those of `p`, where they matter?  (Those of sizes of 1 do not.)"""
    return len(strides) == p.dim() and all(n == 1 or a == b for a, b, n in zip(strides, p.stride(), p.shape))


def grad_norm(params):
    """2-norm of the gradients of `params` (an iterable of tensors; those without a gradient are skipped) as an fp32
    0-dim CUDA tensor, summed in 64 bits and in a fixed order.  No host synchronisation."""
    params = [params] if isinstance(params, torch.Tensor) else list(params)
    norm = _lib.host().grad_norm(params)
    if norm is None:
        return torch.zeros((), dtype=torch.float32, device=params[0].device if params else "cuda")
    return norm


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update for fp32 and bf16 parameters on one GPU, in fp32 arithmetic.

    state_bits: 32 keeps `exp_avg` and `exp_avg_sq` in fp32 (also for bf16 parameters), under torch's names, and loads
        the state_dict of a torch.optim.AdamW.  8 keeps the first moment and the ROOT of the second as E4M3 codes
        with one power of two per 256 elements (`exp_avg`, `exp_avg_scale`, `exp_avg_root`, `exp_avg_root_scale`; value =
        code * scale, elements in memory order, whose strides `layout` keeps), rounded stochastically.  A block that
        holds an infinity, a NaN or a magnitude of 2^51 or more is NaN as a whole from then on.
    max_norm: clip the gradients to this norm over ALL parameter groups, as clip_grad_norm_ in front of the step would,
        but inside it: `p.grad` itself is left as it is.  The norm of the last step is in `grad_norm` (0-dim, on the
        device).  step(grad_norm=...) takes a norm found elsewhere instead, e.g. one that counts shards on other ranks.
    seed: of the stochastic rounding; the bits of an element follow from (seed, its place among the parameters, its step
        count), so replicas that are given the same gradients stay the same and a resumed run goes on as it would have.

    The step count lives on the host, so a step cannot be captured into a CUDA graph; it raises there."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_norm=None,
                 seed=0):
        if not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not eps >= 0.0:
            raise ValueError(f"eps must not be negative, got {eps}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if not weight_decay >= 0.0:
            raise ValueError(f"weight_decay must not be negative, got {weight_decay}")
        if state_bits not in _NAMES:
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError(f"max_norm must be positive or None, got {max_norm}")
        self.state_bits, self.max_norm, self.seed, self.grad_norm, self._flat = state_bits, max_norm, int(seed), None, []
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        if len(set(params)) != len(params):                # the step takes all of them at the same time
            self.param_groups.pop()
            raise ValueError("a parameter stands twice in its group")

    def __getstate__(self):
        mine = {k: getattr(self, k) for k in ("state_bits", "max_norm", "seed", "grad_norm", "_flat")}
        return {**super().__getstate__(), **mine}

    # ---- state ----
    def _make_state(self, params):
        """Zeros for `params` in one buffer per moment; a tensor's part begins at a multiple of BLOCK elements."""
        if not params:
            return
        _lib.cuda_device_of(*params)
        blocks = [-(-p.numel() // BLOCK) for p in params]
        total, dev = sum(blocks) * BLOCK, params[0].device
        if self.state_bits == 32:
            flat = {name: torch.zeros(total, dtype=torch.float32, device=dev) for name in _NAMES[32]}
        else:
            flat = {}
            for name in _NAMES[8]:
                n = total // BLOCK if name.endswith("_scale") else total
                flat[name] = torch.zeros(n, dtype=torch.uint8, device=dev).view(_dtype8(name))
        self._flat.append(flat)
        parts = {name: buf.split(blocks if name.endswith("_scale") else [b * BLOCK for b in blocks]) for name, buf in flat.items()}
        for i, p in enumerate(params):
            if self.state_bits == 32:
                st = {name: t[i].as_strided(p.shape, p.stride()) for name, t in parts.items()}
            else:                                      # (the codes follow the parameter's memory, which must not be reordered)
                st = {**{name: t[i] for name, t in parts.items()}, "layout": tuple(p.stride())}
            self.state[p] = {"step": 0, **st}

    def flat_state(self):
        """The buffers that the moments are views into, in the order they were made: one dict per parameter group, and one
        more for parameters that got their first gradient later."""
        return [dict(flat) for flat in self._flat]

    def load_state_dict(self, state_dict):
        """The state of this class (same state_bits), or of a torch.optim.AdamW when state_bits is 32."""
        pairs = []                                         # (saved state, its parameter) by group

        def take(_, state_dict):                           # behind the other pre-hooks, which may change what is loaded
            pairs.extend(self._saved_pairs(state_dict))
            return {**state_dict, "state": {}}             # (torch would cast the moments to the parameters' dtype)

        def place(_):                                      # in front of the other post-hooks, which look at the loaded state
            self._place(pairs)

        hooks = (self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(place, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _saved_pairs(self, state_dict):
        groups = state_dict["param_groups"]
        for g in groups:
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("amsgrad and maximize are not supported")
            if g["weight_decay"] and not g.get("decoupled_weight_decay", True):
                raise ValueError("the saved state is that of an optimizer whose weight decay is part of the gradient")
        saved = {i: st for i, st in state_dict["state"].items() if st}          # (empty: looked up before its first step)
        names = _NAMES[self.state_bits]
        for i, st in saved.items():
            if any(n not in st for n in ("step", *names)):
                raise ValueError(f"the saved state of parameter {i} is not that of {self.state_bits}-bit moments")
        pairs = [[(saved[i], p) for i, p in zip(old["params"], new["params"]) if i in saved]
                 for old, new in zip(groups, self.param_groups)]
        if any(pairs):
            _lib.cuda_device_of(*(p for group in pairs for _, p in group))
        for st, p in (pair for group in pairs for pair in group):
            if "layout" in st and not _same_order(st["layout"], p):
                raise ValueError(f"the saved moments are in the order of strides {tuple(st['layout'])}, not {p.stride()}")
            blocks = -(-p.numel() // BLOCK)
            for n in names:
                fits = p.numel() if self.state_bits == 32 else blocks if n.endswith("_scale") else blocks * BLOCK
                if st[n].numel() != fits or (self.state_bits == 8 and st[n].dtype != _dtype8(n)):
                    raise ValueError(f"the saved {n} does not fit a parameter of shape {tuple(p.shape)}")
        return pairs

    def _place(self, pairs):
        names = _NAMES[self.state_bits]
        self._flat = []
        to, source = [], []
        for group in pairs:
            self._make_state([p for _, p in group])
            for st, p in group:
                mine = self.state[p]
                mine["step"] = int(st["step"])
                for n in names:
                    eight = self.state_bits == 8
                    to.append(mine[n].view(torch.uint8) if eight else mine[n])
                    source.append(st[n].view(torch.uint8) if eight else st[n].view(p.shape) if st[n].shape != p.shape else st[n])
        if to:
            torch._foreach_copy_(to, source)

    # ---- step ----
    def step(self, closure=None, *, grad_norm=None):
        """One step of every parameter that has a gradient.  grad_norm: one fp32 element on the parameters' device to
        clip by, in place of the norm found here."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if grad_norm is not None and self.max_norm is None:
            raise ValueError("grad_norm is what max_norm clips by: the optimizer was made without max_norm")
        call = lambda: _lib.host().adamw_step(self.param_groups, self.state, self.state_bits, self.max_norm,
                                              self.seed & _M64, grad_norm)
        done = call()
        if isinstance(done, str) and done == "state":
            for g in self.param_groups:
                self._make_state([p for p in g["params"]
                                  if not self.state.get(p) and p.numel() and (p.requires_grad or p.grad is not None)])
            done = call()
        if isinstance(done, str):
            raise _lib.NVFP4Error("AdamW.step cannot be captured into a CUDA graph: its step count lives on the host")
        self.grad_norm = done if isinstance(done, torch.Tensor) else None
        return loss

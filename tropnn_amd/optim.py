"""Adam / AdamW whose update runs as one HIP launch over all parameters.

The reference trains its classifiers with torch.optim.AdamW(weight_decay=0)
(examples/emnist.py:310). FusedAdam is a drop-in torch.optim.Optimizer for
that role: the same update as torch's Adam (non-amsgrad, op order of its
single-tensor path), the same per-parameter state ("step", "exp_avg",
"exp_avg_sq", so state dicts move between the two in both directions),
computed by tropnn_hip_adam_step in libtropnn_hip.so. The step counters live
on the device, so a training step captured in a HIP graph replays with the
current count; lr and the other hyperparameters are read when step() runs (a
captured graph keeps the values it was captured with).

The kernel writes the tensors through raw device pointers, so step() bumps
the autograd version counter of every tensor it updates, as torch's in-place
optimizers do: caches keyed by a parameter's version (PairwiseLinear's f16
LUT copy, the lazy route-debug guard) see the update. A replayed HIP graph
runs no Python and bumps nothing; PairwiseLinear re-casts its f16 copy inside
a captured forward for that reason.

With state_bits=8 both moments are held in 8 bits and a parameter's state is 2
bytes and two sixteenths of a byte instead of 8 (tropnn_hip_adam8_step in
include/tropnn_hip_train.h has the arithmetic): e4m3 numbers with a power of two
for every 32 consecutive elements, of exp_avg and of exp_avg_sq's root, rounded
at random so that their expected value is the one that 32 bits would hold. The
random numbers are a hash of the element's index and the step, so a run repeats
bit for bit.

Only dense f32 parameters on a GPU are supported; anything else raises (there
is no CPU fallback).
"""
from __future__ import annotations

import ctypes
from collections import defaultdict
from contextlib import nullcontext

import torch

from .backends.pairwise_hip import _check, _stream, load_library
from .backends.train_hip import STATE_BLOCK, train_ops


def adam_step_hip(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr: float, beta1: float, beta2: float,
                  eps: float, weight_decay: float, decoupled_weight_decay: bool) -> None:
    """One Adam / AdamW update of equal-length lists of contiguous f32 tensors
    on one GPU (steps: 0-dim f32 tensors, one per parameter), on the current
    stream of that GPU."""
    n = len(params)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == len(steps) == n):
        raise ValueError("params, grads, exp_avgs, exp_avg_sqs and steps must have equal lengths")
    if n == 0:
        return
    dev = params[0].device
    for name, ts in (("params", params), ("grads", grads), ("exp_avgs", exp_avgs), ("exp_avg_sqs", exp_avg_sqs),
                     ("steps", steps)):
        for k, t in enumerate(ts):
            if t.device != dev or t.device.type != "cuda":
                raise ValueError(f"{name}[{k}] is on {t.device}, expected {dev} (a GPU)")
            if t.dtype != torch.float32:
                raise TypeError(f"{name}[{k}] has dtype {t.dtype}, expected torch.float32")
            if not t.is_contiguous():
                raise ValueError(f"{name}[{k}] is not contiguous")
    for k in range(n):
        numel = params[k].numel()
        if grads[k].numel() != numel or exp_avgs[k].numel() != numel or exp_avg_sqs[k].numel() != numel:
            raise ValueError(f"tensor {k}: grad / exp_avg / exp_avg_sq sizes differ from the parameter's {numel}")
        if steps[k].numel() != 1:
            raise ValueError(f"steps[{k}] must hold one element")
    ptrs = ctypes.c_void_p * n
    lib = load_library()
    rc = lib.tropnn_hip_adam_step(
        n,
        ptrs(*[t.data_ptr() for t in params]),
        ptrs(*[t.data_ptr() for t in grads]),
        ptrs(*[t.data_ptr() for t in exp_avgs]),
        ptrs(*[t.data_ptr() for t in exp_avg_sqs]),
        (ctypes.c_int64 * n)(*[t.numel() for t in params]),
        ptrs(*[t.data_ptr() for t in steps]),
        float(lr), float(beta1), float(beta2), float(eps), float(weight_decay), int(bool(decoupled_weight_decay)),
        _stream(dev),
    )
    _check(rc, "tropnn_hip_adam_step")
    # the launch wrote these through raw pointers: tell autograd and the
    # version-keyed caches, as an in-place torch op would
    torch.autograd.graph.increment_version(params + exp_avgs + exp_avg_sqs + steps)


def adam8_step_hip(params, grads, exp_avgs, exp_avg_exponents, roots, root_exponents, steps, *, lr: float, beta1: float,
                   beta2: float, eps: float, weight_decay: float, decoupled_weight_decay: bool) -> None:
    """One Adam / AdamW update of equal-length lists of contiguous tensors on one
    GPU whose states are held in 8 bits, on the current stream of that GPU:
    params and grads f32, exp_avgs and roots as many float8_e4m3fn (or their
    bytes), exponents uint8, one for every 32 elements, steps 0-dim f32 tensors."""
    train_ops().adam8.default(params, grads, exp_avgs, exp_avg_exponents, roots, root_exponents, steps, float(lr), float(beta1),
                      float(beta2), float(eps), float(weight_decay), bool(decoupled_weight_decay))


# A parameter's state with 8 bits, beside "step": the codes in the parameter's
# shape and the exponent bytes of its blocks, for exp_avg and for the root of
# exp_avg_sq. The names differ from torch's, whose loaders would take codes for
# values.
_CODES = ("exp_avg_8bit", "root_8bit")
_EXPONENTS = ("exp_avg_exponents", "root_exponents")
_STATE_KEYS = {32: ("exp_avg", "exp_avg_sq", "step"),
               8: ("exp_avg_8bit", "exp_avg_exponents", "root_8bit", "root_exponents", "step")}
_STATE_TYPES = {"exp_avg_8bit": torch.float8_e4m3fn, "root_8bit": torch.float8_e4m3fn,
                "exp_avg_exponents": torch.uint8, "root_exponents": torch.uint8}


class _Kept:
    """A tensor that torch's loader passes on as it is."""

    def __init__(self, tensor: torch.Tensor) -> None:
        self.tensor = tensor


def _keep_codes(_: torch.optim.Optimizer, state_dict: dict) -> dict:
    def kept(state):
        if not isinstance(state, dict):
            return state
        return {k: _Kept(v) if k in _STATE_TYPES and isinstance(v, torch.Tensor) else v for k, v in state.items()}

    return {**state_dict, "state": {k: kept(state) for k, state in state_dict["state"].items()}}


def _give_codes(optimizer: torch.optim.Optimizer) -> None:
    for p, state in optimizer.state.items():
        for key, dtype in _STATE_TYPES.items():
            if isinstance(state, dict) and isinstance(state.get(key), _Kept):
                t = state[key].tensor.detach()
                state[key] = t.to(device=p.device if isinstance(p, torch.Tensor) else t.device, dtype=dtype, copy=True)


class FusedAdam(torch.optim.Optimizer):
    """torch.optim.Adam's update (amsgrad=False, maximize=False) on the GPU in
    one launch per parameter group and device. decoupled_weight_decay=True
    gives AdamW.

    state_bits: 32 (default; torch's state, which moves between the two), or 8:
    "exp_avg_8bit" and "root_8bit" (float8_e4m3fn, the parameter's shape) with
    "exp_avg_exponents" and "root_exponents" (uint8, one for every 32 elements in
    memory order; an element's value is its code times 2^(exponent - 127), and
    the root is that of exp_avg_sq). A root past f32 (of a gradient from 1.85e19 on)
    is NaN and stands for infinity: its element takes no more steps, as with 32 bits.
    A group of a loaded state dict has the state_bits that it was saved with."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, decoupled_weight_decay: bool = False, *, amsgrad: bool = False,
                 maximize: bool = False, state_bits: int = 32) -> None:
        if isinstance(lr, torch.Tensor):
            raise TypeError("FusedAdam takes lr as a float")
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 0: {betas[0]}")
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 1: {betas[1]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if amsgrad or maximize:
            raise NotImplementedError("FusedAdam supports amsgrad=False and maximize=False only")
        if state_bits not in _STATE_KEYS:
            raise ValueError(f"FusedAdam needs state_bits of 8 or 32, got {state_bits!r}")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                        decoupled_weight_decay=decoupled_weight_decay, state_bits=state_bits)
        super().__init__(params, defaults)

    def load_state_dict(self, state_dict) -> None:
        """torch's loader leaves "step" where it was saved unless the group is
        capturable or fused (Optimizer._process_value_according_to_param_policy),
        e.g. on the CPU for a torch.optim.Adam state dict or a checkpoint
        loaded with map_location="cpu"; the kernel reads it from the
        parameter's device as f32. It also casts all other state to the
        parameter's type, four times the bytes of codes and exponents: those are
        kept from it and copied as they are. A group saved without state_bits has
        32."""
        hooks = (self.register_load_state_dict_pre_hook(_keep_codes),
                 self.register_load_state_dict_post_hook(_give_codes, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
        for group in self.param_groups:
            group.setdefault("state_bits", 32)
        for p, state in self.state.items():
            step = state.get("step")
            if step is None:
                continue
            if not isinstance(step, torch.Tensor):
                step = torch.tensor(float(step))
            if step.device != p.device or step.dtype != torch.float32 or step.dim() != 0:
                state["step"] = step.detach().reshape(()).to(device=p.device, dtype=torch.float32)

    @staticmethod
    def _new_state(p: torch.Tensor, bits: int) -> dict[str, torch.Tensor]:
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        if bits == 32:
            state["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            return state
        blocks = -(-p.numel() // STATE_BLOCK)
        for codes, exponents in zip(_CODES, _EXPONENTS):
            state[codes] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
            state[exponents] = torch.zeros(blocks, dtype=torch.uint8, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            if group.get("amsgrad") or group.get("maximize"):
                # a loaded torch.optim.Adam state dict can carry these flags
                raise NotImplementedError("FusedAdam supports amsgrad=False and maximize=False only")
            bits = group.get("state_bits", 32)  # optimizers pickled before the option
            if bits not in _STATE_KEYS:
                raise ValueError(f"FusedAdam needs state_bits of 8 or 32, got {bits!r}")
            pairs = [(p, g) for p in group["params"] if (g := p.grad) is not None]
            if not pairs:
                continue
            params, grads = map(list, zip(*pairs))
            states = []
            for p, g in pairs:
                if g.is_sparse:
                    raise RuntimeError("FusedAdam does not support sparse gradients")
                if not p.is_cuda or p.dtype != torch.float32:
                    raise TypeError(f"FusedAdam needs f32 parameters on a GPU, got {p.dtype} on {p.device}")
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, bits))
                states.append(state)
            keys = _STATE_KEYS[bits]
            other = next((state for state in states if keys[0] not in state), None)
            if other is not None:
                raise ValueError(f"FusedAdam has state_bits={bits} for a parameter whose state is of other bits: {sorted(other)}")
            beta1, beta2 = group["betas"]
            step_hip = adam_step_hip if bits == 32 else adam8_step_hip
            by_device: dict[int, list[int]] = defaultdict(list)
            for k, p in enumerate(params):
                by_device[p.get_device()].append(k)
            for device, which in by_device.items():
                ps, gs, ss = params, grads, states
                if len(which) < len(params):
                    ps, gs, ss = ([all_of[k] for k in which] for all_of in (params, grads, states))
                # the 8-bit operator makes its tensors' GPU the current one itself
                with torch.cuda.device(device) if bits == 32 else nullcontext():
                    step_hip(ps, gs, *[[state[key] for state in ss] for key in keys], lr=group["lr"], beta1=beta1,
                             beta2=beta2, eps=group["eps"], weight_decay=group["weight_decay"],
                             decoupled_weight_decay=group["decoupled_weight_decay"])
        return loss


class FusedAdamW(FusedAdam):
    """torch.optim.AdamW's update: FusedAdam with decoupled weight decay
    (default 1e-2, as torch.optim.AdamW)."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, amsgrad: bool = False, maximize: bool = False,
                 state_bits: int = 32) -> None:
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled_weight_decay=True,
                         amsgrad=amsgrad, maximize=maximize, state_bits=state_bits)

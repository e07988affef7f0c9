"""Adam for the Gaussian parameter groups, stepped by one HIP launch, and
AdamW for a latent decoder's.

The binary-tree trainer builds one ``torch.optim.Adam`` per parameter group
(``src/models/gaussian_model.py:514-530``) and steps them one after another
(``src/trainers/binary_tree.py:208-210``).  Two drop-ins:

* ``Adam``: a ``torch.optim.Adam`` whose ``step()`` is one launch
  (``r2s_adam_step_f32``) instead of torch's ten-odd element-wise kernels;
  same constructor, state layout (``step`` / ``exp_avg`` / ``exp_avg_sq``),
  ``state_dict`` and arithmetic.
* ``step_all(optimizers)``: one launch for several optimizers (ours or plain
  ``torch.optim.Adam`` with the supported options), replacing the trainer's
  ``for optimizer in optimizers.values(): optimizer.step()``.

Supported: float32 CUDA parameters, dense gradients, coupled weight decay;
not amsgrad, maximize, capturable, differentiable or fused -- those raise
``NotImplementedError`` (the reference uses none of them).

``AdamW`` (no reference counterpart) steps float32, bfloat16 and float16
parameters with decoupled weight decay; its states are float32 or 8 bits.
"""

from __future__ import annotations

import ctypes
import struct
from typing import Iterable, List

import torch
from torch.optim.optimizer import _get_scalar_dtype

from .cuda import _backend
from .cuda import _lib as L
from .cuda import _ops

__all__ = ["Adam", "AdamW", "step_all"]


def _check_group(group: dict) -> None:
    _check_options(group, ("amsgrad", "maximize", "capturable", "differentiable", "fused",
                           "decoupled_weight_decay"))


def _check_options(group: dict, refused) -> None:
    for key in refused:
        if group.get(key):
            raise NotImplementedError(f"the fused Adam step does not support {key}=True")
    for key in ("lr", "eps", "weight_decay"):
        if isinstance(group[key], torch.Tensor):
            raise NotImplementedError(f"the fused Adam step needs a float {key}")
    if any(isinstance(b, torch.Tensor) for b in group["betas"]):
        raise NotImplementedError("the fused Adam step needs float betas")


def _entries(optimizer: torch.optim.Optimizer, out: List[L.AdamTensor], keep: list) -> None:
    """Append one r2s_adam_tensor_t per parameter with a gradient; advances
    each parameter's step count as torch's Adam does."""
    for group in optimizer.param_groups:
        _check_group(group)
        lr, (beta1, beta2) = group["lr"], group["betas"]
        eps, wd = group["eps"], group["weight_decay"]
        for p in group["params"]:
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise RuntimeError("Adam does not support sparse gradients, please consider "
                                   "SparseAdam instead")
            if not p.is_cuda or p.dtype != torch.float32:
                raise NotImplementedError("the fused Adam step needs float32 CUDA parameters")
            state = optimizer.state[p]
            if len(state) == 0:  # torch/optim/adam.py _init_group
                state["step"] = torch.tensor(0.0, dtype=_get_scalar_dtype())
                state["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                state["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            m, v = state["exp_avg"], state["exp_avg_sq"]
            if not (p.is_contiguous() and m.is_contiguous() and v.is_contiguous()):
                raise NotImplementedError("the fused Adam step needs contiguous tensors")
            if m.shape != p.shape or v.shape != p.shape:
                raise RuntimeError("Adam state does not match its parameter")
            grad = p.grad.contiguous()
            state["step"] += 1
            step = float(state["step"].item()) if isinstance(state["step"], torch.Tensor) \
                else float(state["step"])
            # torch/optim/adam.py _multi_tensor_adam, non-capturable branch.
            bias_correction1 = 1 - beta1 ** step
            bias_correction2 = 1 - beta2 ** step
            step_size = (lr / bias_correction1) * -1
            bias_correction2_sqrt = bias_correction2 ** 0.5
            out.append(L.AdamTensor(p.data_ptr(), grad.data_ptr(), m.data_ptr(), v.data_ptr(),
                                    p.numel(), 1 - beta1, beta2, 1 - beta2, wd,
                                    bias_correction2_sqrt, eps, step_size))
            keep.append(grad)


def _launch(entries: List[L.AdamTensor], device) -> None:
    if not entries:
        return
    lib = _backend.library()
    table = (L.AdamTensor * len(entries))(*entries)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        rc = lib.r2s_adam_step_f32(ctypes.cast(table, ctypes.c_void_p), len(entries), stream)
    if rc != 0:
        raise RuntimeError(f"r2s_adam_step_f32 failed ({rc}): "
                           f"{lib.r2s_last_error().decode(errors='replace')}")


def _device_of(optimizers) -> torch.device:
    for opt in optimizers:
        for group in opt.param_groups:
            for p in group["params"]:
                return p.device
    return torch.device("cuda")


def step_all(optimizers: Iterable[torch.optim.Optimizer]) -> None:
    """``optimizer.step()`` for every optimizer, as one launch."""
    opts = list(optimizers.values() if isinstance(optimizers, dict) else optimizers)
    for opt in opts:
        if not isinstance(opt, torch.optim.Adam):
            raise TypeError(f"step_all steps Adam optimizers, got {type(opt).__name__}")
    entries: List[L.AdamTensor] = []
    keep: list = []
    with torch.no_grad():
        for opt in opts:
            _entries(opt, entries, keep)
        _launch(entries, _device_of(opts))


class Adam(torch.optim.Adam):
    """torch.optim.Adam with a one-launch ``step()`` (see module docstring)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0,
                 amsgrad=False, **kwargs):
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                         amsgrad=amsgrad, **kwargs)
        for group in self.param_groups:
            _check_group(group)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        entries: List[L.AdamTensor] = []
        keep: list = []
        _entries(self, entries, keep)
        _launch(entries, _device_of([self]))
        return loss


# Elements that share a scale of 8-bit states, and the fewest that a tensor has
# whose states are kept in 8 bits: below, the scales' and the launch's share is
# larger than what is saved.
_RUN = 256
_FEWEST_8BIT = 4096
_PARAM_TYPES = {torch.float32: L.TYPE_F32, torch.bfloat16: L.TYPE_BF16,
                torch.float16: L.TYPE_F16}
# r2s_adamw_tensor_t, packed without a ctypes object for each tensor.
_ENTRY = struct.Struct("<7Qq8fiI")
assert _ENTRY.size == ctypes.sizeof(L.AdamwTensor)
# The names of states in 32 bits, and in 8 with the scales of each run.
_STATE_32 = ("exp_avg", "exp_avg_sq")
_STATE_8 = ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")
_WANTED_32 = ("master", *_STATE_32, None, None)
_WANTED_8 = ("master", *_STATE_8[::2], *_STATE_8[1::2])


def _check_bits(bits) -> None:
    if bits not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32, got {bits}")


def _check_adamw_group(group: dict) -> None:
    _check_options(group, ("amsgrad", "maximize", "capturable", "differentiable"))
    if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
        raise NotImplementedError("the fused AdamW step does not support "
                                  "decoupled_weight_decay=False")
    _check_bits(group["state_bits"])


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` over float32, bfloat16 and float16 CUDA parameters
    (gradients of their type), one launch for every 32 tensors of a device.

    The step is made in float32.  A 16-bit parameter keeps a float32 copy in its
    state (``master``), taken at its first step, and is that copy's rounding
    after every step; elements that are written in between are taken up by the
    next, and go on from their new values.  With
    ``state_bits=32`` the states are torch's (``exp_avg``, ``exp_avg_sq``) and so
    is the arithmetic, bit for bit in float32.  With ``state_bits=8`` tensors of
    at least 4096 elements keep float8 codes of the average (``exp_avg``) and of
    the root of the average of squares (``exp_avg_sq_root``) with a float32 scale
    for every 256 elements (``exp_avg_scale``, ``exp_avg_sq_root_scale``): a code
    times its scale is the value.  Codes are rounded up by chance, the chances a
    function of the element's index and the step, so that a run can be repeated
    bit for bit.  A gradient that is not finite makes its own element NaN.

    The step's scalars come from the host: ``step()`` refuses to be captured into
    a graph, where they would stay those of the capture."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 state_bits=32):
        _check_bits(state_bits)
        if not isinstance(lr, torch.Tensor) and lr < 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not isinstance(eps, torch.Tensor) and eps < 0.0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for i, beta in enumerate(betas):
            if not isinstance(beta, torch.Tensor) and not 0.0 <= beta < 1.0:
                raise ValueError(f"Invalid beta parameter at index {i}: {beta}")
        if not isinstance(weight_decay, torch.Tensor) and weight_decay < 0.0:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits))

    def add_param_group(self, param_group: dict) -> None:
        _check_adamw_group({**self.defaults, **param_group})
        super().add_param_group(param_group)

    @staticmethod
    def _new_state(p: torch.Tensor, bits: int) -> dict:
        state = {"step": 0}
        if p.dtype != torch.float32:
            state["master"] = p.detach().float()
        if bits == 8 and p.numel() >= _FEWEST_8BIT:
            runs = -(-p.numel() // _RUN)
            for name in _STATE_8[::2]:
                state[name] = torch.zeros_like(p, dtype=torch.float8_e4m3fn)
                state[name + "_scale"] = torch.zeros(runs, dtype=torch.float32, device=p.device)
        else:
            for name in _STATE_32:
                state[name] = torch.zeros_like(p, dtype=torch.float32)
        return state

    @staticmethod
    def _state_tensors(p: torch.Tensor, state: dict, n: int) -> tuple:
        """(master, average, second, their scales), None for those that are not
        there, checked at every step: the kernel takes their addresses."""
        device, f32 = p.get_device(), torch.float32
        if "exp_avg_sq_root" in state:
            wanted, kinds, runs = _WANTED_8, torch.float8_e4m3fn, -(-n // _RUN)
        else:
            wanted, kinds, runs = _WANTED_32, f32, None
        out = []
        for name in wanted:
            if name is None or (name == "master" and p.dtype is f32):
                out.append(None)
                continue
            t, scale = state.get(name), name.endswith("_scale")
            if not isinstance(t, torch.Tensor) or t.get_device() != device \
                    or t.dtype is not (kinds if name != "master" and not scale else f32) \
                    or t.numel() != (runs if scale else n) or not t.is_contiguous():
                raise RuntimeError(f"AdamW state {name!r} does not match its parameter")
            out.append(t)
        return out

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # device -> (packed entries, gradients kept until the launch, what it counts).
        # Nothing of the optimizer changes before every parameter has been looked over.
        work: dict = {}
        for group in self.param_groups:
            _check_adamw_group(group)
            lr, (beta1, beta2) = group["lr"], group["betas"]
            fixed = beta1, 1 - beta1, beta2, 1 - beta2, 1 - lr * group["weight_decay"]
            eps = group["eps"]
            last, scalars = None, ()  # those of one step count serve all that share it
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                if grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                device = p.device
                if grad.dtype != p.dtype or grad.device != device or grad.shape != p.shape:
                    raise RuntimeError("AdamW gradient does not match its parameter")
                if device not in work:
                    if p.is_cuda:
                        with _ops._on(device):
                            if torch.cuda.is_current_stream_capturing():
                                raise RuntimeError("AdamW.step cannot be captured into a graph")
                    work[device] = [], [], []
                entries, kept, counted = work[device]
                kind = _PARAM_TYPES.get(p.dtype)
                if kind is None or not p.is_cuda:
                    raise NotImplementedError("the fused AdamW step needs float32, bfloat16 or "
                                              "float16 CUDA parameters")
                if not p.is_contiguous():
                    raise NotImplementedError("the fused AdamW step needs contiguous parameters")
                state = self.state.get(p) or self._new_state(p, group["state_bits"])
                n = p.numel()
                master, mean, second, scale, second_scale = self._state_tensors(p, state, n)
                if not grad.is_contiguous():
                    grad = grad.contiguous()
                step = int(state["step"]) + 1
                if step != last:
                    last, scalars = step, ((1 - beta2 ** step) ** 0.5, eps,
                                           -lr / (1 - beta1 ** step))
                entries.append(_ENTRY.pack(
                    p.data_ptr(), grad.data_ptr(), 0 if master is None else master.data_ptr(),
                    mean.data_ptr(), second.data_ptr(), 0 if scale is None else scale.data_ptr(),
                    0 if second_scale is None else second_scale.data_ptr(), n, *fixed,
                    *scalars, kind, step & 0xFFFFFFFF))
                kept.append(grad)
                counted.append((p, state, step))
        lib = _backend.library() if work else None
        for device, (entries, _, counted) in work.items():
            table = b"".join(entries)
            with _ops._on(device):
                rc = lib.r2s_adamw_step(table, len(entries), _ops._stream(device))
            if rc != 0:
                raise RuntimeError(f"r2s_adamw_step failed ({rc}): "
                                   f"{lib.r2s_last_error().decode(errors='replace')}")
            for p, state, step in counted:
                state["step"] = step
                self.state[p] = state
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """torch's, with the states in the types that they were saved in (torch
        casts them to their parameters').  Groups saved by torch's AdamW keep the
        ``state_bits`` that they have here; what the step does not do is refused."""
        given: dict = {}

        def settle(_, state_dict):  # behind the caller's hooks
            groups = [{"state_bits": own["state_bits"], **group}
                      for own, group in zip(self.param_groups, state_dict["param_groups"])]
            if len(groups) == len(state_dict["param_groups"]):  # else torch refuses it
                for group in groups:
                    _check_adamw_group(group)
                state_dict = {**state_dict, "param_groups": groups}
            given.update(state_dict)
            return state_dict

        def restore(_):  # and before theirs
            ids = [i for group in given["param_groups"] for i in group["params"]]
            params = [p for group in self.param_groups for p in group["params"]]
            for i, p in zip(ids, params):
                for name, t in given["state"].get(i, {}).items():
                    if name != "step" and isinstance(t, torch.Tensor):
                        self.state[p][name] = t.detach().to(p.device, copy=True).contiguous()

        hooks = (self.register_load_state_dict_pre_hook(settle),
                 self.register_load_state_dict_post_hook(restore, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

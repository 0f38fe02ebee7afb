"""What trains beside Muon: AdamW for the parameters Muon does not take (embeddings, heads, norms,
biases), with moments in 32 bits or in 8, and the clipping of all gradients by their norm.

The reference leaves both to ``torch``; here a step over all tensors is one call of the library
(``fm_adamw_step``): one launch for the step counts and one per kind of tensor, whatever their number
and sizes.

    muon = Muon(matrices, lr=0.02, rank=0, world_size=1)
    adamw = AdamW(others, lr=3e-4, betas=(0.9, 0.95), weight_decay=0.1, state_bits=8)
    ...
    norm = clip_grad_norm_(model.parameters(), 1.0)
    muon.step(); adamw.step()

Where only AdamW needs the clipped gradients, ``norm, scale = grad_norm(grads, 1.0)`` followed by
``adamw.step(grad_scale=scale)`` saves the pass that writes them.

CPU tensors raise ``AssertionError`` like the other operators: there is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
import math
from collections.abc import Iterable, Sequence

import torch
from torch import Tensor

from ._lib import check, dtype_code, lib
from .ops import _raw_stream

__all__ = ["AdamW", "adamw_step", "adamw8_step", "adamw8_values", "adamw8_encode", "grad_norm",
           "clip_grad_norm_"]

_BLOCK = 32  # elements that share an exponent byte of an 8-bit state


def _blocks(n: int) -> int:
    return -(-n // _BLOCK)


@functools.cache
def _host():
    """The extension through which the entries that take lists of tensors are called: it checks the tensors
    and fills the library's arrays.  It is bound to the Python and the torch it was built for, the library is
    not: Muon and the matrix operators run without it, so it is loaded at its first use."""
    try:
        from . import _host as extension
    except ImportError as e:
        raise ImportError("the extension flash_muon_b200._host is missing or was built for another Python or torch: "
                          "build it with `python flash_muon_b200/build.py`") from e
    return extension


(_STEP, _NORM, _NORM_BYTES, _SCALE, _VALUES) = (
    ctypes.cast(fn, ctypes.c_void_p).value for fn in
    (lib.fm_adamw_step, lib.fm_grad_norm, lib.fm_grad_norm_workspace_bytes, lib.fm_scale_multi, lib.fm_adamw8_values))


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], steps: Tensor | Sequence[Tensor], *, lr: float | Tensor,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               masters: Sequence[Tensor] | None = None, grad_scale: Tensor | None = None) -> None:
    """One AdamW step of every tensor, in place, moments in float32.

    Gradients, moments and masters have their parameter's shape, or are flat.
    ``steps`` holds a float32 count per tensor (a 1-D tensor or a list of scalars); the call adds one
    to each.  ``masters`` are float32 copies of 16-bit parameters that carry the bits those lose.
    ``grad_scale``, a float32 scalar on the device, multiplies the gradients; if it is not finite
    nothing is written, the counts included.  ``lr`` may be such a scalar too.  Parameters are
    bfloat16, float16 or float32; a 16-bit parameter takes gradients of its own type or float32.
    """
    rc = _host().adamw_step(_STEP, ((params, grads, masters, exp_avgs, exp_avg_sqs, None, None, steps, None, lr,
                                     *betas, eps, weight_decay),), grad_scale)
    if rc:
        check(rc)


def adamw8_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
                exp_avg_scales: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor],
                exp_avg_sq_scales: Sequence[Tensor], steps: Tensor | Sequence[Tensor], *,
                seeds: int | Sequence[int] = 0, lr: float | Tensor,
                betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                masters: Sequence[Tensor] | None = None, grad_scale: Tensor | None = None) -> None:
    """``adamw_step`` with the moments in 8 bits.

    ``exp_avgs`` and ``exp_avg_sqs`` are uint8, one byte per element padded to a multiple of 32;
    the scales are uint8, one byte per 32 elements; all zeros are zero moments.  Moments are rounded
    up or down at random (include/flash_muon_b200.h gives the format); the random numbers are a
    function of the tensor's seed (``seeds[i]``, or ``seeds + i``), its step count and the element's
    index, so replicas that take the same step stay equal bit for bit.
    """
    if isinstance(seeds, int):
        seeds = range(seeds, seeds + len(params))
    rc = _host().adamw_step(_STEP, ((params, grads, masters, exp_avgs, exp_avg_sqs, exp_avg_scales,
                                     exp_avg_sq_scales, steps, seeds, lr, *betas, eps, weight_decay),), grad_scale)
    if rc:
        check(rc)


def adamw8_values(codes: Tensor, scales: Tensor, *, moment: int, numel: int | None = None,
                  dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The values that 8-bit states stand for, flat: ``moment`` 1 for ``exp_avg``, 2 for ``exp_avg_sq``;
    ``numel`` drops the padding.  bfloat16 and float32 hold them exactly."""
    rc, values = _host().adamw8_values(_VALUES, codes, scales, moment, numel, dtype)
    if rc:
        check(rc)
    return values


def adamw8_encode(values: Tensor, *, moment: int) -> tuple[Tensor, Tensor]:
    """Codes and scales of ``values``, rounded to nearest (``moment`` 1 or 2): how a checkpoint with
    float moments continues with 8-bit ones."""
    assert moment in (1, 2), "moment must be 1 (exp_avg) or 2 (exp_avg_sq)"
    assert values.is_cuda, "Input `values` must be a CUDA tensor"
    values = values.detach().contiguous()
    n = values.numel()
    with torch.cuda.device(values.device):
        codes = torch.empty(_blocks(n) * _BLOCK, dtype=torch.uint8, device=values.device)
        scales = torch.empty(_blocks(n), dtype=torch.uint8, device=values.device)
        check(lib.fm_adamw8_encode(values.data_ptr(), dtype_code(values.dtype), n, moment, codes.data_ptr(),
                                   scales.data_ptr(), _raw_stream(values.device.index)))
    return codes, scales


# ---------------------------------------------------------------- gradients
def grad_norm(grads: Sequence[Tensor], max_norm: float = math.inf) -> tuple[Tensor, Tensor]:
    """Euclidean norm over all elements of ``grads`` and the factor ``min(1, max_norm / (norm + 1e-6))``
    that clips them: two float32 scalars on the device, ready without a synchronisation for
    ``AdamW.step(grad_scale=...)``.  A norm that is not finite gives the factor NaN, with which a step
    is not taken.  Squares are formed in float32: one element above 1.8e19 makes the norm infinite, and elements
    below 1e-23 count for nothing.  Partial sums are added in 64 bits in a fixed order: equal inputs, equal
    bits."""
    rc, norm, scale = _host().grad_norm(_NORM, _NORM_BYTES, grads, max_norm)
    if rc:
        check(rc)
    return norm, scale


def clip_grad_norm_(parameters: Tensor | Iterable[Tensor], max_norm: float) -> Tensor:
    """Scales the gradients of ``parameters`` in place so that their norm is at most ``max_norm`` and
    returns the norm they had (``torch.nn.utils.clip_grad_norm_`` for the Euclidean norm).  Gradients
    within the norm are read once and left alone; if the norm is not finite (an element above 1.8e19 makes it
    infinite) all become NaN.  What torch's function does beyond that is not there: other norms,
    ``error_if_nonfinite``, gradients on several devices, gradients that are not contiguous (channels-last
    ones); a parameter that is given twice is refused."""
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    norm, scale = grad_norm(grads, max_norm)
    rc = _host().scale(_SCALE, grads, scale)
    if rc:
        check(rc)
    return norm


# ---------------------------------------------------------------- optimizer
class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over the library's multi-tensor step.

    ``lr`` (a float, or a float32 scalar on the device that a schedule inside a CUDA graph writes),
    ``betas``, ``eps`` and ``weight_decay`` as in ``torch.optim.AdamW``.  ``state_bits`` 8 keeps the
    moments in 8 bits for parameters of at least ``min_8bit_numel`` elements (10.1 instead of 22 bytes
    of traffic per bfloat16 element and step, 2.06 instead of 8 bytes of state); ``master_weights``
    keeps a float32 copy of 16-bit parameters, made at the first step, from which the parameter is
    written: weights that are loaded later need ``state[p]["master"]`` written too.  Every setting can
    differ between parameter groups.

    State per parameter: ``step`` (float32 scalar on the device), ``exp_avg`` and ``exp_avg_sq``
    (float32 in the parameter's shape, or flat uint8 with ``exp_avg_scale`` and ``exp_avg_sq_scale``),
    ``master`` where asked for.  A checkpoint of ``torch.optim.AdamW`` loads, and so does one of this
    class with other ``state_bits``: the moments are converted.

    Counts live on the device, so ``step()`` can be captured in a CUDA graph after one eager step.
    Parameters and gradients must be contiguous.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=32,
                 min_8bit_numel=4096, master_weights=False, seed=0):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                        min_8bit_numel=min_8bit_numel, master_weights=master_weights, seed=seed)
        super().__init__(params, defaults)

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            assert group["state_bits"] in (8, 32), "state_bits must be 8 or 32"
            beta1, beta2 = group["betas"]
            assert 0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0, "betas must lie in [0, 1)"
            assert group["eps"] >= 0.0, "eps must not be negative"
            lr = group["lr"]
            assert not isinstance(lr, Tensor) or (lr.is_cuda and lr.dtype == torch.float32 and lr.numel() == 1), \
                "`lr` must be a number or a float32 scalar on the parameters' CUDA device"
            for p in group["params"]:
                dtype_code(p.dtype)
        except BaseException:
            self.param_groups.pop()
            raise

    def _eight(self, p: Tensor, group) -> bool:
        return group["state_bits"] == 8 and p.numel() >= group["min_8bit_numel"]

    def _init_state(self, p: Tensor, group) -> None:
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        if self._eight(p, group):
            blocks = _blocks(p.numel())
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(blocks * _BLOCK, dtype=torch.uint8, device=p.device)
                state[name + "_scale"] = torch.zeros(blocks, dtype=torch.uint8, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().float().contiguous().clone()
        self.state[p] = state  # whole, or after an error (out of memory) not at all

    def step(self, closure=None, *, grad_scale: Tensor | None = None):
        """One step of every parameter that has a gradient.  ``grad_scale``: see ``adamw_step``."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        rc = _host().optimizer_step(_STEP, self.param_groups, self.state, grad_scale)
        if isinstance(rc, list):  # parameters that have no state yet
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("take one step before capturing: a parameter has no state yet")
            for p, group in rc:
                with torch.cuda.device(p.device):
                    self._init_state(p, group)
            rc = _host().optimizer_step(_STEP, self.param_groups, self.state, grad_scale)
        if rc:
            check(rc)
        return loss

    def state_values(self, p: Tensor) -> tuple[Tensor, Tensor]:
        """``exp_avg`` and ``exp_avg_sq`` of a parameter in float32 and its shape, whatever their bits."""
        state = self.state[p]
        if "exp_avg_scale" not in state:
            return state["exp_avg"], state["exp_avg_sq"]
        return tuple(adamw8_values(state[k], state[k + "_scale"], moment=i, numel=p.numel(), dtype=torch.float32)
                     .view(p.shape) for i, k in ((1, "exp_avg"), (2, "exp_avg_sq")))

    # ------------------------------------------------------------------ checkpoints
    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Loads a checkpoint of this class or of ``torch.optim.AdamW`` (or ``Adam`` without weight decay).
        Moments keep 32 bits whatever the parameters' type (the base class would round them to it) and are
        converted between 32 and 8 bits where this optimizer's groups ask for the other.  A learning rate
        that is a tensor here stays that tensor and takes the checkpoint's value; else the value becomes a
        float.  The states are new tensors: a step that was captured in a CUDA graph has to be captured
        again."""
        before = [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]
        fresh: dict = {}

        def convert(_, state_dict):  # behind the caller's pre-hooks; the base class gets no state to round
            saved_groups = state_dict["param_groups"]
            own = [g["params"] for g in self.param_groups]
            if [len(g["params"]) for g in saved_groups] != [len(g) for g in own]:
                raise ValueError("loaded state dict has other parameter groups")
            for saved in saved_groups:
                for key in ("amsgrad", "maximize"):
                    if saved.get(key):
                        raise ValueError(f"`{key}` is not supported")
                if saved.get("decoupled_weight_decay") is False and saved.get("weight_decay"):
                    raise ValueError("a checkpoint of Adam, whose weight decay enters the gradient, is not supported")
            for group, saved in zip(self.param_groups, saved_groups):
                for p, pid in zip(group["params"], saved["params"]):
                    if pid in state_dict["state"]:
                        fresh[p] = self._loaded(p, group, state_dict["state"][pid])
            return {**state_dict, "state": {}}

        def install(_):  # ahead of the caller's post-hooks
            for group, settings in zip(self.param_groups, before):
                for key, value in settings.items():  # how states are kept is this optimizer's choice
                    if key in ("state_bits", "min_8bit_numel", "master_weights") or key not in group:
                        group[key] = value
                if "decoupled_weight_decay" in group:
                    group["decoupled_weight_decay"] = True  # without decay Adam is AdamW
                lr = settings["lr"]
                if isinstance(lr, Tensor):               # a schedule holds it
                    lr.copy_(group["lr"]) if isinstance(group["lr"], Tensor) else lr.fill_(group["lr"])
                    group["lr"] = lr
                else:
                    group["lr"] = float(group["lr"])
            self.state.update(fresh)

        hooks = (self.register_load_state_dict_pre_hook(convert),
                 self.register_load_state_dict_post_hook(install, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _loaded(self, p: Tensor, group, saved: dict) -> dict:
        for key in ("step", "exp_avg", "exp_avg_sq"):
            if key not in saved:
                raise ValueError(f"loaded state of a parameter has no `{key}`")
        state = {"step": torch.as_tensor(saved["step"], dtype=torch.float32).to(p.device).reshape(()).clone()}
        eight = self._eight(p, group)
        for moment, key in ((1, "exp_avg"), (2, "exp_avg_sq")):
            x = saved[key].to(p.device)
            if key + "_scale" in saved:
                scale = saved[key + "_scale"].to(p.device)
                if x.numel() != _blocks(p.numel()) * _BLOCK or scale.numel() != _blocks(p.numel()):
                    raise ValueError(f"loaded `{key}` does not have the parameter's size")
                if eight:
                    state[key], state[key + "_scale"] = x.clone(), scale.clone()
                else:
                    state[key] = adamw8_values(x, scale, moment=moment, numel=p.numel(), dtype=torch.float32).view(p.shape)
                continue
            if x.numel() != p.numel():
                raise ValueError(f"loaded `{key}` does not have the parameter's size")
            if eight:
                state[key], state[key + "_scale"] = adamw8_encode(x.float(), moment=moment)
            else:
                state[key] = x.to(torch.float32).reshape(p.shape).contiguous().clone()
        if group["master_weights"] and p.dtype != torch.float32:
            master = saved.get("master")
            state["master"] = (p.detach() if master is None else master.to(p.device)).float().reshape(p.shape).contiguous().clone()
        return state

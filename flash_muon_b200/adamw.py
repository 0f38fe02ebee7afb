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
import math
from array import array
from collections.abc import Iterable, Sequence
from operator import attrgetter

import torch
from torch import Tensor

from ._lib import AdamWGroup, check, dtype_code, lib
from .ops import _current_device, _raw_stream

__all__ = ["AdamW", "adamw_step", "adamw8_step", "adamw8_values", "adamw8_encode", "grad_norm",
           "clip_grad_norm_"]

_BLOCK = 32  # elements that share an exponent byte of an 8-bit state

_dtype_of = attrgetter("dtype")
_is_cuda = attrgetter("is_cuda")


def _blocks(n: int) -> int:
    return -(-n // _BLOCK)


def _addresses(tensors) -> array:
    return array("Q", map(Tensor.data_ptr, tensors))


def _where(a: array | None):
    """Address of a host array's items (the array has to outlive the call)."""
    return a.buffer_info()[0] if a is not None else None


def _check_tensors(name: str, tensors: Sequence[Tensor], device: int) -> None:
    assert all(map(_is_cuda, tensors)), f"`{name}` must be CUDA tensors"
    assert all(map(Tensor.is_contiguous, tensors)), f"`{name}` must be contiguous"
    assert set(map(Tensor.get_device, tensors)) <= {device}, f"`{name}` must be on the parameters' device"


def _check_numels(name: str, tensors: Sequence[Tensor], numels: list[int]) -> None:
    assert list(map(Tensor.numel, tensors)) == numels, f"`{name}` must have the parameters' sizes"


def _check_dtype(name: str, tensors: Sequence[Tensor], dtype: torch.dtype) -> None:
    assert set(map(_dtype_of, tensors)) <= {dtype}, f"`{name}` must be {dtype}"


def _check_scalar(name: str, t: Tensor, device: int) -> None:
    assert t.is_cuda and t.get_device() == device and t.numel() == 1 and t.dtype == torch.float32, \
        f"`{name}` must be a float32 scalar on the parameters' CUDA device"


class _Group:
    """One parameter group of a call: validated lists, to be turned into ``fm_adamw_group``s."""

    def __init__(self, params, grads, exp_avgs, exp_avg_sqs, steps, lr, betas, eps, weight_decay,
                 masters=None, scales=None, seeds=None):
        n = len(params)
        assert n == len(grads) == len(exp_avgs) == len(exp_avg_sqs), "lists must have one entry per parameter"
        device = self.device = params[0].get_device()
        numels = self.numels = list(map(Tensor.numel, params))
        _check_tensors("params", params, device)
        _check_tensors("grads", grads, device)
        _check_numels("grads", grads, numels)
        _check_tensors("exp_avgs", exp_avgs, device)
        _check_tensors("exp_avg_sqs", exp_avg_sqs, device)
        if scales is None:
            _check_numels("exp_avgs", exp_avgs, numels)
            _check_numels("exp_avg_sqs", exp_avg_sqs, numels)
            _check_dtype("exp_avgs", exp_avgs, torch.float32)
            _check_dtype("exp_avg_sqs", exp_avg_sqs, torch.float32)
        else:
            blocks = list(map(_blocks, numels))
            padded = [b * _BLOCK for b in blocks]
            assert n == len(scales[0]) == len(scales[1]) == len(seeds), "lists must have one entry per parameter"
            for name, ts, sizes in (("exp_avgs", exp_avgs, padded), ("exp_avg_sqs", exp_avg_sqs, padded),
                                    ("exp_avg_scales", scales[0], blocks), ("exp_avg_sq_scales", scales[1], blocks)):
                _check_dtype(name, ts, torch.uint8)
                assert list(map(Tensor.numel, ts)) == sizes, \
                    f"`{name}` must have one byte per {'element, padded to 32' if sizes is padded else 'block of 32'}"
            _check_tensors("exp_avg_scales", scales[0], device)
            _check_tensors("exp_avg_sq_scales", scales[1], device)
        if masters is not None:
            assert n == len(masters), "lists must have one entry per parameter"
            assert torch.float32 not in set(map(_dtype_of, params)), "float32 parameters have no master copies"
            _check_tensors("masters", masters, device)
            _check_numels("masters", masters, numels)
            _check_dtype("masters", masters, torch.float32)
        if isinstance(steps, Tensor):
            assert steps.ndim == 1 and steps.numel() == n, "`steps` must have one count per parameter"
            _check_tensors("steps", [steps], device)
            _check_dtype("steps", [steps], torch.float32)
            at = steps.data_ptr()
            self.steps = array("Q", range(at, at + 4 * n, 4))
        else:
            assert len(steps) == n, "lists must have one entry per parameter"
            _check_tensors("steps", steps, device)
            _check_dtype("steps", steps, torch.float32)
            assert all(t.numel() == 1 for t in steps), "`steps` must be scalars"
            self.steps = _addresses(steps)
        self.lr_device = None
        if isinstance(lr, Tensor):
            _check_scalar("lr", lr, device)
            self.lr_device, lr = lr, 0.0
        beta1, beta2 = betas
        # refused here too: a captured call would otherwise fail only in the library
        assert 0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0, "betas must lie in [0, 1)"
        assert eps >= 0.0 and math.isfinite(eps), "eps must be finite and not negative"
        assert math.isfinite(lr) and math.isfinite(weight_decay), "lr and weight_decay must be finite"
        self.settings = (float(lr), float(beta1), float(beta2), float(eps), float(weight_decay))
        self.lists = (params, grads, masters, exp_avgs, exp_avg_sqs, *(scales or (None, None)))
        self.p_dtypes = list(map(_dtype_of, params))
        self.g_dtypes = list(map(_dtype_of, grads))
        self.seeds = None if seeds is None else [int(s) & 0xffffffff for s in seeds]
        self.bits = 32 if scales is None else 8

    def structs(self, keep: list):
        """``fm_adamw_group``s, one per pair of types; what they point to goes into ``keep``."""
        kinds = list(zip(self.p_dtypes, self.g_dtypes))
        for kind in dict.fromkeys(kinds):
            for dt in kind:
                dtype_code(dt)
            rows = None if len(set(kinds)) == 1 else [i for i, k in enumerate(kinds) if k == kind]
            pick = (lambda xs: xs) if rows is None else (lambda xs: [xs[i] for i in rows])
            g = AdamWGroup()
            arrays = [None if ts is None else _addresses(pick(ts)) for ts in self.lists]
            arrays.append(self.steps if rows is None else array("Q", pick(self.steps)))
            arrays.append(array("q", pick(self.numels)))
            arrays.append(None if self.seeds is None else array("I", pick(self.seeds)))
            keep.append(arrays)
            (g.params, g.grads, g.masters, g.exp_avg, g.exp_avg_sq, g.exp_avg_scale, g.exp_avg_sq_scale,
             g.steps, g.numels, g.seeds) = map(_where, arrays)
            g.count, g.state_bits = len(arrays[0]), self.bits
            g.p_dtype, g.g_dtype = dtype_code(kind[0]), dtype_code(kind[1])
            g.lr, g.beta1, g.beta2, g.eps, g.weight_decay = self.settings
            g.lr_device = None if self.lr_device is None else self.lr_device.data_ptr()
            yield g


def _launch(groups: list[_Group], grad_scale: Tensor | None) -> None:
    device = groups[0].device
    assert all(g.device == device for g in groups), "all parameters must be on one device"
    if grad_scale is not None:
        _check_scalar("grad_scale", grad_scale, device)
    keep: list = []
    structs = [s for g in groups for s in g.structs(keep)]
    table = (AdamWGroup * len(structs))(*structs)
    scale = None if grad_scale is None else grad_scale.data_ptr()
    if device != _current_device():
        with torch.cuda.device(device):
            check(lib.fm_adamw_step(table, len(structs), scale, _raw_stream(device)))
        return
    rc = lib.fm_adamw_step(table, len(structs), scale, _raw_stream(device))
    if rc:
        check(rc)


@torch.no_grad()
def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], steps: Tensor | Sequence[Tensor], *, lr: float | Tensor,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               masters: Sequence[Tensor] | None = None, grad_scale: Tensor | None = None) -> None:
    """One AdamW step of every tensor, in place, moments in float32.

    ``steps`` holds a float32 count per tensor (a 1-D tensor or a list of scalars); the call adds one
    to each.  ``masters`` are float32 copies of 16-bit parameters that carry the bits those lose.
    ``grad_scale``, a float32 scalar on the device, multiplies the gradients; if it is not finite
    nothing is written, the counts included.  ``lr`` may be such a scalar too.  Parameters are
    bfloat16, float16 or float32; a 16-bit parameter takes gradients of its own type or float32.
    """
    params = list(params)
    if params:
        _launch([_Group(params, list(grads), list(exp_avgs), list(exp_avg_sqs), steps, lr, betas, eps,
                        weight_decay, masters)], grad_scale)


@torch.no_grad()
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
    params = list(params)
    if params:
        if isinstance(seeds, int):
            seeds = range(seeds, seeds + len(params))
        _launch([_Group(params, list(grads), list(exp_avgs), list(exp_avg_sqs), steps, lr, betas, eps,
                        weight_decay, masters, (list(exp_avg_scales), list(exp_avg_sq_scales)), seeds)], grad_scale)


def _check_state8(codes: Tensor, scales: Tensor, moment: int) -> None:
    assert moment in (1, 2), "moment must be 1 (exp_avg) or 2 (exp_avg_sq)"
    assert codes.is_cuda and scales.is_cuda and codes.device == scales.device, "states must be CUDA tensors on one device"
    assert codes.dtype == scales.dtype == torch.uint8, "states must be uint8"
    assert codes.is_contiguous() and scales.is_contiguous(), "states must be contiguous"
    assert codes.numel() == scales.numel() * _BLOCK, "states must have one scale per 32 codes"


def adamw8_values(codes: Tensor, scales: Tensor, *, moment: int, numel: int | None = None,
                  dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The values that 8-bit states stand for, flat: ``moment`` 1 for ``exp_avg``, 2 for ``exp_avg_sq``;
    ``numel`` drops the padding.  bfloat16 and float32 hold them exactly."""
    _check_state8(codes, scales, moment)
    n = codes.numel() if numel is None else numel
    assert 0 <= n <= codes.numel(), "`numel` exceeds the states"
    with torch.cuda.device(codes.device):
        out = torch.empty(n, dtype=dtype, device=codes.device)
        check(lib.fm_adamw8_values(codes.data_ptr(), scales.data_ptr(), n, moment, out.data_ptr(),
                                   dtype_code(dtype), _raw_stream(codes.device.index)))
    return out


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
def _gradient_table(grads: Sequence[Tensor]):
    device = grads[0].get_device()
    _check_tensors("grads", grads, device)
    return (device, _addresses(grads), array("q", map(Tensor.numel, grads)),
            array("i", [dtype_code(g.dtype) for g in grads]))


@torch.no_grad()
def grad_norm(grads: Sequence[Tensor], max_norm: float = math.inf) -> tuple[Tensor, Tensor]:
    """Euclidean norm over all elements of ``grads`` and the factor ``min(1, max_norm / (norm + 1e-6))``
    that clips them: two float32 scalars on the device, ready without a synchronisation for
    ``AdamW.step(grad_scale=...)``.  A norm that is not finite gives the factor NaN, with which a step
    is not taken.  Partial sums are added in 64 bits in a fixed order: equal inputs, equal bits."""
    grads = list(grads)
    assert grads, "`grads` must not be empty"
    max_norm = float(max_norm)
    assert max_norm >= 0.0, "`max_norm` must not be negative"
    device, ptrs, numels, dtypes = _gradient_table(grads)
    if device != _current_device():
        with torch.cuda.device(device):
            return _grad_norm(grads, ptrs, numels, dtypes, max_norm, device)
    return _grad_norm(grads, ptrs, numels, dtypes, max_norm, device)


def _grad_norm(grads, ptrs, numels, dtypes, max_norm, device):
    need = int(lib.fm_grad_norm_workspace_bytes(len(grads)))
    # the result and, behind it, the scratch; fresh memory for every call: calls on other streams, and
    # graphs captured apart, have their own
    mem = torch.empty(4 + need // 4, dtype=torch.float32, device=grads[0].device)
    at = mem.data_ptr()
    rc = lib.fm_grad_norm(_where(ptrs), _where(numels), _where(dtypes), len(grads), max_norm, at, at + 16, need,
                          _raw_stream(device))
    if rc:
        check(rc)
    return mem[0], mem[1]


@torch.no_grad()
def clip_grad_norm_(parameters: Tensor | Iterable[Tensor], max_norm: float) -> Tensor:
    """Scales the gradients of ``parameters`` in place so that their norm is at most ``max_norm`` and
    returns the norm they had (``torch.nn.utils.clip_grad_norm_`` for the Euclidean norm).  Gradients
    within the norm are read once and left alone; if the norm is not finite all become NaN."""
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    norm, scale = grad_norm(grads, max_norm)
    device, ptrs, numels, dtypes = _gradient_table(grads)
    with torch.cuda.device(device):
        check(lib.fm_scale_multi(_where(ptrs), _where(numels), _where(dtypes), len(grads), scale.data_ptr(),
                                 _raw_stream(device)))
    return norm


# ---------------------------------------------------------------- optimizer
class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over the library's multi-tensor step.

    ``lr`` (a float, or a float32 scalar on the device that a schedule inside a CUDA graph writes),
    ``betas``, ``eps`` and ``weight_decay`` as in ``torch.optim.AdamW``.  ``state_bits`` 8 keeps the
    moments in 8 bits for parameters of at least ``min_8bit_numel`` elements (10.1 instead of 22 bytes
    of traffic per bfloat16 element and step, 2.06 instead of 8 bytes of state); ``master_weights``
    keeps a float32 copy of 16-bit parameters.  Every setting can differ between parameter groups.

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
            for p in group["params"]:
                dtype_code(p.dtype)
        except BaseException:
            self.param_groups.pop()
            raise

    def _eight(self, p: Tensor, group) -> bool:
        return group["state_bits"] == 8 and p.numel() >= group["min_8bit_numel"]

    def _init_state(self, p: Tensor, group) -> dict:
        state = self.state[p]
        state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
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
        return state

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: Tensor | None = None):
        """One step of every parameter that has a gradient.  ``grad_scale``: see ``adamw_step``."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        by_device: dict[int, list[_Group]] = {}
        index = 0
        for group in self.param_groups:
            kinds: dict[tuple, list] = {}
            for p in group["params"]:
                index += 1
                if p.grad is None:
                    continue
                assert not p.grad.is_sparse, "AdamW takes no sparse gradients"
                assert p.is_cuda, "AdamW parameters must be CUDA tensors"
                state = self.state.get(p)
                if not state:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("take one step before capturing: a parameter has no state yet")
                    state = self._init_state(p, group)
                kinds.setdefault((p.get_device(), "exp_avg_scale" in state, "master" in state), []).append((p, state, group["seed"] + index))
            for (device, eight, masters), rows in kinds.items():
                ps = [p for p, _, _ in rows]
                states = [s for _, s, _ in rows]
                by_device.setdefault(device, []).append(_Group(
                    ps, [p.grad for p in ps], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                    [s["step"] for s in states], group["lr"], group["betas"], group["eps"], group["weight_decay"],
                    [s["master"] for s in states] if masters else None,
                    ([s["exp_avg_scale"] for s in states], [s["exp_avg_sq_scale"] for s in states]) if eight else None,
                    [i for _, _, i in rows] if eight else None))
        for groups in by_device.values():
            _launch(groups, grad_scale)
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
        """Loads a checkpoint of this class or of ``torch.optim.AdamW``.  Moments keep 32 bits whatever the
        parameters' type (the base class would round them to it) and are converted between 32 and 8
        bits where this optimizer's groups ask for the other."""
        saved_groups = state_dict["param_groups"]
        own = [g["params"] for g in self.param_groups]
        if [len(g["params"]) for g in saved_groups] != [len(g) for g in own]:
            raise ValueError("loaded state dict has other parameter groups")
        for saved in saved_groups:
            for key in ("amsgrad", "maximize"):
                if saved.get(key):
                    raise ValueError(f"`{key}` is not supported")
        before = [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]
        fresh: dict = {}
        for group, saved in zip(self.param_groups, saved_groups):
            for p, pid in zip(group["params"], saved["params"]):
                if pid in state_dict["state"]:
                    fresh[p] = self._loaded(p, group, state_dict["state"][pid])
        super().load_state_dict({"state": {}, "param_groups": saved_groups})
        for group, settings in zip(self.param_groups, before):
            for key, value in settings.items():  # how states are kept is this optimizer's choice
                if key in ("state_bits", "min_8bit_numel", "master_weights") or key not in group:
                    group[key] = value
            if isinstance(group["lr"], Tensor) and not group["lr"].is_cuda:
                group["lr"] = float(group["lr"])
        self.state.update(fresh)

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

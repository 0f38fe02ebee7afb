"""AdamW, its 8-bit states and the gradient norm, as far as no GPU is needed: the arithmetic of the
states compiled for the host, the oracle's own consistency, and the refusals of the C entries (checked
before any CUDA call) and of the Python operators."""
import ctypes
import math
import shutil
import subprocess
from array import array
from pathlib import Path

import pytest
import torch

import flash_muon_b200 as fm
from flash_muon_b200 import _lib
from flash_muon_b200._lib import AdamWGroup, lib
from oracle import adamw_oracle as A

ROOT = Path(__file__).resolve().parents[1]
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -5


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_state8_arithmetic(tmp_path):
    exe = tmp_path / "state8_check"
    build = subprocess.run(
        ["g++", "-O2", "-std=c++17", "-I", str(ROOT / "flash_muon_b200" / "csrc"),
         "-x", "c++", str(ROOT / "tests" / "state8_check.cpp"), "-o", str(exe)],
        capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert run.stdout.startswith("OK ")


@pytest.mark.parametrize("moment", [1, 2])
def test_oracle_codes_round_trip(moment):
    """decode and rounding_position of the oracle agree: a code's value lies at the code."""
    codes = torch.arange(127 if moment == 1 else 255, dtype=torch.uint8)
    codes = A.pad(codes)
    scales = torch.full((len(codes) // 32,), 100, dtype=torch.uint8)
    pos = A.rounding_position(A.decode(codes, scales, moment), scales, moment)
    assert torch.equal(pos, codes.double())


def test_oracle_random_numbers_differ_between_moments_steps_and_seeds():
    u, w = A.random_numbers(3, 5, 200)
    assert (u != w).any() and ((0 <= u) & (u < 1)).all()
    for other in (A.random_numbers(4, 5, 200), A.random_numbers(3, 6, 200), A.random_numbers(3, 5, 200, 1 << 32)):
        assert (other[0] != u).float().mean() > 0.9
    assert torch.equal(A.random_numbers(3, 5, 100, 100)[0], u[100:])


# ---------------------------------------------------------------- refusals of the C entry
class Call:
    """A valid one-tensor group over made-up addresses (nothing is launched by a refused call)."""

    def __init__(self, bits=32, n=64, **change):
        at = dict(params=0x10000, grads=0x20000, masters=0x30000, exp_avg=0x40000, exp_avg_sq=0x50000,
                  exp_avg_scale=0x60000, exp_avg_sq_scale=0x70000, steps=0x80000)
        at.update({k: v for k, v in change.items() if k in at})
        self.keep = {k: array("Q", [v]) for k, v in at.items() if v is not None}
        self.keep["numels"] = array("q", [change.get("numel", n)])
        self.keep["seeds"] = array("I", [1])
        g = self.g = AdamWGroup()
        for k, a in self.keep.items():
            setattr(g, k, a.buffer_info()[0])
        if "masters" not in change:
            g.masters = None
        if bits == 32:
            g.exp_avg_scale = g.exp_avg_sq_scale = g.seeds = None
        g.count, g.p_dtype, g.g_dtype, g.state_bits = 1, _lib.FM_F32, _lib.FM_F32, bits
        g.lr, g.beta1, g.beta2, g.eps, g.weight_decay = 1e-3, 0.9, 0.999, 1e-8, 0.01
        for k in ("count", "p_dtype", "g_dtype", "state_bits", "lr", "beta1", "beta2", "eps", "weight_decay", "lr_device"):
            if k in change:
                setattr(g, k, change[k])
        for k in change.get("null", ()):
            setattr(g, k, None)

    def __call__(self, scale=None):
        return lib.fm_adamw_step(self.g, 1, scale, None)


@pytest.mark.parametrize("change, status, message", [
    (dict(count=-1), INVALID, b"negative count"),
    (dict(null=["params"]), INVALID, b"null array"),
    (dict(null=["steps"]), INVALID, b"null array"),
    (dict(state_bits=16), UNSUPPORTED, b"32 or 8 bits"),
    (dict(bits=8, null=["seeds"]), INVALID, b"scales and seeds"),
    (dict(p_dtype=7), UNSUPPORTED, b"dtype"),
    (dict(p_dtype=_lib.FM_BF16, g_dtype=_lib.FM_F16), UNSUPPORTED, b"16-bit parameters"),
    (dict(masters=0x30000), UNSUPPORTED, b"no master copies"),
    (dict(beta1=1.0), INVALID, b"betas"),
    (dict(beta2=float("nan")), INVALID, b"betas"),
    (dict(eps=-1e-8), INVALID, b"eps"),
    (dict(lr=float("inf")), INVALID, b"finite"),
    (dict(weight_decay=float("nan")), INVALID, b"finite"),
    (dict(lr_device=0x90002), INVALID, b"misaligned lr"),
    (dict(numel=-1), INVALID, b"element count"),
    (dict(numel=(1 << 38) + 1), INVALID, b"element count"),
    (dict(params=0), INVALID, b"null tensor"),
    (dict(exp_avg_sq=0), INVALID, b"null tensor"),
    (dict(params=0x10002), INVALID, b"misaligned tensor"),
    (dict(steps=0x80001), INVALID, b"bad step count"),
    (dict(steps=0), INVALID, b"bad step count"),
    (dict(bits=8, exp_avg=0x40008), INVALID, b"misaligned tensor"),
    (dict(bits=8, exp_avg_scale=0), INVALID, b"null scales"),
    # memory that is written and overlaps other memory of the call
    (dict(exp_avg=0x50000), INVALID, b"overlap"),
    (dict(exp_avg=0x50000 + 4 * 63), INVALID, b"overlap"),
    (dict(grads=0x10000), INVALID, b"overlap"),
    (dict(steps=0x10000 + 4 * 63), INVALID, b"overlap"),
    (dict(bits=8, exp_avg_scale=0x70001), INVALID, b"overlap"),
])
def test_step_refuses(change, status, message):
    assert Call(**change)() == status
    assert message in lib.fm_last_error()


def test_step_refuses_the_same_parameter_twice_and_shared_counts():
    for twice in ("params", "steps"):
        two = {k: array("Q", [v, v if k == twice else v + 0x100000]) for k, v in
               dict(params=0x10000, grads=0x20000, exp_avg=0x40000, exp_avg_sq=0x50000, steps=0x80000).items()}
        two["numels"] = array("q", [64, 64])
        g = Call().g
        for k, a in two.items():
            setattr(g, k, a.buffer_info()[0])
        g.count = 2
        assert lib.fm_adamw_step(g, 1, None, None) == INVALID
        assert b"overlap" in lib.fm_last_error()


def test_step_refuses_bad_group_lists_and_scale():
    assert lib.fm_adamw_step(None, 1, None, None) == INVALID
    assert lib.fm_adamw_step(None, -1, None, None) == INVALID
    assert lib.fm_adamw_step(None, 0, None, None) == 0
    assert Call(count=0)() == 0
    assert Call()(0x90002) == INVALID and b"gradient scale" in lib.fm_last_error()
    assert Call()(0x10000 + 8) == INVALID and b"overlap" in lib.fm_last_error()          # inside the parameter
    assert Call(lr_device=0x80000)() == INVALID and b"overlap" in lib.fm_last_error()    # the count itself


def test_struct_layout_is_the_header_s():
    assert ctypes.sizeof(AdamWGroup) == 10 * 8 + 4 * 4 + 5 * 8 + 8


def test_values_and_encode_refuse():
    assert lib.fm_adamw8_values(None, None, 32, 1, None, 0, None) == INVALID
    assert lib.fm_adamw8_values(0x1000, 0x2000, 32, 3, 0x3000, 0, None) == INVALID
    assert lib.fm_adamw8_values(0x1000, 0x2000, 32, 1, 0x3000, 9, None) == UNSUPPORTED
    assert lib.fm_adamw8_values(None, None, -1, 1, None, 0, None) == INVALID
    assert lib.fm_adamw8_values(None, None, 0, 1, None, 0, None) == 0
    assert lib.fm_adamw8_encode(None, 0, 1, 1, None, None, None) == INVALID
    assert lib.fm_adamw8_encode(0x1000, 5, 1, 1, 0x2000, 0x3000, None) == UNSUPPORTED


def test_norm_and_scale_refuse():
    one = lambda v, t="Q": array(t, [v])  # noqa: E731
    ptr, n, dt = one(0x1000), one(4, "q"), one(0, "i")
    at = lambda a: a.buffer_info()[0]  # noqa: E731

    def norm(p=ptr, n=n, dt=dt, count=1, max_norm=1.0, result=0x2000, ws=0x3000, size=None):
        size = lib.fm_grad_norm_workspace_bytes(1) if size is None else size
        return lib.fm_grad_norm(at(p), at(n), at(dt), count, max_norm, result, ws, size, None)

    assert norm(count=-1) == INVALID
    assert norm(p=one(0)) == INVALID and norm(p=one(0x1001)) == INVALID
    assert norm(n=one(-1, "q")) == INVALID and norm(dt=one(3, "i")) == UNSUPPORTED
    assert norm(max_norm=-1.0) == INVALID and norm(max_norm=math.nan) == INVALID
    assert norm(result=0) == INVALID and norm(result=0x2002) == INVALID
    assert norm(ws=0) == INVALID and norm(ws=0x3004) == INVALID and norm(size=8) == WORKSPACE
    assert lib.fm_grad_norm(None, None, None, 1, 1.0, 0x2000, 0x3000, 1 << 20, None) == INVALID
    assert lib.fm_grad_norm_workspace_bytes(-1) == 0
    assert lib.fm_scale_multi(at(ptr), at(n), at(dt), 1, None, None) == INVALID
    assert lib.fm_scale_multi(at(ptr), at(n), at(dt), -1, 0x1000, None) == INVALID
    assert lib.fm_scale_multi(None, None, None, 0, 0x1000, None) == 0
    two = [array("Q", [0x2000, 0x1000]), array("q", [4, 2049]), array("i", [0, 0])]      # bf16: the second ends at 0x2002
    assert lib.fm_scale_multi(*map(at, two), 2, 0x8000, None) == INVALID and b"overlap" in lib.fm_last_error()
    two[0][1] = 0x2000
    assert lib.fm_scale_multi(*map(at, two), 2, 0x8000, None) == INVALID
    assert lib.fm_scale_multi(at(ptr), at(n), at(dt), 1, 0x1004, None) == INVALID        # the factor inside a tensor


# ---------------------------------------------------------------- refusals of the Python operators
def test_cpu_tensors_are_refused():
    p, g = torch.zeros(8), torch.zeros(8)
    with pytest.raises(AssertionError, match="`params` must be CUDA tensors"):
        fm.adamw_step([p], [g], [p.clone()], [p.clone()], torch.zeros(1), lr=1e-3)
    with pytest.raises(AssertionError, match="must be CUDA tensors"):
        fm.adamw8_step([p], [g], [p.byte()], [p.byte()], [p.byte()], [p.byte()], torch.zeros(1), lr=1e-3)
    with pytest.raises(AssertionError, match="must be CUDA tensors"):
        fm.grad_norm([g])
    with pytest.raises(AssertionError, match="must be a CUDA tensor"):
        fm.adamw8_encode(g, moment=1)
    with pytest.raises(AssertionError, match="must be CUDA tensors"):
        fm.adamw8_values(torch.zeros(32, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8), moment=1)
    p = torch.nn.Parameter(p)
    p.grad = g
    with pytest.raises(AssertionError, match="must be CUDA tensors"):
        fm.AdamW([p]).step()
    with pytest.raises(AssertionError, match="must be CUDA tensors"):
        fm.clip_grad_norm_([p], 1.0)


def test_operators_refuse_bad_arguments():
    with pytest.raises(AssertionError, match="one entry per parameter"):
        fm.adamw_step([torch.zeros(8)], [], [], [], torch.zeros(1), lr=1e-3)
    fm.adamw_step([], [], [], [], [], lr=1e-3)                     # nothing to do
    with pytest.raises(AssertionError, match="empty"):
        fm.grad_norm([])
    with pytest.raises(AssertionError, match="max_norm"):
        fm.grad_norm([torch.zeros(3)], -1.0)
    with pytest.raises(AssertionError, match="moment"):
        fm.adamw8_values(torch.zeros(32), torch.zeros(1), moment=0)
    assert float(fm.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0


@pytest.mark.parametrize("bad, message", [(dict(state_bits=4), "state_bits"), (dict(betas=(1.0, 0.9)), "betas"),
                                          (dict(eps=-1.0), "eps")])
def test_optimizer_refuses_bad_settings(bad, message):
    with pytest.raises(AssertionError, match=message):
        fm.AdamW([torch.nn.Parameter(torch.zeros(3))], **bad)
    opt = fm.AdamW([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(AssertionError, match=message):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(3))], **bad))
    assert len(opt.param_groups) == 1


def test_optimizer_refuses_types_and_foreign_checkpoints():
    with pytest.raises(TypeError, match="bfloat16"):
        fm.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    p = torch.nn.Parameter(torch.zeros(3))
    opt = fm.AdamW([p])
    with pytest.raises(ValueError, match="parameter groups"):
        opt.load_state_dict({"state": {}, "param_groups": []})
    saved = opt.state_dict()
    saved["state"] = {0: {"step": 1.0, "exp_avg": torch.zeros(4), "exp_avg_sq": torch.zeros(4)}}
    with pytest.raises(ValueError, match="size"):
        opt.load_state_dict(saved)
    saved["state"] = {0: {"step": 1.0}}
    with pytest.raises(ValueError, match="exp_avg"):
        opt.load_state_dict(saved)
    amsgrad = torch.optim.AdamW([torch.nn.Parameter(torch.zeros(3))], amsgrad=True).state_dict()
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(amsgrad)
    assert not opt.state and opt.param_groups[0]["state_bits"] == 32


def test_a_torch_checkpoint_loads_in_32_bits():
    """Moments of 16-bit parameters stay float32 (the base class would round them to the parameter)."""
    q = torch.nn.Parameter(torch.zeros(5, 3, dtype=torch.bfloat16))
    theirs = torch.optim.AdamW([q], lr=0.5, weight_decay=0.25)
    q.grad = torch.randn(5, 3).bfloat16()
    theirs.step()
    saved = theirs.state_dict()
    saved["state"][0]["exp_avg"] = torch.full((5, 3), 1 + 2.0 ** -20)
    opt = fm.AdamW([torch.nn.Parameter(torch.zeros(5, 3, dtype=torch.bfloat16))], master_weights=True)
    opt.load_state_dict(saved)
    p = opt.param_groups[0]["params"][0]
    state = opt.state[p]
    assert state["exp_avg"].dtype == torch.float32 and (state["exp_avg"] == 1 + 2.0 ** -20).all()
    assert state["exp_avg"].shape == (5, 3) and float(state["step"]) == 1.0
    assert state["master"].dtype == torch.float32
    assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["weight_decay"] == 0.25
    assert opt.param_groups[0]["master_weights"] and opt.param_groups[0]["seed"] == 0
    again = fm.AdamW([p])
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[p]["exp_avg"], state["exp_avg"])

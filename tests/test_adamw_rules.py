"""What AdamW, its 8-bit states and the clipping promise besides the step itself, as far as no GPU is
needed."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import flash_muon_b200 as fm
from flash_muon_b200 import _lib
from flash_muon_b200._lib import lib

ROOT = Path(__file__).resolve().parents[1]
INVALID = -1


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_codes_at_every_exponent_byte(tmp_path):
    exe = tmp_path / "state8_range_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(ROOT / "flash_muon_b200" / "csrc"), "-x", "c++",
                    str(ROOT / "tests" / "state8_range_check.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("dtype, size", [(_lib.FM_BF16, 2), (_lib.FM_F16, 2), (_lib.FM_F32, 4)])
def test_misaligned_values_are_refused(dtype, size):
    """By the host, ahead of the launch: on the GPU such an access is a fault."""
    for off in range(1, size):
        assert lib.fm_adamw8_values(0x1000, 0x2000, 32, 1, 0x3000 + off, dtype, None) == INVALID
        assert b"misaligned" in lib.fm_last_error()
        assert lib.fm_adamw8_encode(0x1000 + off, dtype, 32, 2, 0x2000, 0x3000, None) == INVALID
        assert b"misaligned" in lib.fm_last_error()


def test_muon_needs_no_extension():
    """Where the Python extension does not load the rest of the package does; what needs it names the build."""
    code = """if True:
        import sys
        sys.modules["flash_muon_b200._host"] = None          # its import fails
        import torch, flash_muon_b200 as fm
        fm.Muon, fm.matmul_transpose, fm.fast_newtonschulz
        assert fm.newtonschulz_workspace_bytes(4, 4) > 0
        p = torch.nn.Parameter(torch.zeros(4, 4))
        p.grad = torch.zeros(4, 4)
        for call in (lambda: fm.grad_norm([p]), lambda: fm.clip_grad_norm_([p], 1.0), lambda: fm.AdamW([p]).step(),
                     lambda: fm.adamw8_values(p, p, moment=1), lambda: fm.adamw_step([p], [p], [p], [p], p, lr=1.0),
                     lambda: fm.adamw8_step([p], [p], [p], [p], [p], [p], p, lr=1.0)):
            try:
                call()
            except ImportError as e:
                assert "python flash_muon_b200/build.py" in str(e)
            else:
                raise AssertionError
        print("fine")
    """
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert run.stdout.strip() == "fine", run.stderr


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_cannot_be_made_is_not_left_half_made(bits, monkeypatch):
    p = torch.nn.Parameter(torch.zeros(64, dtype=torch.bfloat16))
    opt = fm.AdamW([p], state_bits=bits, min_8bit_numel=0, master_weights=True)
    zeros, left = torch.zeros, [2]

    def failing(*args, **kwargs):
        left[0] -= 1
        if left[0] < 0:
            raise torch.OutOfMemoryError("no memory")
        return zeros(*args, **kwargs)

    monkeypatch.setattr(torch, "zeros", failing)
    with pytest.raises(torch.OutOfMemoryError):
        opt._init_state(p, opt.param_groups[0])
    assert p not in opt.state
    left[0] = 100
    opt._init_state(p, opt.param_groups[0])
    assert {"step", "exp_avg", "exp_avg_sq", "master"} <= set(opt.state[p])


def checkpoint(n=5, value=0.25, cls=torch.optim.AdamW, **settings):
    q = torch.nn.Parameter(torch.zeros(n))
    theirs = cls([q], **settings)
    q.grad = torch.ones(n)
    theirs.step()
    saved = theirs.state_dict()
    saved["state"][0]["exp_avg"] = torch.full((n,), value)
    return saved


def test_load_hooks_see_and_change_the_states():
    opt = fm.AdamW([torch.nn.Parameter(torch.zeros(5))])
    p, seen = opt.param_groups[0]["params"][0], []

    def before(o, state_dict):
        seen.append(len(state_dict["state"]))
        state = {k: {**v, "exp_avg": 2 * v["exp_avg"]} for k, v in state_dict["state"].items()}
        return {**state_dict, "state": state}

    def after(o):
        seen.append((o is opt, float(o.state[p]["exp_avg"][0]), o.param_groups[0]["state_bits"]))

    handles = [opt.register_load_state_dict_pre_hook(before), opt.register_load_state_dict_post_hook(after)]
    opt.load_state_dict(checkpoint())
    assert seen == [1, (True, 0.5, 32)] and (opt.state[p]["exp_avg"] == 0.5).all()
    for handle in handles:
        handle.remove()
    opt.load_state_dict(checkpoint(value=3.0))               # nothing of the first load stays registered
    assert (opt.state[p]["exp_avg"] == 3.0).all() and len(seen) == 2


def test_a_refused_checkpoint_changes_nothing():
    opt = fm.AdamW([torch.nn.Parameter(torch.zeros(5))], lr=0.5)
    p = opt.param_groups[0]["params"][0]
    opt.load_state_dict(checkpoint(lr=0.125))
    keep = opt.state[p]
    with pytest.raises(ValueError, match="size"):
        opt.load_state_dict(checkpoint(n=6))
    with pytest.raises(ValueError, match="maximize"):
        opt.load_state_dict(checkpoint(maximize=True, lr=0.75))
    assert opt.state[p] is keep and opt.param_groups[0]["lr"] == 0.125
    opt.load_state_dict(checkpoint(value=1.0))
    assert (opt.state[p]["exp_avg"] == 1.0).all()


def test_a_learning_rate_on_the_device_loads_as_a_float():
    """Where this optimizer's own is one; the checkpoint's tensor may lie anywhere."""
    opt = fm.AdamW([torch.nn.Parameter(torch.zeros(5))], lr=0.5)
    saved = checkpoint()
    saved["param_groups"][0]["lr"] = torch.tensor(0.125)
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 0.125 and isinstance(opt.param_groups[0]["lr"], float)


def test_checkpoints_of_adam():
    """Its weight decay is another; without one it is the same optimizer."""
    opt = fm.AdamW([torch.nn.Parameter(torch.zeros(5))], lr=0.5)
    with pytest.raises(ValueError, match="Adam"):
        opt.load_state_dict(checkpoint(cls=torch.optim.Adam, weight_decay=0.1))
    assert not opt.state and opt.param_groups[0]["lr"] == 0.5
    opt.load_state_dict(checkpoint(cls=torch.optim.Adam, weight_decay=0.0))
    assert opt.param_groups[0]["weight_decay"] == 0.0 and len(opt.state) == 1
    opt.param_groups[0]["weight_decay"] = 0.1                # decoupled from here on: its own checkpoint loads
    saved = opt.state_dict()
    fm.AdamW([torch.nn.Parameter(torch.zeros(5))]).load_state_dict(saved)
    opt.load_state_dict(checkpoint(weight_decay=0.25))
    assert opt.param_groups[0]["weight_decay"] == 0.25


def test_a_learning_rate_on_the_host_is_refused_at_once():
    """As the step does, where it would come too late."""
    new = lambda: [torch.nn.Parameter(torch.zeros(5))]  # noqa: E731
    with pytest.raises(AssertionError, match="`lr` must be"):
        fm.AdamW(new(), lr=torch.tensor(0.1))
    opt = fm.AdamW(new())
    with pytest.raises(AssertionError, match="`lr` must be"):
        opt.add_param_group(dict(params=new(), lr=torch.tensor(0.1)))
    assert len(opt.param_groups) == 1

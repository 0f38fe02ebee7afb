"""What AdamW, its 8-bit states and the clipping promise besides the step itself."""
import pytest
import torch

import flash_muon_b200 as fm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = torch.float32


@pytest.mark.parametrize("moment", [1, 2])
@pytest.mark.parametrize("b", [0, 1, 5, 16, 17, 31, 32, 127, 253, 254, 255])
def test_values_do_not_depend_on_where_a_block_lies(b, moment):
    """A whole block and the same codes in a last block that is not whole take different code paths."""
    for codes in range(0, 256, 32):
        codes = torch.arange(codes, codes + 32, dtype=torch.uint8, device=DEV)
        scales = torch.full((1,), b, dtype=torch.uint8, device=DEV)
        whole = fm.adamw8_values(codes, scales, moment=moment, dtype=F32)
        part = fm.adamw8_values(codes, scales, moment=moment, numel=31, dtype=F32)
        assert torch.equal(whole[:31].isnan(), part.isnan())
        assert torch.equal(whole[:31].nan_to_num(nan=7.0), part.nan_to_num(nan=7.0))


@pytest.mark.parametrize("n", [100, 5000])
@pytest.mark.parametrize("eps", [1e-37, 2e-38, 1e-40, 1e-60])
def test_any_positive_eps_keeps_the_division_by_zero_away(n, eps):
    """eps sqrt(1 - b2^t) is 3e-39 and less here, no normal number.  Elements without gradient have a zero
    update; beside the root of any other second moment, 4e-23 at least, such an eps vanishes."""
    g = torch.zeros(n, device=DEV)
    g[::3] = torch.linspace(-1, 1, len(g[::3]), device=DEV) + 0.01
    out = []
    for e in (eps, 0.0):
        p, m, v, steps = torch.ones(n, device=DEV), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), torch.zeros(1, device=DEV)
        for _ in range(2):
            fm.adamw_step([p], [g], [m], [v], steps, lr=0.1, weight_decay=0.0, eps=e)
        out.append(p)
    assert (out[0][g == 0] == 1).all()
    assert torch.equal(out[0][g != 0], out[1][g != 0]) and out[0].isfinite().all()


def test_out_of_memory_is_torch_s_own_error():
    """The allocator's limit for this process is lowered; the device has memory left."""
    codes, scales = torch.zeros(1 << 28, dtype=torch.uint8, device=DEV), torch.zeros(1 << 23, dtype=torch.uint8, device=DEV)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(DEV).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (64 << 20)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            fm.adamw8_values(codes, scales, moment=1, dtype=F32)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert fm.adamw8_values(codes, scales, moment=1, numel=100, dtype=F32).numel() == 100

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

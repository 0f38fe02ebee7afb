"""The norm's one-launch form (a cluster of eight blocks) with as little work as there is, over and over,
alone and while other work holds most of the SMs: seven blocks have nothing to load and reach the exchange
of the partial sums at once."""
import pytest
import torch

import flash_muon_b200 as fm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("busy", [False, True], ids=["alone", "beside"])
@pytest.mark.parametrize("sizes", [[1], [1000], [1] * 9], ids=["one", "unit", "nine"])
def test_small_norms_over_and_over(sizes, busy):
    reps = 2000
    grads = [[torch.full((n,), float(k % 97 + 1), device=DEV) for n in sizes] for k in range(97)]
    noise = torch.randn(4096, 4096, device=DEV)
    side = torch.cuda.Stream()
    got = []
    torch.cuda.synchronize()
    for k in range(reps):
        if busy and k % 10 == 0:
            with torch.cuda.stream(side):
                noise.mul_(1.0)
        got.append(fm.grad_norm(grads[k % 97], 1.0)[0])
    torch.cuda.synchronize()
    # every element is k + 1: a sum of equal squares, exact in 64 bits and within half an ulp after the root
    want = torch.tensor([float(k % 97 + 1) for k in range(reps)], dtype=torch.float64) * sum(sizes) ** 0.5
    off = (torch.stack(got).double().cpu() / want - 1).abs()
    assert float(off.max()) <= 17 * 2.0 ** -24, off.argmax()

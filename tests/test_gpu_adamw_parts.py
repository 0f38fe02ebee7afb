"""AdamW with 8-bit states where a block takes several parts of a tensor, one after the other through the same
shared memory: bit for bit what small calls give, which test_gpu_adamw.py compares with the definition.

A block takes parts of 2048 elements, as many (up to 8) as leave every SM 12 blocks, so the number depends
on all elements of the kind in the call: a tensor stepped alone takes one part per block, beside a large one
several."""
import pytest
import torch

import flash_muon_b200 as fm
from test_gpu_adamw import DEV, HYPER, IDS, KINDS, encode_state, random_state

pytestmark = pytest.mark.gpu
PART = 2048


def buffers(s):
    return [s[k] for k in ("p", "g", "m", "ms", "v", "vs", "w") if s.get(k) is not None]


@pytest.mark.parametrize("parts", [3, 5, 8])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_several_parts_per_block(kind, offset, parts):
    p_dtype, g_dtype, master = kind
    # two whole tiles, then one whose last part is whole, and one with a remainder, which is not a multiple of 32
    sizes = [2 * parts * PART, 3 * parts * PART - PART, 2 * parts * PART + 2 * PART + 777]
    per_part = PART * 12 * torch.cuda.get_device_properties(DEV).multi_processor_count + 1
    rest = parts * per_part - sum(sizes)
    assert (sum(sizes) + rest) // per_part == parts and max(sizes) < per_part
    alone, beside = ([s for s in random_state(sizes, p_dtype, g_dtype, master, offset, 4)] for _ in range(2))
    for s in alone + beside:
        encode_state(s)
    byte, blocks = torch.uint8, -(-rest // 32)
    filler = dict(p=torch.zeros(rest, dtype=p_dtype, device=DEV), g=torch.ones(rest, dtype=g_dtype, device=DEV),
                  m=torch.zeros(32 * blocks, dtype=byte, device=DEV), v=torch.zeros(32 * blocks, dtype=byte, device=DEV),
                  ms=torch.zeros(blocks, dtype=byte, device=DEV), vs=torch.zeros(blocks, dtype=byte, device=DEV),
                  w=torch.zeros(rest, device=DEV) if master else None)
    counts = [torch.full((), 5.0, device=DEV) for _ in range(2 * len(sizes) + 1)]
    scale = torch.tensor(0.75, device=DEV)

    def step(tensors, counts, seeds):
        fm.adamw8_step(*([t[k] for t in tensors] for k in ("p", "g", "m", "ms", "v", "vs")), counts, seeds=seeds,
                       masters=[t["w"] for t in tensors] if master else None, grad_scale=scale, **HYPER)

    views = lambda ss: [{k: x.t if x is not None else None for k, x in s.items()} for s in ss]  # noqa: E731
    for k in range(3):
        for i, t in enumerate(views(alone)):
            step([t], [counts[i]], [i + 9])
        a, b, c = views(beside)
        step([a, filler, b, c], [counts[3], counts[6], counts[4], counts[5]], [9, 77, 10, 11])
        for x, y in zip(alone, beside):
            for u, v in zip(buffers(x), buffers(y)):
                assert torch.equal(u.t.view(torch.uint8), v.t.view(torch.uint8))
                v.check()
        if k == 0:  # equal elements take equal first steps: moments enter before they are rounded at random
            assert (filler["p"] == filler["p"][0]).all() and -0.1 < float(filler["p"][0]) < 0
    assert all(float(c) == 8.0 for c in counts) and filler["p"].isfinite().all()

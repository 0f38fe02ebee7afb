"""AdamW with 8-bit states where a block takes several parts of a tensor, one after the other through the same
shared memory, and calls of many kinds of tensors: bit for bit what small calls of one kind give, which
test_gpu_adamw.py compares with the definition.

A block takes parts of 2048 elements, as many (up to 8) as leave every SM 12 blocks, so the number depends
on all elements of the kind in the call: a tensor stepped alone takes one part per block, beside a large one
several."""
from array import array

import pytest
import torch

import flash_muon_b200 as fm
from flash_muon_b200 import _lib
from flash_muon_b200._lib import AdamWGroup, check, lib
from test_gpu_adamw import DEV, F32, HYPER, IDS, KINDS, encode_state, random_state

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


def c_group(states, counts, kind, bits, settings, seeds):
    """An fm_adamw_group over the tensors, and what has to outlive the call."""
    p_dtype, g_dtype, master = kind
    g, keep = AdamWGroup(), []

    def put(name, tensors):
        keep.append(array("Q", [t.data_ptr() for t in tensors]))
        setattr(g, name, keep[-1].buffer_info()[0])

    for name, k in (("params", "p"), ("grads", "g"), ("exp_avg", "m"), ("exp_avg_sq", "v")):
        put(name, [s[k].t for s in states])
    if master:
        put("masters", [s["w"].t for s in states])
    if bits == 8:
        put("exp_avg_scale", [s["ms"].t for s in states])
        put("exp_avg_sq_scale", [s["vs"].t for s in states])
        keep.append(array("I", seeds))
        g.seeds = keep[-1].buffer_info()[0]
    put("steps", counts)
    keep.append(array("q", [s["p"].n for s in states]))
    g.numels = keep[-1].buffer_info()[0]
    g.count, g.state_bits = len(states), bits
    g.p_dtype, g.g_dtype = _lib.dtype_code(p_dtype), _lib.dtype_code(g_dtype)
    g.lr, g.beta1, g.beta2, g.eps, g.weight_decay = settings
    return g, keep


@pytest.mark.parametrize("sizes", [(33, 5000), (33, 4096)], ids=["tiled", "whole"])
def test_groups_of_all_kinds_and_widths_in_one_c_call(sizes):
    """Two groups of every kind with settings of their own, mixed gradient types and both widths among them:
    each as a call of its own."""
    kinds = [(kind, bits) for kind in KINDS for bits in (32, 8)] * 2
    sides = []
    for _ in range(2):
        groups = []
        for i, (kind, bits) in enumerate(kinds):
            states = random_state(sizes, *kind, 0, 50 + i)
            if bits == 8:
                for s in states:
                    encode_state(s)
            groups.append((states, [torch.full((), float(i), device=DEV) for _ in sizes]))
        sides.append(groups)
    made = [[c_group(states, counts, kind, bits, (1e-3 * (i + 1), 0.5 + 0.01 * i, 0.9 + 0.002 * i, 1e-8 * (i + 1), 0.01 * i),
                     [100 * i + 1, 100 * i + 2])
             for i, ((states, counts), (kind, bits)) in enumerate(zip(groups, kinds))] for groups in sides]
    stream = torch.cuda.current_stream().cuda_stream
    table = (AdamWGroup * len(kinds))(*[g for g, _ in made[0]])
    for _ in range(2):
        check(lib.fm_adamw_step(table, len(kinds), None, stream))
        for g, _ in made[1]:
            check(lib.fm_adamw_step(g, 1, None, stream))
    for i, ((one, c1), (many, c2)) in enumerate(zip(*sides)):
        assert [float(c) for c in c1 + c2] == [i + 2.0] * 4
        for x, y in zip(one, many):
            for u, v in zip(buffers(x), buffers(y)):
                assert torch.equal(u.t.view(torch.uint8), v.t.view(torch.uint8)), i
                u.check()


def test_optimizer_groups_of_both_widths():
    """One optimizer of many groups against one per group, weights, moments and codes bit for bit; a parameter's
    seed is its group's plus its place among all parameters."""
    def make(split):
        torch.manual_seed(0)
        groups = [dict(params=[torch.nn.Parameter(torch.randn(n, device=DEV).to(pd)) for n in (33, 5000)], lr=1e-3 * (i + 1),
                       weight_decay=0.01 * i, master_weights=master, state_bits=8 if i % 2 else 32, min_8bit_numel=0,
                       seed=100 * i + (2 * i if split else 0))
                  for i, (pd, _, master) in enumerate(KINDS * 2)]
        for g in groups:
            for p in g["params"]:
                p.grad = torch.randn_like(p)
        return [fm.AdamW([g]) for g in groups] if split else [fm.AdamW(groups)]

    one, many = make(False), make(True)
    for _ in range(3):
        for opt in one + many:
            opt.step()
    for a, opt in zip(one[0].param_groups, many):
        for p, q in zip(a["params"], opt.param_groups[0]["params"]):
            assert torch.equal(p, q)
            x, y = one[0].state[p], opt.state[q]
            assert set(x) == set(y) and all(torch.equal(x[k], y[k]) for k in x) and float(x["step"]) == 3.0
            assert x["exp_avg"].dtype == (torch.uint8 if a["state_bits"] == 8 else F32)

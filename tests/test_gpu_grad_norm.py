"""The norm over many gradients and the scaling by it, against 64 bits.

Tolerance of the norm (u = 2^-24): a thread adds at most 36 squares of a chunk in fp32 with fused
multiply-adds, each within 1 u of a partial sum of positive numbers, so the sum is within 36 u, in the
worst case; everything after that is 64 bits; the root halves it and is rounded once: 19 u.  The
factor adds the sum with 1e-6, the division and the minimum: 22 u."""
import math

import pytest
import torch

import flash_muon_b200 as fm
from flash_muon_b200._lib import FlashMuonError
from oracle import adamw_oracle as A

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
B16, H16, F32 = torch.bfloat16, torch.float16, torch.float32


def tensors(sizes, dtypes, offset=0, seed=0, size=1e-2):
    r = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        buf = torch.full((n + offset + 9,), 100.0, device=DEV, dtype=dt)   # what lies around is not counted
        buf[offset:offset + n] = (torch.randn(n, device=DEV, generator=r) * size).to(dt)
        out.append(buf[offset:offset + n])
    return out


@pytest.mark.parametrize("dtypes", [[B16], [H16], [F32], [B16, F32, H16]], ids=["bf16", "f16", "f32", "mixed"])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("sizes", [[1], [7, 0, 33], [8191, 8192, 8193, 100000], [3] * 200, [500_003], [65] * 2500,
                                   [1024] * 255 + [1000], [1024] * 255 + [1025], [1] * 256, [1] * 257, [1023, 1024, 1025, 70_000]],
                         ids=["one", "few", "chunks", "vectors", "long", "tables", "cluster", "past-cluster", "ones", "past-ones", "units"])
def test_norm_against_64_bits(dtypes, offset, sizes):
    g = tensors(sizes, dtypes, offset, len(sizes))
    keep = [x.clone() for x in g]
    norm, scale = fm.grad_norm(g, 0.01)
    want, factor = A.grad_norm(g, 0.01)
    assert norm.dtype == scale.dtype == F32 and norm.dim() == scale.dim() == 0
    assert abs(float(norm) / want - 1) <= 19 * U
    assert abs(float(scale) / factor - 1) <= 22 * U
    again = fm.grad_norm(g, 0.01)
    assert torch.equal(again[0], norm) and torch.equal(again[1], scale)
    assert all(torch.equal(a, b) for a, b in zip(g, keep))
    assert float(fm.grad_norm(g)[1]) == 1.0               # no limit


def test_norm_limits():
    zero = [torch.zeros(100, device=DEV, dtype=B16), torch.zeros(0, device=DEV)]
    norm, scale = fm.grad_norm(zero, 1.0)
    assert float(norm) == 0.0 and float(scale) == 1.0
    assert [float(x) for x in fm.grad_norm([zero[1]], 1.0)] == [0.0, 1.0]
    one = [torch.full((5,), 1.0, device=DEV)]
    assert float(fm.grad_norm(one, 0.0)[1]) == 0.0
    for bad in (math.nan, math.inf, 1e25):                # 1e25 squared is infinite in fp32
        g = torch.ones(20000, device=DEV)
        g[777] = bad
        norm, scale = fm.grad_norm([g, one[0]], 1.0)
        assert not math.isfinite(float(norm)) and math.isnan(float(scale))
    tiny = [torch.full((1000,), 2.0 ** -70, device=DEV)]  # squares are subnormal: a multiple of 2^-149
    assert abs(float(fm.grad_norm(tiny)[0]) / (2.0 ** -70 * math.sqrt(1000)) - 1) <= 1e-2


@pytest.mark.parametrize("dtypes", [[B16], [H16], [F32], [B16, F32, H16]], ids=["bf16", "f16", "f32", "mixed"])
@pytest.mark.parametrize("offset", [0, 1])
def test_clip_in_place(dtypes, offset):
    sizes = [1, 0, 33, 8192, 8193, 70000] + [5] * 100
    values = tensors(sizes, dtypes, offset, 3)
    params = []
    for v in values:
        p = torch.nn.Parameter(torch.empty_like(v))
        p.grad = v
        params.append(p)
    params.append(torch.nn.Parameter(torch.zeros(3, device=DEV)))        # has no gradient
    raw = [v.clone() for v in values]
    want, factor = A.grad_norm(raw, 0.5)
    norm = fm.clip_grad_norm_(params, 0.5)
    assert abs(float(norm) / want - 1) <= 19 * U
    for v, r in zip(values, raw):
        exact = r.double() * factor
        fi = torch.finfo(v.dtype)
        # rounding to the type, from a product that is off by the factor's 22 u and its own
        bound = exact.abs() * (fi.eps / 2 + 24 * U) + fi.tiny * fi.eps / 2
        assert ((v.double() - exact).abs() <= bound).all()
    clipped = [v.clone() for v in values]
    fm.clip_grad_norm_(params, 2.0 * want)                               # within: not touched
    assert all(torch.equal(a, b) for a, b in zip(values, clipped))
    values[5][123] = math.nan
    assert math.isnan(float(fm.clip_grad_norm_(params, 1.0)))
    assert all(v.isnan().all() for v in values)


def test_the_same_gradient_twice():
    """Counted twice by the norm, which only reads; refused where it would be scaled twice."""
    p = torch.nn.Parameter(torch.zeros(4, device=DEV))
    p.grad = torch.full((4,), 3.0, device=DEV)
    assert float(fm.grad_norm([p.grad, p.grad])[0]) == pytest.approx(math.sqrt(72.0), rel=1e-6)
    with pytest.raises(FlashMuonError, match="overlap"):
        fm.clip_grad_norm_([p, p], 1.0)
    assert (p.grad == 3.0).all()


def test_iterables_and_single_parameters():
    p = torch.nn.Parameter(torch.zeros(4, device=DEV))
    p.grad = torch.full((4,), 3.0, device=DEV)
    assert float(fm.clip_grad_norm_(iter([p]), 3.0)) == 6.0
    assert float(fm.clip_grad_norm_(p, 100.0)) == pytest.approx(3.0, rel=1e-6)


def test_norm_on_two_streams_at_once():
    """Calls on different streams share no scratch."""
    a, b = tensors([3_000_000] * 4, [B16], seed=1), tensors([2_000_000] * 5, [F32], seed=2)
    want = [fm.grad_norm(x, 1.0)[0].clone() for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(fm.grad_norm(x, 1.0)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])

"""The AdamW step (32-bit and 8-bit states) on the GPU against the 64-bit definition, one step at a
time: the definition takes the state that the kernel's step took, so the tolerances below count the
roundings of a single step.

Tolerances (u = 2^-24, half a step of fp32; every fp32 operation is off by at most u relative, the
sum of the fused multiply-adds too):
  m = fma(b1, m, o1 g'), with 32-bit states g' = s g rounded (1 u), o1 = 1 - b1 rounded (1 u), o1 g' (1 u),
  b1 rounded (1 u), the fma (1 u); with 8-bit states o1 s is one constant (2 u) times g (1 u): the same.
  |dm| <= u (2 |b1 m| + 4 |o1 g'|).
  v, with 32-bit states fma(b2, v, o2 (g' g')): g' g' carries 2 u of g' and 1 u of its own, o2 1 u, the
  product 1 u, the fma 1 u: 6 u of that part, 2 u of b2 v.  With 8-bit states fma(h, h, b2 v) with
  h = (sqrt(o2) s) g: the root rounded (1 u), times s (1 u), times g (1 u), squared: 6 u; b2 v 2 u; the fma 1 u.
  |dv| <= 7 u v either way.
  The update is x = size m / (sqrt(v) + e), size = lr / (1 - b1^t) sqrt(1 - b2^t), e = eps sqrt(1 - b2^t).
  sqrt(1 - b2^t): rounded, root, 1.5 u.  size: lr, 1 - b1^t, quotient, times the root, 5.5 u.  e: 1 + 1.5 + 1 u.
  sqrt(v): 3.5 u from v, 2 u for the approximate root (1 ulp); the sum 1 u.  Reciprocal 2 u, two products 2 u:
  |dx| <= (5.5 + 6.5 + 4) u |x| + |dm / m| |x|, and 20 u is asserted for the 16.
  w = fma(w, decay, -x): decay 1 u, fma 1 u: 2 u (|w| + |x|).
  A stored 16-bit parameter adds half its step, eps / 2 relative (or half the smallest subnormal).
"""
import ctypes
import math

import pytest
import torch

import flash_muon_b200 as fm
from flash_muon_b200 import _lib
from flash_muon_b200._lib import FlashMuonError
from oracle import adamw_oracle as A
from oracle import muon_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
B16, H16, F32 = torch.bfloat16, torch.float16, torch.float32
KINDS = [(B16, B16, False), (B16, F32, False), (H16, H16, False), (H16, F32, False), (F32, F32, False),
         (F32, B16, False), (F32, H16, False), (B16, B16, True), (B16, F32, True), (H16, H16, True), (H16, F32, True)]
IDS = [f"{str(p)[6:]}-{str(g)[6:]}{'-master' if w else ''}" for p, g, w in KINDS]
# the first list has tensors of several blocks, in the others a block takes each tensor whole
SIZES = {"several": [1, 3, 16, 31, 32, 33, 255, 1000, 4095, 4096, 4097, 8192 + 17, 20000],
         "whole": [1, 31, 32, 33, 1000, 2047, 2048, 2049, 4095, 4096], "one": [1000], "least": [4097], "short": [33, 8191, 8192]}
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Guarded:
    """A tensor inside a larger allocation whose other elements must stay as they are."""

    def __init__(self, value, offset=0, tail=40):
        self.n, self.offset = value.numel(), offset
        fill = 77 if value.dtype == torch.uint8 else 3.0
        self.buf = torch.full((offset + value.numel() + tail,), fill, dtype=value.dtype, device=DEV)
        self.t = self.buf[offset:offset + self.n]
        self.t.copy_(value)
        self.fill = fill

    def check(self):
        assert (self.buf[:self.offset] == self.fill).all() and (self.buf[self.offset + self.n:] == self.fill).all()


def random_state(sizes, p_dtype, g_dtype, master, offset, seed, grad_size=1e-3):
    r = gen(seed)
    out = []
    for n in sizes:
        g = (torch.randn(n, device=DEV, generator=r) * grad_size * 10 ** (2 * torch.rand(n, device=DEV, generator=r) - 1)).to(g_dtype)
        w = torch.randn(n, device=DEV, generator=r) * 0.05
        p = w.to(p_dtype)
        m = torch.randn(n, device=DEV, generator=r) * grad_size * 0.3
        v = (grad_size * torch.rand(n, device=DEV, generator=r)) ** 2
        out.append(dict(p=Guarded(p, offset), g=Guarded(g, offset), m=Guarded(m, offset), v=Guarded(v, offset),
                        w=Guarded(p.float() * (1 + 1e-4 * torch.randn(n, device=DEV, generator=r)), offset) if master else None))
    return out


def tolerances(w0, g, m0, v0, w1, scale, t, hyper):
    """Bounds on what the kernel's m, v and w may be off, from the docstring."""
    b1, b2 = hyper["betas"]
    gs = g.double().abs() * abs(scale)
    m0, v0, w0 = m0.double().abs(), v0.double().abs(), w0.double().abs()
    dm = U * (2 * b1 * m0 + 4 * (1 - b1) * gs) * 1.001 + 2.0 ** -149
    v = b2 * v0 + (1 - b2) * gs ** 2
    dv = 7 * U * v * 1.001 + 2 * 2.0 ** -149
    size = hyper["lr"] / (1 - b1 ** t)
    den = v.sqrt() / math.sqrt(1 - b2 ** t) + hyper["eps"]
    x = size * (b1 * m0 + (1 - b1) * gs) / den          # at least |x|
    dx = 20 * U * x + size * dm / den
    dw = 2 * U * (w0 + x) + dx
    return dm, dv, dw * 1.001


def half_step(x, dtype):
    fi = torch.finfo(dtype)
    return torch.maximum(x.double().abs() * (fi.eps / 2), torch.tensor(fi.tiny * fi.eps / 2, dtype=torch.float64))


def check_weights(s, w64, dw, p_dtype):
    w = s["w"].t if s["w"] is not None else None
    if w is not None:
        assert ((w.double().cpu() - w64).abs() <= dw).all()
        assert torch.equal(s["p"].t, w.to(p_dtype))      # the parameter is the master, rounded
    else:
        off = (s["p"].t.double().cpu() - w64).abs()
        bound = dw + (0 if p_dtype == F32 else half_step(w64, p_dtype) + 0)
        assert (off <= bound).all(), float((off - bound).max())


# ---------------------------------------------------------------- 32 bits
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES)
def test_step_against_64_bits(kind, offset, sizes):
    p_dtype, g_dtype, master = kind
    states = random_state(sizes, p_dtype, g_dtype, master, offset, 1)
    start = [0.0 if i % 2 else 137.0 for i in range(len(sizes))]
    steps = torch.tensor(start, device=DEV)
    for k in range(1, 4):
        before = [{x: s[x].t.clone().cpu() for x in "gmv"} | {"w": (s["w"] or s["p"]).t.clone().cpu()} for s in states]
        grads_before = [s["g"].t.clone() for s in states]
        fm.adamw_step([s["p"].t for s in states], [s["g"].t for s in states], [s["m"].t for s in states],
                      [s["v"].t for s in states], steps, masters=[s["w"].t for s in states] if master else None, **HYPER)
        assert steps.tolist() == [t + k for t in start]
        for s, b, t, g0 in zip(states, before, start, grads_before):
            w, m, v = A.adamw(b["w"], b["g"], b["m"], b["v"], int(t) + k, **HYPER)
            dm, dv, dw = tolerances(b["w"], b["g"], b["m"], b["v"], w, 1.0, int(t) + k, HYPER)
            assert ((s["m"].t.double().cpu() - m).abs() <= dm).all()
            assert ((s["v"].t.double().cpu() - v).abs() <= dv).all()
            check_weights(s, w, dw, p_dtype)
            assert torch.equal(s["g"].t, g0)
            for x in s.values():
                if x is not None:
                    x.check()


def test_first_steps_equal_the_definition_in_closed_form():
    """From zero moments the first step moves by lr * g / (|g| + eps) whatever the gradient's size."""
    g = torch.tensor([1e-6, -1e-3, 1.0, -1e4, 0.0], device=DEV)
    p = torch.zeros(5, device=DEV)
    m, v, steps = torch.zeros(5, device=DEV), torch.zeros(5, device=DEV), torch.zeros(1, device=DEV)
    fm.adamw_step([p], [g], [m], [v], steps, lr=0.5, weight_decay=0.0)
    want = -0.5 * g.double() / (g.double().abs() + 1e-8)
    assert torch.allclose(p.double(), want, rtol=30 * U, atol=0)


def test_scale_lr_tensor_and_steps_list():
    states = random_state([700, 5000], F32, F32, False, 0, 3)
    other = random_state([700, 5000], F32, F32, False, 0, 3)
    args = lambda ss: ([s["p"].t for s in ss], [s["g"].t for s in ss], [s["m"].t for s in ss], [s["v"].t for s in ss])  # noqa: E731
    scale = torch.tensor(0.25, device=DEV)
    fm.adamw_step(*args(states), torch.zeros(2, device=DEV), grad_scale=scale, **HYPER)
    for s in other:
        s["g"].t.mul_(0.25)                              # exact
    counts = [torch.zeros((), device=DEV), torch.zeros(1, device=DEV)]
    fm.adamw_step(*args(other), counts, **{**HYPER, "lr": torch.tensor(HYPER["lr"], device=DEV, dtype=F32)})
    assert [float(c) for c in counts] == [1.0, 1.0]
    for s, o in zip(states, other):
        assert torch.equal(s["m"].t, o["m"].t) and torch.equal(s["v"].t, o["v"].t)
        # lr as a float has 64 bits, as a device scalar 32: the update may differ by 1 u of lr
        assert torch.allclose(s["p"].t, o["p"].t, rtol=2 * U, atol=3 * U * 0.1)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [3000, 70000])
def test_a_factor_that_is_not_finite_takes_no_step(bad, bits, n):
    p, g = torch.randn(n, device=DEV), torch.randn(n, device=DEV)
    steps = torch.tensor([4.0], device=DEV)
    scale = torch.tensor(bad, device=DEV)
    if bits == 32:
        st = [torch.randn(n, device=DEV), torch.rand(n, device=DEV)]
        call = lambda: fm.adamw_step([p], [g], [st[0]], [st[1]], steps, lr=0.1, grad_scale=scale)  # noqa: E731
    else:
        st = [*fm.adamw8_encode(torch.randn(n, device=DEV), moment=1), *fm.adamw8_encode(torch.rand(n, device=DEV), moment=2)]
        call = lambda: fm.adamw8_step([p], [g], *[[x] for x in st], steps, lr=0.1, grad_scale=scale)  # noqa: E731
    before = [x.clone() for x in (p, g, steps, *st)]
    call()
    assert all(torch.equal(a, b) for a, b in zip(before, (p, g, steps, *st)))


@pytest.mark.parametrize("n", [4096, 12000])
def test_nan_and_inf_gradients_stay_where_they_are(n):
    p, g = torch.randn(n, device=DEV), torch.randn(n, device=DEV)
    g[7], g[4090] = math.nan, math.inf
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    fm.adamw_step([p], [g], [m], [v], torch.zeros(1, device=DEV), lr=0.1)
    ok = torch.ones(n, dtype=torch.bool, device=DEV)
    ok[7] = ok[4090] = False
    assert p[ok].isfinite().all() and m[ok].isfinite().all() and v[ok].isfinite().all()
    assert p[~ok].isnan().all() and math.isinf(m[4090]) and math.isinf(v[4090]) and math.isnan(m[7])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count, largest", [(24, 9000), (25, 9000), (96, 9000), (97, 100), (360, 9000), (361, 100), (1000, 9000)])
def test_tables_of_all_lengths_and_empty_tensors(bits, count, largest):
    """Up to 1000 tensors, empty ones among them, equal one call per tensor bit for bit."""
    r = gen(5)
    sizes = [(i * 37) % 131 if i % 10 else 0 for i in range(count)]
    sizes[count // 2] = largest
    p = [torch.randn(n, device=DEV, generator=r) for n in sizes]
    g = [torch.randn(n, device=DEV, generator=r) for n in sizes]
    q = [x.clone() for x in p]
    steps, again = torch.zeros(count, device=DEV), torch.zeros(count, device=DEV)

    def states():
        if bits == 32:
            return [[torch.zeros(n, device=DEV) for n in sizes] for _ in range(2)]
        return [[torch.zeros(-(-n // 32) * k, dtype=torch.uint8, device=DEV) for n in sizes] for k in (32, 1, 32, 1)]

    step = fm.adamw_step if bits == 32 else fm.adamw8_step
    a, b = states(), states()
    for _ in range(2):
        step(p, g, *a, steps, lr=0.1, **({} if bits == 32 else {"seeds": 50}))
        for i in range(count):
            step([q[i]], [g[i]], *[[x[i]] for x in b], again[i:i + 1], lr=0.1, **({} if bits == 32 else {"seeds": [50 + i]}))
    assert (steps == 2).all() and (again == 2).all()
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    for xs, ys in zip(a, b):
        assert all(torch.equal(x, y) for x, y in zip(xs, ys))


@pytest.mark.parametrize("n", [500, 9000])
def test_many_groups_of_one_kind(n):
    """More groups than one launch holds, each with its own settings."""
    make = lambda: [torch.nn.Parameter(torch.linspace(-1, 1, n, device=DEV)) for _ in range(20)]  # noqa: E731
    ps, qs = make(), make()
    a = fm.AdamW([dict(params=[p], lr=0.01 * (i + 1), betas=(0.5 + 0.02 * i, 0.9), eps=1e-8 * (i + 1), weight_decay=0.05 * i)
                  for i, p in enumerate(ps)])
    b = [fm.AdamW([q], **{k: g[k] for k in ("lr", "betas", "eps", "weight_decay")}) for q, g in zip(qs, a.param_groups)]
    for p, q in zip(ps, qs):
        p.grad = torch.randn(n, device=DEV)
        q.grad = p.grad.clone()
    for _ in range(2):
        a.step()
        for opt in b:
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert len({float(p.detach()[0]) for p in ps}) == 20


def test_groups_of_all_kinds_in_one_call():
    """More groups than one launch holds, of every kind: each as if alone."""
    opts = []
    for together in (True, False):
        torch.manual_seed(0)
        groups = []
        for i, (pd, _, master) in enumerate(KINDS * 2):
            ps = [torch.nn.Parameter(torch.randn(n, device=DEV).to(pd)) for n in (33, 5000)]
            groups.append(dict(params=ps, lr=1e-3 * (i + 1), weight_decay=0.01 * i, master_weights=master,
                               state_bits=8 if i % 3 == 0 else 32, min_8bit_numel=0, seed=100 * i))
        opts.append([fm.AdamW(groups)] if together else [fm.AdamW([g]) for g in groups])
    for opt_list in opts:
        torch.manual_seed(1)
        gi = 0
        for opt in opt_list:
            for group in opt.param_groups:
                for p in group["params"]:
                    p.grad = torch.randn_like(p)
                gi += 1
        for _ in range(3):
            for opt in opt_list:
                opt.step()
    one, many = opts[0][0].param_groups, [o.param_groups[0] for o in opts[1]]
    for i, (x, y) in enumerate(zip(one, many)):
        for p, q in zip(x["params"], y["params"]):
            if x["state_bits"] == 32:                    # (positions enter the random numbers)
                assert torch.equal(p, q)
            sp, sq = opts[0][0].state[p], opts[1][i].state[q]
            assert float(sp["step"]) == float(sq["step"]) == 3.0
            assert set(sp) == set(sq)


# ---------------------------------------------------------------- 8 bits
def encode_state(s):
    """8-bit states near the float ones, with guards; padding zero."""
    for k, moment in (("m", 1), ("v", 2)):
        codes, scales = fm.adamw8_encode(s[k].t.clone(), moment=moment)
        s[k] = Guarded(codes, 16, 48)
        s[k + "s"] = Guarded(scales, 3, 5)


def check_codes(got, got_scales, x, dx, u, moment):
    """Codes of the kernel against the definition's rounding of x (float64, padded) with its random numbers
    u; x itself may be off by dx."""
    want_lo = A.block_scales((x.abs() - dx).clamp(min=0), moment)
    want_hi = A.block_scales(x.abs() + dx, moment)
    scales = got_scales.cpu().long()
    assert ((scales >= want_lo) & (scales <= want_hi)).all()
    pos = lambda y: torch.floor(A.rounding_position(y, scales, moment) + u)  # noqa: E731
    # the random number is added in fp32 below the code's last bit: 2^-20 of a step more
    lo = torch.floor(A.rounding_position((x.abs() - dx).clamp(min=0), scales, moment) + u - 2.0 ** -19)
    hi = torch.floor(A.rounding_position(x.abs() + dx, scales, moment) + u + 2.0 ** -19)
    codes = got.cpu().long()
    mag = codes & 127 if moment == 1 else codes
    if moment == 2:
        lo, hi = torch.where(x > 0, lo.clamp(min=1), lo), torch.where(x > 0, hi.clamp(min=1), hi)
    assert ((mag >= lo) & (mag <= hi)).all(), (mag - lo).abs().max()
    if moment == 1:
        assert ((codes >= 128) == (x < 0))[(mag > 0) & (x.abs() > dx)].all()
    assert (lo == hi).double().mean() > 0.999            # the check decides nearly every code
    return pos


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES)
def test_step8_against_64_bits(kind, offset, sizes):
    p_dtype, g_dtype, master = kind
    states = random_state(sizes, p_dtype, g_dtype, master, offset, 2)
    for s in states:
        encode_state(s)
    start = [0.0 if i % 2 else 137.0 for i in range(len(sizes))]
    steps = torch.tensor(start, device=DEV)
    scale = torch.tensor(0.75, device=DEV)
    seeds = [i * 1000003 + 5 for i in range(len(sizes))]
    for k in range(1, 4):
        before = [{x: s[x].t.clone().cpu() for x in ("g", "m", "v", "ms", "vs")} | {"w": (s["w"] or s["p"]).t.clone().cpu()}
                  for s in states]
        fm.adamw8_step([s["p"].t for s in states], [s["g"].t for s in states], [s["m"].t for s in states],
                       [s["ms"].t for s in states], [s["v"].t for s in states], [s["vs"].t for s in states], steps,
                       seeds=seeds, masters=[s["w"].t for s in states] if master else None, grad_scale=scale, **HYPER)
        assert steps.tolist() == [t + k for t in start]
        for s, b, t0, seed in zip(states, before, start, seeds):
            n, t = len(b["g"]), int(t0) + k
            m0, v0 = A.decode(b["m"], b["ms"], 1), A.decode(b["v"], b["vs"], 2)
            w, m, v = A.adamw(b["w"], b["g"], m0[:n], v0[:n], t, scale=0.75, **HYPER)
            dm, dv, dw = tolerances(b["w"], b["g"], m0[:n], v0[:n], w, 0.75, t, HYPER)
            um, uv = A.random_numbers(seed, t, len(m0))
            check_codes(s["m"].t, s["ms"].t, A.pad(m), A.pad(dm), um, 1)
            check_codes(s["v"].t, s["vs"].t, A.pad(v), A.pad(dv), uv, 2)
            check_weights(s, w, dw, p_dtype)
            assert (s["m"].t[n:] == 0).all() and (s["v"].t[n:] == 0).all()   # padding of the last block
            for x in s.values():
                if x is not None:
                    x.check()


@pytest.mark.parametrize("moment", [1, 2])
@pytest.mark.parametrize("dtype", [F32, B16, H16])
@pytest.mark.parametrize("n", [0, 1, 32, 1000, 4096 + 31])
def test_values_and_encode(moment, dtype, n):
    x = torch.randn(n, device=DEV, generator=gen(n + moment)) * 0.01
    x = (x if moment == 1 else x.square()).to(dtype)
    codes, scales = fm.adamw8_encode(x, moment=moment)
    assert codes.numel() == -(-n // 32) * 32 == 32 * scales.numel()
    ref = A.pad(x.double().cpu())
    assert torch.equal(scales.cpu().long(), A.block_scales(ref, moment))
    want = torch.floor(A.rounding_position(ref, scales.cpu().long(), moment) + 0.5)
    if moment == 2:
        want = torch.where(ref > 0, want.clamp(min=1), want)
    assert torch.equal((codes.cpu().long() & (127 if moment == 1 else 255)).double(), want)
    for out in (F32, B16):
        vals = fm.adamw8_values(codes, scales, moment=moment, numel=n, dtype=out)
        assert vals.dtype == out and torch.equal(vals.double().cpu(), A.decode(codes, scales, moment)[:n])


@pytest.mark.parametrize("offset", [0, 3, 32])
def test_values_of_states_at_any_address(offset):
    n = 5 * 4096 + 32
    codes, scales = fm.adamw8_encode(torch.randn(n, device=DEV, generator=gen(1)), moment=1)
    moved = Guarded(codes, offset)
    for dtype in (F32, B16, H16):
        assert torch.equal(fm.adamw8_values(moved.t, scales, moment=1, dtype=dtype),
                           fm.adamw8_values(codes, scales, moment=1, dtype=F32).to(dtype))


def test_step8_values_that_are_not_finite():
    """An element that is not finite costs neither its neighbours nor the block's scale."""
    n = 96
    g = torch.full((n,), 1e-3, device=DEV)
    g[5], g[40], g[70] = math.nan, math.inf, 1e25         # 1e25 squared is infinite in fp32
    p = torch.zeros(n, device=DEV)
    st = [torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(3, dtype=torch.uint8, device=DEV),
          torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(3, dtype=torch.uint8, device=DEV)]
    fm.adamw8_step([p], [g], *[[x] for x in st], torch.zeros(1, device=DEV), lr=0.1, weight_decay=0.0)
    m = fm.adamw8_values(st[0], st[1], moment=1, dtype=F32)
    v = fm.adamw8_values(st[2], st[3], moment=2, dtype=F32)
    assert m[5].isnan() and m[40].isnan() and v[5].isinf() and v[40].isinf() and v[70].isinf()
    ok = torch.ones(n, dtype=torch.bool, device=DEV)
    ok[[5, 40, 70]] = False
    assert p[ok].isfinite().all() and p[[5, 40]].isnan().all()
    near = ok.clone()
    near[64:] = False                                     # the third block's scale is that of 1e24
    assert ((m[near] / 1e-4 - 1).abs() <= 0.125).all() and ((v[ok] / 1e-9 - 1).abs() <= 0.125).all()
    assert m[70].isfinite()
    fm.adamw8_step([p], [g * 0], *[[x] for x in st], torch.ones(1, device=DEV), lr=0.1, weight_decay=0.0)
    assert p[near].isfinite().all()


def test_step8_without_eps():
    """Gradients whose squares are subnormal, or zero: no division by zero although eps is zero."""
    n = 3000
    g = torch.zeros(n, device=DEV)
    for i, x in enumerate((1e-25, 1e-21, 1e-19, 1e-17, 1e-12, 1.0)):
        g[i * 320 + 5:(i + 1) * 320] = x
    p = torch.zeros(n, device=DEV)
    st = [[torch.zeros(-(-n // 32) * k, dtype=torch.uint8, device=DEV)] for k in (32, 1, 32, 1)]
    steps = torch.zeros(1, device=DEV)
    for _ in range(3):
        fm.adamw8_step([p], [g], *st, steps, lr=1.0, weight_decay=0.0, eps=0.0)
        assert p.isfinite().all() and (p[g == 0] == 0).all()
        g.mul_(0.5)
    # where the squares are normal numbers a first step is lr, later ones with shrinking gradients less than 2
    assert (p[g > 1e-18].abs() <= 5.0).all() and (p[g > 1e-18].abs() >= 1.0).all()


def test_step8_is_right_on_average():
    """The mean over 4096 seeds of the stored moments is the moment: rounding is unbiased.  A code's
    step is at most 1/8 of the value, so the mean of N values has a standard deviation of at most
    1/16 / sqrt(N) of it; five of those, and the roundings of the step (10 u) beside it."""
    n, reps = 32, 4096
    g = torch.linspace(0.5, 1.0, n, device=DEV) * 1e-3
    m0, v0 = g * 0.7, g.square() * 1.3
    cm, sm = fm.adamw8_encode(m0, moment=1)
    cv, sv = fm.adamw8_encode(v0, moment=2)
    p = [torch.zeros(n, device=DEV) for _ in range(reps)]
    st = [[x.clone() for _ in range(reps)] for x in (cm, sm, cv, sv)]
    fm.adamw8_step(p, [g] * reps, *st, torch.full((reps,), 9.0, device=DEV), seeds=11, lr=0.0, betas=(0.9, 0.999))
    _, m, v = A.adamw(p[0], g, A.decode(cm, sm, 1), A.decode(cv, sv, 2), 10, lr=0.0, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    for moment, want, codes, scales in ((1, m, st[0], st[1]), (2, v, st[2], st[3])):
        got = fm.adamw8_values(torch.cat(codes), torch.cat(scales), moment=moment, dtype=F32).double().view(reps, n).mean(0).cpu()
        assert ((got / want - 1).abs() <= 5 / 16 / math.sqrt(reps) + 10 * U).all()


def test_equal_calls_give_equal_bits_and_seeds_matter():
    def go(seeds):
        s = random_state([50000, 33], B16, B16, False, 0, 9)
        for x in s:
            encode_state(x)
        steps = torch.zeros(2, device=DEV)
        for _ in range(3):
            fm.adamw8_step([x["p"].t for x in s], [x["g"].t for x in s], [x["m"].t for x in s], [x["ms"].t for x in s],
                           [x["v"].t for x in s], [x["vs"].t for x in s], steps, seeds=seeds, **HYPER)
        return [x[k].t for x in s for k in ("p", "m", "ms", "v", "vs")]
    a, b, c = go(4), go(4), go(5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(a[1], c[1])


def test_indices_beyond_32_bits():
    """A tensor of 2^32 + 100 elements: the tail gets its own random numbers and addresses."""
    n = (1 << 32) + 100
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    tail = 4096 + 100
    lo = n - tail                                        # a multiple of 4096
    p, g = torch.zeros(n, dtype=B16, device=DEV), torch.zeros(n, dtype=B16, device=DEV)
    g[lo:] = torch.randn(tail, device=DEV, generator=gen(0)).to(B16)
    pad = -(-n // 32) * 32
    st = [torch.zeros(pad, dtype=torch.uint8, device=DEV), torch.zeros(pad // 32, dtype=torch.uint8, device=DEV),
          torch.zeros(pad, dtype=torch.uint8, device=DEV), torch.zeros(pad // 32, dtype=torch.uint8, device=DEV)]
    steps = torch.zeros(1, device=DEV)
    fm.adamw8_step([p], [g], *[[x] for x in st], steps, seeds=[77], **HYPER)
    gt, zero = g[lo:].cpu(), torch.zeros(tail)
    w, m, v = A.adamw(zero, gt, zero, zero, 1, **HYPER)
    dm, dv, dw = tolerances(zero, gt, zero, zero, w, 1.0, 1, HYPER)
    um, uv = A.random_numbers(77, 1, pad - lo, lo)
    check_codes(st[0][lo:], st[1][lo // 32:], A.pad(m), A.pad(dm), um, 1)
    check_codes(st[2][lo:], st[3][lo // 32:], A.pad(v), A.pad(dv), uv, 2)
    assert ((p[lo:].double().cpu() - w).abs() <= dw + half_step(w, B16)).all()
    assert not p[:lo].any() and not st[0][:lo].any() and not st[2][:lo].any()
    norm, scale = fm.grad_norm([g], 1.0)
    want = A.grad_norm([gt], 1.0)
    # 32 squares summed in fp32 per thread and chunk, then 64 bits; the root and its rounding
    assert abs(float(norm) / want[0] - 1) <= 20 * U and abs(float(scale) / want[1] - 1) <= 25 * U


# ---------------------------------------------------------------- streams and graphs
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_advances_its_counts(bits):
    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(n, device=DEV).to(dt)) for n, dt in ((5000, B16), (300, F32), (70000, B16))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    lr = torch.tensor(1e-2, device=DEV)
    a, b = fm.AdamW(ps, lr=lr, state_bits=bits, seed=3), fm.AdamW(qs, lr=lr, state_bits=bits, seed=3)

    def step(opt, params):
        _, scale = fm.grad_norm([p.grad for p in params], 1.0)
        opt.step(grad_scale=scale)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, ps)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, ps)
    for i in range(5):
        lr.fill_(1e-2 / (i + 1))                         # a schedule, seen by the replay
        graph.replay()
    lr.fill_(1e-2)
    step(b, qs)
    for i in range(5):
        lr.fill_(1e-2 / (i + 1))
        step(b, qs)
    torch.cuda.synchronize()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        assert float(a.state[p]["step"]) == float(b.state[q]["step"]) == 6.0
        assert all(torch.equal(a.state[p][k], b.state[q][k]) for k in a.state[p])


def test_capture_without_state_is_refused():
    p = torch.nn.Parameter(torch.randn(100, device=DEV))
    p.grad = torch.randn_like(p)
    opt = fm.AdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="one step before capturing"):
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
    assert float(opt.state[p]["step"]) == 1.0


@pytest.mark.parametrize("bits", [32, 8])
def test_two_optimizers_on_two_streams_at_once(bits):
    def make(seed):
        torch.manual_seed(seed)
        ps = [torch.nn.Parameter(torch.randn(n, device=DEV).to(B16)) for n in (2_000_000, 5000, 33)]
        for p in ps:
            p.grad = torch.randn_like(p)
        return ps, fm.AdamW(ps, state_bits=bits, seed=seed)

    def go(ps, opt):
        for _ in range(10):
            _, scale = fm.grad_norm([p.grad for p in ps], 1.0)
            opt.step(grad_scale=scale)

    apart = [make(1), make(2)]
    for x in apart:
        go(*x)
    together = [make(1), make(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for stream, (ps, opt) in zip(streams, together):
            with torch.cuda.stream(stream):
                _, scale = fm.grad_norm([p.grad for p in ps], 1.0)
                opt.step(grad_scale=scale)
    torch.cuda.synchronize()
    for (ps, _), (qs, _) in zip(apart, together):
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_step_waits_for_the_gradients_of_its_stream():
    """Gradients written just ahead on the same stream, over and over: the step reads the new ones."""
    n = 3_000_000
    p = torch.zeros(n, device=DEV)
    g, m, v, steps = torch.empty_like(p), torch.zeros_like(p), torch.zeros_like(p), torch.zeros(1, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for k in range(1, 30):
            g.fill_(float(k))
            fm.adamw_step([p], [g], [m], [v], steps, lr=0.0, betas=(0.0, 0.0), weight_decay=0.0)
            bad = (m != float(k)).any() | (v != float(k * k)).any()
            assert not bool(bad)
    assert float(steps) == 29.0


# ---------------------------------------------------------------- the optimizer
@pytest.mark.parametrize("dtype", [F32, B16])
def test_optimizer_against_torch(dtype):
    """Ten steps beside torch.optim.AdamW.  In float32 both compute the same formula with at most 30 u of
    an update's size and 2 u of the weight per step (docstring; torch's order of operations likewise):
    10 steps, both sides, and lr 1e-2 as the largest update (|m| / sqrt(v) below 2 in this run of
    gradients).  bfloat16 parameters with masters round the same float32 weights."""
    torch.manual_seed(0)
    shapes = [(50, 60), (7,), (1000,), (), (3, 5, 9)]
    ours = [torch.nn.Parameter(torch.randn(s, device=DEV).to(dtype)) for s in shapes]
    theirs = [torch.nn.Parameter(p.detach().float().clone()) for p in ours]
    a = fm.AdamW([{"params": ours[:2], "weight_decay": 0.1}, {"params": ours[2:], "lr": 5e-3}], lr=1e-2,
                 master_weights=dtype != F32)
    b = torch.optim.AdamW([{"params": theirs[:2], "weight_decay": 0.1}, {"params": theirs[2:], "lr": 5e-3}], lr=1e-2)
    for _ in range(10):
        for p, q in zip(ours, theirs):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.float()
        a.step()
        b.step()
    for p, q in zip(ours, theirs):
        w = a.state[p]["master"] if dtype != F32 else p
        bound = 10 * 2 * (30 * U * 2e-2 + 2 * U * q.abs())
        assert ((w - q).abs() <= bound).all()
        if dtype != F32:
            assert torch.equal(p, w.to(dtype))
        assert torch.allclose(a.state[p]["exp_avg_sq"], b.state[q]["exp_avg_sq"], rtol=10 * 2 * 7 * U, atol=0)


def test_optimizer_checkpoints():
    """Round trips in both widths; a torch checkpoint; 8 bits loaded into 32 and back."""
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(200, 33, device=DEV).to(B16))
    small = torch.nn.Parameter(torch.randn(10, device=DEV).to(B16))

    def run(opt, count, seed=1):
        torch.manual_seed(seed)
        for _ in range(count):
            for x in (p, small):
                x.grad = torch.randn_like(x) * 1e-2
            opt.step()

    for bits in (8, 32):
        with torch.no_grad():
            start = [x.clone() for x in (p, small)]
        a = fm.AdamW([p, small], state_bits=bits, master_weights=True, seed=9)
        run(a, 3)
        saved = {k: v for k, v in a.state_dict().items()}
        saved = torch.utils._pytree.tree_map(lambda x: x.clone().cpu() if torch.is_tensor(x) else x, saved)
        mid = [x.detach().clone() for x in (p, small)]
        run(a, 3, 2)
        end = [x.detach().clone() for x in (p, small)]
        with torch.no_grad():
            p.copy_(mid[0]), small.copy_(mid[1])
        b = fm.AdamW([p, small], state_bits=bits, master_weights=True)
        b.load_state_dict(saved)
        assert b.param_groups[0]["seed"] == 9
        run(b, 3, 2)
        assert torch.equal(p, end[0]) and torch.equal(small, end[1])
        # the small tensor keeps 32 bits in both
        assert b.state[small]["exp_avg"].dtype == F32
        other = fm.AdamW([p, small], state_bits=40 - bits)
        other.load_state_dict(saved)
        m, v = other.state_values(p)
        b.load_state_dict(saved)
        m0, v0 = b.state_values(p)
        # 8 to 32 bits is exact; 32 to 8 rounds to nearest: half a step is 1/16 of the value, and
        # below the smallest normal code 2^-17 of the block's largest (2^-32 for the second moment)
        rel = 0 if bits == 8 else 1 / 16
        assert ((m - m0).abs() <= rel * m0.abs() + (rel > 0) * 2.0 ** -16 * m0.abs().max()).all()
        assert ((v - v0).abs() <= rel * v0 + (rel > 0) * 2.0 ** -30 * v0.max()).all()
        with torch.no_grad():
            p.copy_(start[0]), small.copy_(start[1])
    theirs = torch.optim.AdamW([p, small], lr=3e-3)
    for x in (p, small):
        x.grad = torch.randn_like(x)
    theirs.step()
    c = fm.AdamW([p, small], state_bits=8)
    c.load_state_dict(theirs.state_dict())
    assert c.state[p]["exp_avg"].dtype == torch.uint8 and float(c.state[p]["step"]) == 1.0
    c.step()
    assert p.isfinite().all()


def test_optimizer_skips_parameters_without_gradients_and_counts_for_each():
    p, q = (torch.nn.Parameter(torch.randn(100, device=DEV)) for _ in range(2))
    opt = fm.AdamW([p, q])
    p.grad = torch.randn_like(p)
    keep = q.detach().clone()
    opt.step()
    assert torch.equal(q, keep) and q not in opt.state
    q.grad = torch.randn_like(q)
    opt.step()
    assert float(opt.state[p]["step"]) == 2.0 and float(opt.state[q]["step"]) == 1.0
    assert opt.step(lambda: 5.0) == 5.0


def test_operators_refuse_mismatched_tensors():
    z = lambda n, dt=F32: torch.zeros(n, dtype=dt, device=DEV)  # noqa: E731
    ok = dict(params=[z(64)], grads=[z(64)], exp_avgs=[z(64)], exp_avg_sqs=[z(64)], steps=z(1))

    def refuse(message, exc=AssertionError, step=fm.adamw_step, lr=0.1, **change):
        with pytest.raises(exc, match=message):
            step(**{**ok, **change}, lr=lr)

    refuse("`grads` must have the parameters' sizes", grads=[z(63)])
    refuse("`exp_avgs` must be torch.float32", exp_avgs=[z(64, B16)])
    refuse("contiguous", grads=[z(128)[::2]])
    refuse("one count per parameter", steps=z(2))
    refuse("`steps` must be scalars", steps=[z(2)])
    refuse("no master copies", masters=[z(64)])
    refuse("`grad_scale` must be", grad_scale=z(1, B16))
    refuse("`lr` must be", lr=torch.tensor(0.1))
    refuse("float32, got", exc=TypeError, params=[z(64, torch.float64)])
    refuse("16-bit parameters", exc=FlashMuonError, params=[z(64, B16)], grads=[z(64, H16)])
    same = z(64)
    refuse("overlap", exc=FlashMuonError, params=[same, same], grads=[z(64)] * 2, exp_avgs=[z(64), z(64)],
           exp_avg_sqs=[z(64), z(64)], steps=z(2))
    codes = dict(exp_avgs=[z(64, torch.uint8)], exp_avg_scales=[z(2, torch.uint8)], exp_avg_sqs=[z(64, torch.uint8)],
                 exp_avg_sq_scales=[z(2, torch.uint8)])
    refuse("per element", step=fm.adamw8_step, **{**codes, "exp_avgs": [z(60, torch.uint8)]})
    refuse("per block", step=fm.adamw8_step, **{**codes, "exp_avg_scales": [z(3, torch.uint8)]})
    refuse("must be torch.uint8", step=fm.adamw8_step, **{**codes, "exp_avg_sqs": [z(64)]})
    refuse("one entry per parameter", step=fm.adamw8_step, seeds=[], **codes)
    fm.adamw_step(**ok, lr=0.1)                          # and this one runs


# ---------------------------------------------------------------- the set together
@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_muon_and_adamw_with_clipping(bits):
    """Clip all gradients, Muon on the matrices, AdamW on the rest, as a training loop does, against the
    oracles: the clipped gradient and AdamW's weights in 64 bits, Muon's step bit for bit as without
    this module on the same clipped gradients."""
    torch.manual_seed(0)
    mats = [torch.nn.Parameter((torch.randn(128, 192, device=DEV) * 0.02).to(B16)) for _ in range(3)]
    rest = [torch.nn.Parameter((torch.randn(s, device=DEV) * 0.02).to(B16)) for s in ((500, 128), (128,), (7,))]
    twin = [torch.nn.Parameter(m.detach().clone()) for m in mats]
    muon, plain = (fm.Muon(x, lr=0.02, rank=0, world_size=1) for x in (mats, twin))
    adamw = fm.AdamW(rest, lr=3e-3, betas=(0.9, 0.95), weight_decay=0.1, state_bits=bits, master_weights=True)
    for k in range(3):
        for p in mats + rest:
            p.grad = (torch.randn(p.shape, device=DEV) * (1e-4 if k == 1 else 1.0)).to(B16)
        raw = [p.grad.clone() for p in mats + rest]
        norm = fm.clip_grad_norm_(mats + rest, 1.0)
        want, scale = A.grad_norm(raw, 1.0)
        assert abs(float(norm) / want - 1) <= 20 * U
        for p, r in zip(mats + rest, raw):
            if k == 1:
                assert torch.equal(p.grad, r)            # within the norm: left alone
            exact = r.double().cpu() * scale
            assert ((p.grad.double().cpu() - exact).abs() <= half_step(exact, B16) + 30 * U * exact.abs()).all()
        for q, p in zip(twin, mats):
            q.grad = p.grad.clone()
        before = [adamw.state[p]["master"].clone() if adamw.state.get(p) else p.detach().float() for p in rest]
        moments = [[x.clone() for x in adamw.state_values(p)] if adamw.state.get(p) else [torch.zeros_like(p, dtype=F32)] * 2 for p in rest]
        muon.step()
        adamw.step()
        plain.step()
        assert all(torch.equal(q, p) for q, p in zip(twin, mats))
        for p, w0, (m0, v0) in zip(rest, before, moments):
            hyper = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
            w, _, _ = A.adamw(w0, p.grad, m0, v0, k + 1, **hyper)
            _, _, dw = tolerances(w0.cpu(), p.grad.cpu(), m0.cpu(), v0.cpu(), w, 1.0, k + 1, hyper)
            assert ((adamw.state[p]["master"].double().cpu() - w).abs() <= dw).all()
            assert torch.equal(p, adamw.state[p]["master"].to(B16))
    _lib.device_status()

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


def test_a_backward_pass_over_what_was_written_is_refused():
    """The step and the scaling raise the version counters of what they write, and of nothing else."""
    w = torch.nn.Parameter(torch.randn(100, device=DEV))
    w.grad = torch.randn_like(w)
    saved = (w * w).sum()
    fm.AdamW([w]).step()
    with pytest.raises(RuntimeError, match="inplace"):
        saved.backward()
    factor = torch.ones(100, device=DEV, requires_grad=True)
    saved = (factor * w.grad).sum()
    fm.clip_grad_norm_([w], 1e-3)
    with pytest.raises(RuntimeError, match="inplace"):
        saved.backward()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("listed", [False, True], ids=["1-D steps", "list of steps"])
def test_version_counters(bits, listed):
    sizes = (100, 5000, 0)
    new = lambda dt, f=lambda n: n: [torch.zeros(f(n), dtype=dt, device=DEV) for n in sizes]  # noqa: E731
    p, g, w = new(torch.bfloat16), new(torch.bfloat16), new(F32)
    steps = [torch.zeros((), device=DEV) for _ in sizes] if listed else torch.zeros(len(sizes), device=DEV)
    blocks, byte = lambda n: -(-n // 32), torch.uint8  # noqa: E731
    padded = lambda n: 32 * blocks(n)  # noqa: E731
    st = [new(F32), new(F32)] if bits == 32 else [new(byte, padded), new(byte, blocks), new(byte, padded), new(byte, blocks)]
    step = fm.adamw_step if bits == 32 else fm.adamw8_step
    written = [*p, *w, *(steps if listed else [steps]), *(x for xs in st for x in xs)]
    before = [x._version for x in written]
    step(p, g, *st, steps, masters=w, lr=0.1)
    assert [x._version for x in written] == [v + 1 for v in before]
    assert all(x._version == 0 for x in g)
    with pytest.raises(AssertionError):
        step(p, g[::-1], *st, steps, masters=w, lr=0.1)
    with pytest.raises(fm._lib.FlashMuonError):
        step(p, p, *st, steps, masters=w, lr=0.1)
    assert [x._version for x in written] == [v + 1 for v in before]


def test_inference_tensors_are_stepped_too():
    """They have no version counters."""
    with torch.inference_mode():
        p, g, m, v, steps = (torch.ones(n, device=DEV) for n in (100, 100, 100, 100, 1))
    fm.adamw_step([p], [g], [m], [v], steps, lr=0.1)
    with torch.inference_mode():
        fm.adamw_step([p], [g], [m], [v], steps, lr=0.1)
        q = torch.nn.Parameter(p)
        q.grad = g
        fm.clip_grad_norm_([q], 1.0)
    assert float(steps) == 3.0 and float(g[0]) == pytest.approx(0.1, rel=1e-6)


def test_tensors_given_by_iterators():
    p, g, m, v = ([torch.ones(n, device=DEV) for n in (100, 5000)] for _ in range(4))
    steps = torch.zeros(2, device=DEV)
    fm.adamw_step(iter(p), iter(g), iter(m), (x for x in v), iter(steps.unbind()), lr=0.1)
    assert steps.tolist() == [1.0, 1.0] and all((x < 1).all() for x in p)


def test_shapes_that_do_not_fit_are_refused():
    """As many elements in another shape are another order of the elements; flat ones have but one."""
    z = lambda *shape: torch.zeros(shape, device=DEV)  # noqa: E731
    half = torch.zeros(4, 16, device=DEV, dtype=torch.bfloat16)
    ok = dict(params=[half], grads=[z(4, 16)], exp_avgs=[z(4, 16)], exp_avg_sqs=[z(4, 16)], masters=[z(4, 16)], steps=z(1), lr=0.1)
    for name in ("grads", "exp_avgs", "exp_avg_sqs", "masters"):
        for shape in ((16, 4), (8, 8), (4, 16, 1), (2, 2, 16)):
            with pytest.raises(AssertionError, match=f"`{name}` must have the parameters' sizes"):
                fm.adamw_step(**{**ok, name: [z(*shape)]})
        fm.adamw_step(**{**ok, name: [z(64)]})
    fm.adamw_step(**{**ok, "params": [half.view(-1)]})
    fm.adamw_step(**ok)
    assert float(ok["steps"]) == 6.0
    codes = [torch.zeros(n, dtype=torch.uint8, device=DEV) for n in (64, 2, 64, 2)]
    with pytest.raises(AssertionError, match="`grads` must have"):
        fm.adamw8_step([half], [z(16, 4)], *[[c] for c in codes], z(1), lr=0.1)
    scalar = z()
    fm.adamw_step([scalar], [z(1)], [z()], [z(1)], z(1), lr=0.1)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_a_factor_on_one_of_two_devices_is_refused_before_any_step():
    ps = [torch.nn.Parameter(torch.ones(10, device=f"cuda:{i}")) for i in range(2)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = fm.AdamW(ps)
    opt.step()
    before = [p.detach().clone() for p in ps]
    with pytest.raises(AssertionError, match="`grad_scale` must be"):
        opt.step(grad_scale=torch.ones((), device="cuda:0"))
    assert all(torch.equal(p, b) for p, b in zip(ps, before))


@pytest.mark.parametrize("saved_as", ["cpu", "device", "float"])
def test_a_learning_rate_tensor_outlives_a_checkpoint(saved_as):
    """A schedule holds the tensor itself: it takes the loaded value and stays."""
    p = torch.nn.Parameter(torch.zeros(5, device=DEV))
    p.grad = torch.ones_like(p)
    lr = torch.tensor(0.5, device=DEV)
    opt = fm.AdamW([p], lr=lr, weight_decay=0.0)
    opt.step()
    saved = opt.state_dict()
    value = {"cpu": torch.tensor(0.125), "device": torch.tensor(0.125, device=DEV), "float": 0.125}[saved_as]
    saved["param_groups"][0]["lr"] = value
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.125
    lr.fill_(0.25)
    before = p.detach().clone()
    opt.step()
    # equal gradients: m / sqrt(v), both corrected, is 1 but for eps
    assert torch.allclose(before - p, torch.full_like(p, 0.25), rtol=1e-4)
    other = fm.AdamW([p], lr=0.75)
    other.load_state_dict(saved)
    assert other.param_groups[0]["lr"] == 0.125 and isinstance(other.param_groups[0]["lr"], float)
    other.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_and_steps_in_two_graphs(bits):
    """Graphs captured apart share no scratch, and each replay clips the gradients that are there."""
    ps = [torch.nn.Parameter(torch.randn(n, device=DEV)) for n in (300, 50000, 0, 8)]
    for p in ps:
        p.grad = torch.randn_like(p)
    opt = fm.AdamW(ps, lr=0.01, state_bits=bits, min_8bit_numel=0)
    opt.step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = fm.clip_grad_norm_(ps, 1.0)
            opt.step()
        graphs.append((graph, norm))
    for i in range(6):
        for p in ps:
            p.grad.normal_()
        want = sum(float(p.grad.double().square().sum()) for p in ps) ** 0.5
        graph, norm = graphs[i % 2]
        graph.replay()
        # 17 u for the norm; the factor and the products of the clipped elements 5 u more
        assert abs(float(norm) / want - 1) <= 17 * 2.0 ** -24
        assert abs(sum(float(p.grad.double().square().sum()) for p in ps) ** 0.5 - 1) <= 24 * 2.0 ** -24 + 1e-6 / want
    assert all(float(opt.state[p]["step"]) == 7.0 for p in ps)

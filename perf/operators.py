"""The optimizer operators that stand beside Muon, as they are measured: the AdamW step with states
in 32 bits, the AdamW step with states in 8 bits, and the norm of all gradients with the factor that
clips them.  ``run`` computes them in elementary torch operations, or, where ``own`` is true, calls
the package.

All tensors of a case lie in one buffer per kind (parameters, gradients, moments ...), each tensor at
a multiple of 32 elements, with zeros between them; a step leaves those zeros as they are, so the
plain form works on the whole buffer at once and the buffers are what a pass returns.

States in 8 bits: blocks of 32 elements of a tensor share a byte b, the exponent byte of the block's
largest finite magnitude, but at least 17 (first moment) or 32 (second), so that no code stands for a
subnormal fp32 number.  The first moment is sign | e4m3 times 2**(b - 134), the second unsigned e5m3
times 2**(b - 127) (table below).  Values are rounded up or down at random, the chance of "up" being
the distance to the value below: the random number is a function of the tensor's seed, the step's
count and the element's index.
"""
import random

import torch

own = False

BLOCK = 32
BETA1, BETA2, EPS = 0.9, 0.95, 1e-8
LR, WEIGHT_DECAY = 3e-4, 0.1
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _case(op, p, g, big, vectors, width, **more):
    """`big`: elements of one large tensor (0: none); `vectors` tensors of `width` elements, or of
    one element up to `width` where `ragged`."""
    return {"op": op, "p": p, "g": g, "big": big, "vectors": vectors, "width": width,
            "ragged": False, "master": False, "shift": 0, "scaled": False, **more}


def listed():
    return [
        # one bias, the smallest call: latency alone
        dict(_case("adamw", "f32", "f32", 0, 1, 1000), name="adamw one bias"),
        # the norm weights of a 32-layer model of width 4096, kept in float32
        dict(_case("adamw", "f32", "f32", 0, 65, 4096), name="adamw norm weights f32"),
        # what Muon leaves over in a small model: odd sizes, gradients accumulated in float32,
        # storage that starts at an odd element
        dict(_case("adamw", "bf16", "f32", 0, 120, 2_000_003, ragged=True, shift=1), name="adamw ragged bf16, f32 grads"),
        # an embedding of 32000 rows of 4096 and the norms beside it, all bfloat16
        dict(_case("adamw", "bf16", "bf16", 32000 * 4096, 65, 4096), name="adamw embedding bf16"),
        # the same kind of table with float32 master copies of bfloat16 weights
        dict(_case("adamw", "bf16", "bf16", 50000 * 1024, 49, 1024, master=True), name="adamw masters"),
        # the largest: embedding of 128000 rows of 4096 in float32
        dict(_case("adamw", "f32", "f32", 128000 * 4096, 0, 1), name="adamw largest f32"),
        # 8-bit states of biases and norms: latency
        dict(_case("adamw8", "bf16", "bf16", 0, 48, 4096), name="adamw8 biases"),
        # odd sizes in float16, gradients that still carry a loss scale
        dict(_case("adamw8", "f16", "f16", 0, 90, 3_000_001, ragged=True, scaled=True), name="adamw8 ragged f16"),
        # the largest embedding with 8-bit states, bfloat16
        dict(_case("adamw8", "bf16", "bf16", 128000 * 4096, 65, 4096), name="adamw8 largest bf16"),
        # the norm over gradients of norms and biases: latency
        dict(_case("norm", "bf16", "bf16", 0, 97, 1024), name="norm of vectors"),
        # the norm over all gradients of 24 layers of width 1024 and an embedding
        dict(_case("norm", "bf16", "bf16", 50000 * 1024, 288, 1024 * 1024), name="norm of a model bf16"),
        # clipping and the step together: the factor goes into the step, gradients stay as they are
        dict(_case("clip_adamw", "bf16", "f32", 32000 * 2048, 65, 2048, master=True), name="clip and adamw, masters"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "norm", "clip_adamw"])
    p, g = rng.choice([("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32"),
                       ("f32", "bf16"), ("f32", "f16")])
    big = rng.choice([0, log(1000, 300_000_000)])
    vectors = log(1, 300)
    width = log(1, min(4_000_000, 300_000_000 // vectors))
    return _case(op, p, g, big, vectors, width, ragged=rng.random() < 0.6,
                 master=op != "norm" and p != "f32" and rng.random() < 0.5,
                 shift=rng.choice([0, 0, 1, 3]), scaled=op in ("adamw", "adamw8") and g == "f16")


def _sizes(case):
    r = random.Random(case["vectors"] * 1_000_003 + case["width"])
    vec = [int(round(case["width"] ** r.random())) if case["ragged"] else case["width"]
           for _ in range(case["vectors"])]
    return ([case["big"]] if case["big"] else []) + vec


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def work(case):
    n = sum(_sizes(case))
    ps, gs = BYTES[case["p"]], BYTES[case["g"]]
    if case["op"] == "norm":
        return {"bytes": n * gs, "flops": 2 * n}
    weights = 8 + ps if case["master"] else 2 * ps       # masters in and out, parameters out
    if case["op"] == "adamw8":
        # codes in and out, a byte of scale per block and moment in and out, and the two moments'
        # values, which the pass returns in bfloat16
        return {"bytes": n * (weights + gs + 4 + 4) + 4 * n / BLOCK, "flops": 40 * n}
    return {"bytes": n * (weights + gs + 16), "flops": 14 * n + (2 * n if case["op"] == "clip_adamw" else 0)}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    sizes = _sizes(case)
    pads = [_padded(n) for n in sizes]
    total = sum(pads)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dev = "cuda"

    def normal():
        return torch.randn(total, device=dev, generator=gen)

    # magnitudes differ from stretch to stretch of 1024 elements; in every fourth the gradient is
    # zero, as in the rows of an embedding whose token did not occur
    stretch = -(-total // 1024)
    mag = 10.0 ** (torch.rand(stretch, device=dev, generator=gen) * 3 - 5)
    seen = (torch.rand(stretch, device=dev, generator=gen) < 0.75).float()
    mag_e = mag.repeat_interleave(1024)[:total]
    seen_e = seen.repeat_interleave(1024)[:total]
    hold = torch.ones(total, device=dev)                  # zero between the tensors
    at = 0
    for n, m in zip(sizes, pads):
        hold[at + n:at + m] = 0
        at += m

    loss_scale = 1024.0 if case["scaled"] else 1.0
    grad = normal() * mag_e * seen_e * hold * loss_scale
    weight = normal() * 0.02 * hold
    state = {"case": case, "sizes": sizes, "pads": pads, "total": total}
    state["blocks"] = torch.tensor([m // BLOCK for m in pads], device=dev)
    state["starts"] = state["blocks"].cumsum(0) * BLOCK - state["blocks"] * BLOCK

    def kept(x, dtype):                                   # storage that starts at an odd element, or not
        buf = torch.zeros(total + case["shift"], device=dev, dtype=dtype)
        buf[case["shift"]:] = x.to(dtype)
        return buf[case["shift"]:]

    def views(flat, lengths=None):
        return [x[:n] for x, n in zip(flat.split(pads), lengths or sizes)]

    state["grad"] = kept(grad, TYPES[case["g"]])
    state["grads"] = views(state["grad"])
    if case["op"] in ("norm", "clip_adamw"):
        state["max_norm"] = 0.01
    del grad, seen_e
    if case["op"] == "norm":
        return state
    state["param"] = kept(weight, TYPES[case["p"]])
    state["params"] = views(state["param"])
    state["master"], state["masters"] = None, None
    if case["master"]:
        # a master differs from its rounded parameter in the bits below
        state["master"] = state["param"].float() * (1 + 1e-4 * normal())
        state["masters"] = views(state["master"])
    state["steps"] = torch.tensor([200.0 + i % 7 for i in range(len(sizes))], device=dev)
    state["scale"] = torch.full((), 1.0 / loss_scale, device=dev) if case["scaled"] else None
    exp_avg = normal() * 0.3 * mag_e * hold
    exp_avg_sq = mag_e.square() * (0.2 + torch.rand(total, device=dev, generator=gen)) * hold
    if case["op"] == "adamw8":
        half = torch.tensor(0.5, device=dev)
        state["m_code"], state["m_exp"] = _encode(exp_avg, half, 1)
        state["v_code"], state["v_exp"] = _encode(exp_avg_sq, half, 2)
        state["seeds"] = [1234 + 17 * i for i in range(len(sizes))]
        state["seed_of"] = torch.tensor(state["seeds"], device=dev)
        blocks = [m // BLOCK for m in pads]
        for k in ("m", "v"):
            state[k + "_codes"] = list(state[k + "_code"].split(pads))
            state[k + "_exps"] = list(state[k + "_exp"].split(blocks))
    else:
        state["exp_avg"], state["exp_avg_sq"] = exp_avg, exp_avg_sq
        state["exp_avgs"], state["exp_avg_sqs"] = views(exp_avg), views(exp_avg_sq)
    return state


# ---------------------------------------------------------------- plain form
def _spread(x, state):
    """One value per tensor, for each of its blocks, as a column."""
    if x.numel() == 1:
        return x
    return x.repeat_interleave(state["blocks"], output_size=state["total"] // BLOCK).unsqueeze(1)


def _power(b):
    """2.0 ** (b - 127) for 1 <= b <= 254."""
    return (b.to(torch.int32) << 23).view(torch.float32)


def _table(moment, device):
    c = torch.arange(256, device=device)
    k = c & 127 if moment == 1 else c
    e, f = k >> 3, (k & 7).float()
    low = -16 if moment == 1 else -31                    # exponent of the smallest step
    value = torch.where(e == 0, f, (8 + f) * _power(126 + e)) * 2.0 ** low
    if moment == 1:
        value = torch.where(c >= 128, -value, value)
        return torch.where(k == 127, float("nan"), value)
    return torch.where(k == 255, float("inf"), value)


def _decode(code, exps, moment):
    return _table(moment, code.device)[code.to(torch.int32)].view(-1, BLOCK) * _power(exps).unsqueeze(1)


def _encode(x, up, moment):
    """Codes and exponent bytes of `x`; a value goes up where its distance to the code below, in
    steps, and `up` (0 <= up < 1) together reach one."""
    blocks = x.abs().view(-1, BLOCK)
    finite = blocks.isfinite()
    largest = torch.where(finite, blocks, 0.0).amax(1)
    b = (largest.view(torch.int32) >> 23).clamp(17 if moment == 1 else 32, 253)
    y = blocks * _power(254 - b).unsqueeze(1)
    low = -13 if moment == 1 else -28                    # exponent of the smallest normal value
    e = ((y.contiguous().view(torch.int32) >> 23) - 127).clamp(min=low)
    k = torch.floor(y * _power(130 - e) + up)
    code = k.to(torch.int32) + 8 * (e - low)
    if moment == 1:
        code = torch.where(finite, code.clamp(max=126), 127) | ((x.view(-1, BLOCK) < 0).to(torch.int32) << 7)
    else:
        code = torch.where(finite, code.clamp(max=254), 255)
        code = torch.where(blocks > 0, code.clamp(min=1), code)
    return code.to(torch.uint8).view(-1), b.to(torch.uint8)


def _mix(x):
    """A bijection of 32 bits (in int64) that spreads every bit over all of them."""
    x = x ^ (x >> 16)
    x = (x * 0xa1c7d3e7) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x2e3ad36d) & 0xffffffff
    return x ^ (x >> 16)


def _random_bits(state, count):
    """32 bits for each element, from its tensor's seed, the step's count and its index."""
    key = _mix((_mix(state["seed_of"]) + count.to(torch.int64)) & 0xffffffff)
    index = torch.arange(state["total"], device=count.device).view(-1, BLOCK) - _spread(state["starts"], state)
    return _mix((index & 0xffffffff) ^ _mix((_spread(key, state) + (index[:, :1] >> 32)) & 0xffffffff))


def _plain_norm(state):
    norm = state["grad"].double().square().sum().sqrt().float()
    scale = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return norm, scale


def _plain_adamw(state, scale):
    grad = state["grad"].view(-1, BLOCK).float()
    if scale is not None:
        grad = grad * scale
    weight = (state["param"].float() if state["master"] is None else state["master"]).view(-1, BLOCK)
    count = state["steps"].add_(1)
    t = count.double()
    size = _spread((LR / (1 - BETA1 ** t)).float(), state)
    root = _spread((1 - BETA2 ** t).sqrt().float(), state)
    eight = "m_code" in state
    m = _decode(state["m_code"], state["m_exp"], 1) if eight else state["exp_avg"].view(-1, BLOCK)
    v = _decode(state["v_code"], state["v_exp"], 2) if eight else state["exp_avg_sq"].view(-1, BLOCK)
    m = m * BETA1 + grad * (1 - BETA1)
    v = v * BETA2 + grad * grad * (1 - BETA2)
    weight = weight * (1 - LR * WEIGHT_DECAY) - size * m / (v.sqrt() / root + EPS)
    weight = weight.view(-1)
    state["param"].copy_(weight)
    out = {"param": state["param"], "steps": count}
    if state["master"] is not None:
        out["master"] = state["master"].copy_(weight)
    if not eight:
        out["exp_avg"] = state["exp_avg"].copy_(m.view(-1))
        out["exp_avg_sq"] = state["exp_avg_sq"].copy_(v.view(-1))
        return out
    bits = _random_bits(state, count)
    for k, x, u, moment in (("m", m, bits & 0xfffff, 1), ("v", v, bits >> 12, 2)):
        code, exps = _encode(x, u.float() * 2.0 ** -20, moment)
        state[k + "_code"].copy_(code)
        state[k + "_exp"].copy_(exps)
        # a code's value has four significant bits: bfloat16 holds it as it is
        out[k + "_value"] = _decode(code, exps, moment).view(-1).bfloat16()
    return out


# ---------------------------------------------------------------- the package's calls
def _own_norm(state):
    import flash_muon_b200 as fm
    return fm.grad_norm(state["grads"], state["max_norm"])


def _own_adamw(state, scale):
    import flash_muon_b200 as fm
    settings = dict(lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=WEIGHT_DECAY,
                    masters=state["masters"], grad_scale=scale)
    out = {"param": state["param"], "steps": state["steps"]}
    if state["master"] is not None:
        out["master"] = state["master"]
    if "m_code" not in state:
        fm.adamw_step(state["params"], state["grads"], state["exp_avgs"], state["exp_avg_sqs"],
                      state["steps"], **settings)
        return {**out, "exp_avg": state["exp_avg"], "exp_avg_sq": state["exp_avg_sq"]}
    fm.adamw8_step(state["params"], state["grads"], state["m_codes"], state["m_exps"],
                   state["v_codes"], state["v_exps"], state["steps"], seeds=state["seeds"], **settings)
    return {**out, "m_value": fm.adamw8_values(state["m_code"], state["m_exp"], moment=1),
            "v_value": fm.adamw8_values(state["v_code"], state["v_exp"], moment=2)}


def run(state):
    op = state["case"]["op"]
    norm_of, step = (_own_norm, _own_adamw) if own else (_plain_norm, _plain_adamw)
    if op == "norm":
        norm, scale = norm_of(state)
        return {"norm": norm, "scale": scale}
    if op == "clip_adamw":
        norm, scale = norm_of(state)
        return {"norm": norm, "scale": scale, **step(state, scale)}
    return step(state, state["scale"])


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_codes(moment):
    """The values of the non-negative finite codes in units of 2 ** (b - 127), ascending."""
    if moment == 1:
        return [(f if e == 0 else (8 + f) * 2.0 ** (e - 1)) * 2.0 ** -16 for e in range(16) for f in range(8)][:127]
    return [(f if e == 0 else (8 + f) * 2.0 ** (e - 1)) * 2.0 ** -31 for e in range(32) for f in range(8)][:255]


def _exact_rounded(x, chance, moment):
    """The value that stands for each element after rounding, blocks of 32."""
    values = torch.tensor(_exact_codes(moment), dtype=torch.float64, device=x.device)
    mag = x.abs().view(-1, BLOCK)
    _, e = torch.frexp(mag.amax(1, keepdim=True))        # largest = f * 2**e with 0.5 <= f < 1
    exponent = (e - 1).clamp(-110 if moment == 1 else -95, 126)
    exponent = torch.where(mag.amax(1, keepdim=True) == 0, -110 if moment == 1 else -95, exponent)
    unit = torch.ones_like(mag[:, :1]).ldexp(exponent)
    y = (mag / unit).view(-1)
    below = torch.searchsorted(values, y, right=True) - 1
    above = (below + 1).clamp(max=len(values) - 1)
    step = (values[above] - values[below]).clamp(min=1e-300)
    k = torch.where((y - values[below]) / step + chance >= 1, above, below)
    if moment == 2:
        k = torch.where(y > 0, k.clamp(min=1), k)
    return (values[k].view(-1, BLOCK) * unit).view(-1) * x.sign()


def _exact_hash(seed, count, index):
    def turn(h):
        for shift, factor in ((16, 2714227687), (15, 775607149)):
            h = (h ^ (h >> shift)) * factor % 2 ** 32
        return h ^ (h >> 16)

    def turn_all(h):
        h = (h ^ (h >> 16)) * 2714227687 & 4294967295
        h = (h ^ (h >> 15)) * 775607149 & 4294967295
        return h ^ (h >> 16)

    key = turn((turn(seed) + count) % 2 ** 32)           # indices below 2**32 only
    return turn_all(index ^ turn(key))


def exact(case, seed):
    s = prepare(case, seed)
    out = {}
    scale = 1.0 if s.get("scale") is None else s["scale"].double()
    if case["op"] in ("norm", "clip_adamw"):
        total = sum(x.double().pow(2).sum() for x in s["grad"].split(1 << 26))
        norm = total.sqrt()
        scale = torch.minimum(s["max_norm"] / (norm + 1e-6), torch.ones_like(norm))
        out = {"norm": norm, "scale": scale}
        if case["op"] == "norm":
            return out
    eight = case["op"] == "adamw8"
    names = ["param", "master", "m_value", "v_value"] if eight else ["param", "master", "exp_avg", "exp_avg_sq"]
    parts = {k: [] for k in names}
    if eight:
        tables = {}
        for moment in (1, 2):
            pos = _exact_codes(moment)
            full = pos + [float("nan")] + [-x for x in pos] + [float("nan")] if moment == 1 else pos + [float("inf")]
            tables[moment] = torch.tensor(full, dtype=torch.float64, device="cuda")
    at = 0
    for i, pad in enumerate(s["pads"]):
        count = int(s["steps"][i].item()) + 1
        size = LR / (1 - BETA1 ** count)
        root = (1 - BETA2 ** count) ** 0.5
        for lo in range(0, pad, 1 << 26):
            hi = min(pad, lo + (1 << 26))
            here = slice(at + lo, at + hi)
            g = s["grad"][here].double() * scale
            w = (s["param"] if s["master"] is None else s["master"])[here].double()
            if eight:
                blocks = slice((at + lo) // BLOCK, (at + hi) // BLOCK)
                m, v = ((tables[k][s[c + "_code"][here].long()].view(-1, BLOCK)
                         * torch.pow(2.0, s[c + "_exp"][blocks].double() - 127).unsqueeze(1)).view(-1)
                        for k, c in ((1, "m"), (2, "v")))
            else:
                m, v = s["exp_avg"][here].double(), s["exp_avg_sq"][here].double()
            m = BETA1 * m + (1 - BETA1) * g
            v = BETA2 * v + (1 - BETA2) * g ** 2
            w = w - LR * WEIGHT_DECAY * w - size * m / (torch.sqrt(v) / root + EPS)
            if eight:
                h = _exact_hash(s["seeds"][i], count, torch.arange(lo, hi, device="cuda"))
                m = _exact_rounded(m, (h % 2 ** 20).double() / 2 ** 20, 1)
                v = _exact_rounded(v, (h // 2 ** 12).double() / 2 ** 20, 2)
            for name, x in zip(names, (w, w, m, v)):
                if name != "master" or s["master"] is not None:
                    parts[name].append(x)
        at += pad
    out["steps"] = (s["steps"] + 1).double()
    for name, xs in parts.items():
        if xs:
            out[name] = torch.cat(xs)
    return out

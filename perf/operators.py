"""The gated feed-forward block (forward and backward), AdamW over many tensors and the norm of all gradients: the calls that are timed, their
plain forms in elementary torch operations, and their values in 64 bits."""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256            # values that share a scale of an 8-bit state
E4M3_MAX = 448.0       # first moments: e4m3 codes
ROOT_MAX = 4032.0      # roots of second moments: codes of 3 bits of exponent and 5 of mantissa that stand for 0 .. 31, 32 .. 63, 64, 66 .. 4032
FLT_MIN = 2.0 ** -126
BETAS, EPS = (0.9, 0.999), 1e-8


def listed():
    return [
        # one token of a served model: latency counts
        {"name": "ffn token bf16", "op": "ffn_forward", "dtype": "bf16", "rows": 1, "d": 1024, "f": 4096, "act": "silu", "bias": False, "pad": 0},
        # a few sequences decoded side by side through a wide block: the weights' bytes count
        {"name": "ffn 8 tokens bf16", "op": "ffn_forward", "dtype": "bf16", "rows": 8, "d": 4096, "f": 16384, "act": "silu", "bias": False, "pad": 0},
        # the samples of one training batch, 4096 rays of 64, at the trunk's width
        {"name": "ffn ray samples bf16", "op": "ffn_forward", "dtype": "bf16", "rows": 262144, "d": 256, "f": 1024, "act": "gelu", "bias": True, "pad": 0},
        # a ragged prompt through a block of odd sizes, in 32 bits
        {"name": "ffn odd f32", "op": "ffn_forward", "dtype": "f32", "rows": 1999, "d": 1001, "f": 2731, "act": "gelu_tanh", "bias": True, "pad": 3},
        # a training batch of 8192 tokens
        {"name": "ffn grads bf16", "op": "ffn_backward", "dtype": "bf16", "rows": 8192, "d": 2048, "f": 8192, "act": "silu", "bias": False, "pad": 0},
        # the samples of a batch of 1024 rays in the default type
        {"name": "ffn grads ray samples f32", "op": "ffn_backward", "dtype": "f32", "rows": 65536, "d": 256, "f": 1024, "act": "gelu", "bias": True, "pad": 0},
        # a short batch, odd sizes, a strided input
        {"name": "ffn grads odd f16", "op": "ffn_backward", "dtype": "f16", "rows": 777, "d": 519, "f": 1411, "act": "relu", "bias": True, "pad": 5},
        # the two networks of the default radiance field: 48 tensors, a million values, biases without decay
        {"name": "adamw field f32", "op": "adamw", "dtype": "f32", "grads": "f32", "bits": 32, "master": False, "clip": 0.0, "kind": "field", "total": 1060360, "count": 48, "mix": 0},
        # four blocks of a token network, 16-bit weights with 32-bit copies, clipped
        {"name": "adamw blocks master", "op": "adamw", "dtype": "bf16", "grads": "bf16", "bits": 32, "master": True, "clip": 1.0, "kind": "blocks", "total": 201326592, "count": 12, "mix": 0},
        # the same weights without copies and with states in 8 bits
        {"name": "adamw blocks 8-bit", "op": "adamw", "dtype": "bf16", "grads": "bf16", "bits": 8, "master": False, "clip": 0.0, "kind": "blocks", "total": 201326592, "count": 12, "mix": 0},
        # the norms on their own
        {"name": "grad norm field f32", "op": "grad_norm", "dtype": "f32", "grads": "f32", "bits": 8, "master": False, "clip": 0.5, "kind": "field", "total": 1060360, "count": 48, "mix": 0},
        {"name": "grad norm blocks bf16", "op": "grad_norm", "dtype": "bf16", "grads": "bf16", "bits": 8, "master": False, "clip": 1.0, "kind": "blocks", "total": 201326592, "count": 12, "mix": 0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ffn_forward", "ffn_forward", "ffn_backward", "ffn_backward", "adamw", "adamw", "grad_norm"])
    if op.startswith("ffn"):
        dtype = rng.choice(["bf16", "f16", "f32"])
        most = 2.0e12 if dtype != "f32" else 4.0e11
        while True:
            rows = _log(rng, 1, 262144) if op == "ffn_forward" else _log(rng, 16, 131072)
            d, f = _log(rng, 32, 4096), _log(rng, 64, 16384)
            if rng.random() < 0.6:  # as models have them; the rest odd
                d, f = max(32, d // 32 * 32), max(64, f // 64 * 64)
            case = {"op": op, "dtype": dtype, "rows": rows, "d": d, "f": f, "act": rng.choice(["silu", "gelu", "gelu_tanh", "relu"]),
                    "bias": rng.random() < 0.5, "pad": rng.choice([0, 0, 8, rng.randrange(1, 64)])}
            if work(case)["flops"] <= most and rows * f <= 3.0e8:
                return case
    dtype = rng.choice(["f32", "bf16", "f16"])
    return {"op": op, "dtype": dtype, "grads": rng.choice([dtype, "f32"]), "bits": rng.choice([8, 32]), "master": dtype != "f32" and rng.random() < 0.5,
            "clip": rng.choice([0.0, 0.1, 1.0]), "kind": "ragged", "total": _log(rng, 2000, 120000000), "count": _log(rng, 1, 200), "mix": rng.randrange(1 << 30)}


def _shapes(case):
    """Sizes of the tensors, and whether each is a matrix."""
    if case["kind"] == "field":
        one = []
        for out, inp in [(256, 63)] + [(256, 256)] * 4 + [(256, 319)] + [(256, 256)] * 2 + [(1, 256), (128, 256), (128, 27), (3, 128)]:
            one += [(out * inp, True), (out, False)]
        return one * 2
    if case["kind"] == "blocks":
        n = case["total"] // case["count"]
        return [(n, True)] * case["count"]
    rng, left, got = random.Random(case["mix"]), case["total"], []
    for k in range(case["count"] - 1):
        n = max(1, min(left - (case["count"] - 1 - k), int(2 * rng.random() * left / (case["count"] - k))))
        got.append((n, rng.random() < 0.7))
        left -= n
    return got + [(max(1, left), True)]


def _offsets(case):
    """Where each tensor starts in a flat buffer, and the buffer's size. Tensors follow one another; with 8-bit states each starts a block of its own."""
    step = BLOCK if case["bits"] == 8 else 1
    at, starts = 0, []
    for n, _ in _shapes(case):
        starts.append(at)
        at += -(-n // step) * step
    return starts, at


def _quantised(t, top):
    """Blocks of 256 over their scales, and the scales."""
    t = t.view(-1, BLOCK)
    scale = (t.abs().amax(1) * (1.0 / top)).clamp(min=FLT_MIN)
    return t * scale.reciprocal()[:, None], scale


def _codes_m(m):
    q, scale = _quantised(m, E4M3_MAX)
    return q.to(torch.float8_e4m3fn).view(-1), scale


def _values_m(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _codes_r(r):
    """To the nearest code, ties to even; a positive value never becomes zero."""
    q, scale = _quantised(r, ROOT_MAX)
    bits = q.clamp(min=1.0).view(torch.int32)
    bits = (bits + 0x1FFFF + ((bits >> 18) & 1)) >> 18
    code = torch.where(q < 64.0, torch.round(q).to(torch.int32), bits - (131 << 5))
    code = torch.maximum(code, (q > 0).to(torch.int32))
    return code.to(torch.uint8).view(-1), scale


def _values_r(codes, scale):
    c = codes.view(-1, BLOCK).to(torch.int32)
    value = torch.where(c < 32, c.float(), ((c + (131 << 5)) << 18).view(torch.float32))
    return (value * scale[:, None]).view(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    dtype = TYPES[case["dtype"]]
    s = {"case": case}
    if case["op"].startswith("ffn"):
        n, d, f = case["rows"], case["d"], case["f"]
        wide = d + case["pad"]
        s["x"] = normal(n, wide).to(dtype)[:, :d]
        s["w_gate"] = (normal(f, d) / math.sqrt(d)).to(dtype)
        s["w_up"] = (normal(f, d) / math.sqrt(d)).to(dtype)
        s["w_down"] = (normal(d, f) / math.sqrt(f)).to(dtype)
        for name, k in (("b_gate", f), ("b_up", f), ("b_down", d)):
            s[name] = (0.1 * normal(k)).to(dtype) if case["bias"] else None
        if case["op"] == "ffn_backward":
            s["dy"] = (0.01 * normal(n, wide)).to(dtype)[:, :d]
        if own:
            from nerf_amd import GatedFFN
            s["ffn"] = GatedFFN(d, f, dtype=case["dtype"], activation=case["act"], bias=case["bias"], device=0)
        return s
    starts, size = _offsets(case)
    shapes = _shapes(case)
    real = torch.zeros(size, dtype=torch.bool, device="cuda") if case["bits"] == 8 else None
    spread, decay = torch.empty(size, device="cuda"), torch.zeros(size, device="cuda")
    rng = random.Random(seed)
    for at, (n, matrix) in zip(starts, shapes):
        spread[at:at + n] = 10.0 ** rng.uniform(-4.0, -2.0)
        decay[at:at + n] = 0.1 if matrix else 0.0
        if real is not None:
            real[at:at + n] = True

    def filled(t):
        return t if real is None else t * real

    g = filled(normal(size) * spread).to(TYPES[case["grads"]])
    p = filled(0.02 * normal(size))
    m = filled(0.3 * spread * normal(size))
    r = filled(spread * (0.5 + torch.rand(size, generator=gen, device="cuda")))
    s.update(p=p.to(dtype), g=g, decay=0.1 if all(x for _, x in shapes) else decay, step=100, lr=1e-4)
    if case["master"]:
        s["master"] = p
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _codes_m(m)
        s["r"], s["r_scale"] = _codes_r(r)
    else:
        s["m"], s["v"] = m, r * r
    if own:
        from nerf_amd import AdamW

        def views(flat, div=1):
            return [flat[at // div:at // div + -(-n // div)] for at, (n, _) in zip(starts, shapes)]

        if case["bits"] == 8:
            state = {"exp_avg": views(s["m"]), "exp_avg_scale": views(s["m_scale"], BLOCK),
                     "exp_avg_sq": views(s["r"]), "exp_avg_sq_scale": views(s["r_scale"], BLOCK)}
        else:
            state = {"exp_avg": views(s["m"]), "exp_avg_sq": views(s["v"])}
        if case["master"]:
            state["master"] = views(s["master"])
        s["opt"] = AdamW(views(s["p"]), views(s["g"]), lr=s["lr"], betas=BETAS, eps=EPS, weight_decay=[0.1 if x else 0.0 for _, x in shapes],
                         state_bits=case["bits"], master=case["master"], state=state, step=s["step"])
    return s


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        q = 1.0 / (1.0 + torch.exp(-g))
        return g * q, q * (1.0 + g * (1.0 - q))
    if kind == "gelu":
        c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    if kind == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * k * (1.0 + 3.0 * 0.044715 * g * g)
    on = (g > 0).to(g.dtype)
    return g * on, on


def _ffn_forward(s):
    c, x = s["case"], s["x"].float()
    g, u = x @ s["w_gate"].float().t(), x @ s["w_up"].float().t()
    if c["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    y = (_act(g, c["act"])[0] * u) @ s["w_down"].float().t()
    if c["bias"]:
        y = y + s["b_down"].float()
    return y.to(s["x"].dtype)


def _ffn_backward(s):
    c, t = s["case"], s["x"].dtype
    x, dy, wg, wu, wd = (s[k].float() for k in ("x", "dy", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    if c["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    a, slope = _act(g, c["act"])
    dh = dy @ wd
    dg, du = dh * u * slope, dh * a
    out = {"dx": (dg @ wg + du @ wu).to(t), "dw_gate": (dg.t() @ x).to(t), "dw_up": (du.t() @ x).to(t), "dw_down": (dy.t() @ (a * u)).to(t)}
    if c["bias"]:
        out.update(db_gate=dg.sum(0).to(t), db_up=du.sum(0).to(t), db_down=dy.sum(0).to(t))
    return out


def _norm(s):
    norm = s["g"].double().square().sum().sqrt()
    scale = torch.clamp(s["case"]["clip"] / (norm + 1e-6), max=1.0) if s["case"]["clip"] else torch.ones_like(norm)
    return torch.stack([norm, scale]).float()


def _adamw(s):
    c, (b1, b2) = s["case"], BETAS
    s["step"] += 1
    norm = _norm(s) if c["clip"] else None
    g = s["g"].float()
    if norm is not None:
        g = g * norm[1]
    p = s["master"] if c["master"] else s["p"].float()
    if c["bits"] == 8:
        m, r = _values_m(s["m"], s["m_scale"]), _values_r(s["r"], s["r_scale"])
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    r = v.sqrt()
    denominator = r * (1.0 / math.sqrt(1.0 - b2 ** s["step"])) + EPS
    p = p * (1.0 - s["lr"] * s["decay"]) - (s["lr"] / (1.0 - b1 ** s["step"])) * (m / denominator)
    s["p"].copy_(p)
    if c["master"]:
        s["master"].copy_(p)
    if c["bits"] == 8:
        for codes, scale, new in ((s["m"], s["m_scale"], _codes_m(m)), (s["r"], s["r_scale"], _codes_r(r))):
            codes.copy_(new[0])
            scale.copy_(new[1])
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_out(s, norm)


def _adamw_out(s, norm):
    if s["case"]["bits"] == 8:
        out = {"p": s["p"], "m": s["m"], "m_scale": s["m_scale"], "r": _values_r(s["r"], s["r_scale"]), "r_scale": s["r_scale"]}
    else:
        out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if s["case"]["master"]:
        out["master"] = s["master"]
    if norm is not None:
        out["norm"] = norm
    return out


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"ffn_forward": _ffn_forward, "ffn_backward": _ffn_backward, "adamw": _adamw, "grad_norm": _norm}[op](s)
    if op == "ffn_forward":
        return s["ffn"].forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], b_gate=s["b_gate"], b_up=s["b_up"], b_down=s["b_down"])
    if op == "ffn_backward":
        return s["ffn"].backward(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["dy"], b_gate=s["b_gate"], b_up=s["b_up"])
    clip = s["case"]["clip"]
    if op == "grad_norm":
        return s["opt"].grad_norm(max_norm=clip or None)
    norm = None
    if clip:
        norm = s["opt"].grad_norm(max_norm=clip)
        s["opt"].step(grad_scale=norm[1:])
    else:
        s["opt"].step()
    return _adamw_out(s, norm)


def work(case):
    if case["op"].startswith("ffn"):
        n, d, f, b = case["rows"], case["d"], case["f"], BYTES[case["dtype"]]
        if case["op"] == "ffn_forward":
            return {"bytes": b * (2 * n * d + 3 * d * f + (2 * f + d if case["bias"] else 0)), "flops": 6 * n * d * f}
        # gate and up again (4), the gradient of their product (2), of x (4), of the three weights (6)
        return {"bytes": b * (3 * n * d + 6 * d * f + (4 * f + d if case["bias"] else 0)), "flops": 16 * n * d * f}
    n, p, g = case["total"], BYTES[case["dtype"]], BYTES[case["grads"]]
    if case["op"] == "grad_norm":
        return {"bytes": n * g, "flops": 2 * n}
    # each gradient counted once, also where the norm of all of them has to be known first
    weights = p + 8 if case["master"] else 2 * p
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (weights + g + state), "flops": 16 * n}


def exact(case, seed):
    """What run() returns for a new state, in 64 bits; the first moments' codes as the values before their rounding."""
    s, op = prepare(case, seed), case["op"]
    if op.startswith("ffn"):
        w = {k: (None if s[k] is None else s[k].double()) for k in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")}
        none = torch.zeros((), dtype=torch.float64, device="cuda")
        g = torch.addmm(none if w["b_gate"] is None else w["b_gate"], w["x"], w["w_gate"].t())
        u = torch.addmm(none if w["b_up"] is None else w["b_up"], w["x"], w["w_up"].t())
        if op == "ffn_backward":
            g.requires_grad_()
        a = {"silu": lambda z: z * torch.sigmoid(z), "gelu": torch.nn.functional.gelu, "relu": torch.relu,
             "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]](g)
        if op == "ffn_forward":
            return torch.addmm(none if w["b_down"] is None else w["b_down"], a * u, w["w_down"].t())
        dy = s["dy"].double()
        dh = torch.mm(dy, w["w_down"])
        dg, = torch.autograd.grad(a, g, dh * u)
        a = a.detach()
        du = dh * a
        out = {"dx": torch.addmm(torch.mm(dg, w["w_gate"]), du, w["w_up"]), "dw_gate": torch.mm(dg.t(), w["x"]), "dw_up": torch.mm(du.t(), w["x"]),
               "dw_down": torch.mm(dy.t(), a * u)}
        if case["bias"]:
            out.update(db_gate=dg.sum(0), db_up=du.sum(0), db_down=dy.sum(0))
        return out
    g = s["g"].double()
    norm = torch.dot(g, g).sqrt()
    scale = torch.minimum(torch.ones_like(norm), case["clip"] / (norm + 1e-6)) if case["clip"] else torch.ones_like(norm)
    both = torch.stack([norm, scale])
    if op == "grad_norm":
        return both
    if case["clip"]:
        g = g * scale
    t, (b1, b2) = s["step"] + 1, BETAS
    old = (s["master"] if case["master"] else s["p"]).double()
    if case["bits"] == 8:
        m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
        code = torch.arange(256, dtype=torch.float64, device="cuda")
        code = torch.where(code < 32, code, torch.ldexp(32 + code % 32, torch.div(code, 32, rounding_mode="floor") - 1))
        v = (code[s["r"].long()] * s["r_scale"].double().repeat_interleave(BLOCK)) ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g * g, v, b2)
    p = old - s["lr"] * s["decay"] * old - s["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    out = {"p": p}
    if case["bits"] == 8:
        for name, x, most in (("m", m, E4M3_MAX), ("r", v.sqrt(), ROOT_MAX)):
            top = torch.clamp(x.abs().view(-1, BLOCK).amax(1) / most, min=FLT_MIN)
            out[name], out[name + "_scale"] = (x.view(-1, BLOCK) / top[:, None]).view(-1), top
        out["r"] = None  # its codes are finer than e4m3's, but no value in 64 bits stands for their rounding
    else:
        out.update(m=m, v=v)
    if case["master"]:
        out["master"] = p
    if case["clip"]:
        out["norm"] = both
    return out

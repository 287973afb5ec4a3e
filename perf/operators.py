"""The feed-forward operators as cases that can be run and timed: the gated
feed-forward product and its backward pass (fp16), row quantisation to 8-bit
integers and the 8-bit integer product with token and channel scales.

Each case runs in two forms on the same inputs.  ``own`` false: elementary
torch operations in 32 bits, rounded once at the end.  ``own`` true: the calls
a user makes of pax_b200.  ``exact`` gives the same results from the
definitions in 64 bits.
"""
import torch

own = False

DEV = "cuda"
ACTS = ("silu", "gelu_tanh", "gelu_erf")


def listed():
    return [
        # H = act(X Wg) * (X Wu), X [m, d], Wg and Wu [d, f].
        # One new token in a mid-sized model's layer: weights are read once, latency counts.
        {"name": "glu_one_token", "op": "glu", "m": 1, "d": 2048, "f": 5504, "act": "silu", "save": False},
        # A decoding batch of 24 requests in a large layer: bound by the weights' bytes.
        {"name": "glu_decode_24", "op": "glu", "m": 24, "d": 4096, "f": 11264, "act": "silu", "save": False},
        # A prompt of ragged length in a layer whose widths divide by nothing but 8.
        {"name": "glu_prompt_777", "op": "glu", "m": 777, "d": 1544, "f": 4104, "act": "gelu_tanh", "save": False},
        # A training step's forward pass: the pre-activations are kept for the backward pass.
        {"name": "glu_train_4096", "op": "glu", "m": 4096, "d": 4096, "f": 11264, "act": "silu", "save": True},
        # The backward pass: dX, dWg and dWu from dH and the kept pre-activations.
        # A short sequence in a small model.
        {"name": "glu_back_130", "op": "glu_backward", "m": 130, "d": 768, "f": 2048, "act": "gelu_erf"},
        # A packed batch of odd length, ragged widths.
        {"name": "glu_back_2051", "op": "glu_backward", "m": 2051, "d": 2056, "f": 5480, "act": "gelu_tanh"},
        # A training step's micro-batch in a large layer.
        {"name": "glu_back_4096", "op": "glu_backward", "m": 4096, "d": 4096, "f": 8192, "act": "silu"},
        # Rows of fp16 activations to int8 codes and one fp32 scale each.
        # One token: a launch's latency.
        {"name": "quantize_one_token", "op": "quantize", "m": 1, "k": 4096},
        # A long prompt's activations: memory bound.
        {"name": "quantize_8192", "op": "quantize", "m": 8192, "k": 8192},
        # C = (A B^T) * sa[i] * sb[j] (+ bias[j]), A [m, k] and B [n, k] int8.
        # One token through a wide projection, with its bias.
        {"name": "i8_one_token", "op": "gemm_i8", "m": 1, "n": 16384, "k": 4096, "bias": True, "out": "f16"},
        # A ragged prompt against an output width that is odd (a vocabulary), fp32 results.
        {"name": "i8_prompt_1235", "op": "gemm_i8", "m": 1235, "n": 4099, "k": 2064, "bias": False, "out": "f32"},
        # A batch of long prompts: bound by the integer tensor pipe.
        {"name": "i8_prompt_8192", "op": "gemm_i8", "m": 8192, "n": 8192, "k": 4096, "bias": True, "out": "f16"},
    ]


def _log(rng, lo, hi, step=1):
    """A size between lo and hi, spread evenly over its logarithm, a multiple of step."""
    v = lo * (hi / lo) ** rng.random()
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["glu", "glu_backward", "quantize", "gemm_i8"])
    while True:
        if op == "glu":
            m = _log(rng, 1, 4096)
            c = {"op": op, "m": m, "d": _log(rng, 256, 4096, 8), "f": _log(rng, 256, 11264, 8), "act": rng.choice(ACTS),
                 "save": m > 64 and rng.random() < 0.5}
            if m * c["d"] * c["f"] <= 4096 * 4096 * 11264:
                return c
        elif op == "glu_backward":
            c = {"op": op, "m": _log(rng, 32, 4096), "d": _log(rng, 256, 4096, 8), "f": _log(rng, 256, 8192, 8),
                 "act": rng.choice(ACTS)}
            if c["m"] * c["d"] * c["f"] <= 4096 * 4096 * 8192:
                return c
        elif op == "quantize":
            c = {"op": op, "m": _log(rng, 1, 16384), "k": _log(rng, 64, 16384, 8)}
            if c["m"] * c["k"] <= 8192 * 8192:
                return c
        else:
            c = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 256, 16384, rng.choice([1, 8])), "k": _log(rng, 256, 8192, 16),
                 "bias": rng.random() < 0.5, "out": rng.choice(["f16", "f32"])}
            if c["m"] * c["n"] * c["k"] <= 8192 * 8192 * 4096:
                return c


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _activations(g, m, k):
    """Normalised activations with a few channels much larger than the rest; from 8 rows up, one padding row of zeros."""
    x = _randn(g, m, k)
    big = torch.randint(0, k, (max(1, k // 256),), generator=g, device=DEV)
    x[:, big] *= 12.0
    if m >= 8:
        x[3] = 0.0
    return x


def _codes(w):
    """int8 codes and scales of the rows of w, as a quantised model file holds them."""
    s = w.abs().amax(dim=1) / 127.0
    return torch.round(w / torch.where(s > 0, s, torch.ones_like(s))[:, None]).clamp_(-127, 127).to(torch.int8), s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, s = case, {"case": dict(case)}
    if c["op"] in ("glu", "glu_backward"):
        s["X"] = _randn(g, c["m"], c["d"]).half()
        s["Wg"] = (_randn(g, c["d"], c["f"]) * c["d"] ** -0.5).half()
        s["Wu"] = (_randn(g, c["d"], c["f"]) * c["d"] ** -0.5).half()
    if c["op"] == "glu_backward":
        # what the forward pass kept, and the gradient from above (loss-scaled, as fp16 training has it)
        s["G"] = (s["X"] @ s["Wg"]).contiguous()
        s["U"] = (s["X"] @ s["Wu"]).contiguous()
        s["dH"] = (_randn(g, c["m"], c["f"]) * 0.5).half()
    if c["op"] == "quantize":
        s["X"] = _activations(g, c["m"], c["k"]).half()
    if c["op"] == "gemm_i8":
        s["A"], s["sa"] = _codes(_activations(g, c["m"], c["k"]))
        s["B"], s["sb"] = _codes(_randn(g, c["n"], c["k"]) * c["k"] ** -0.5)
        s["bias"] = _randn(g, c["n"]).half() if c["bias"] else None
    return s


# ------------------------------------------------------------------ the plain form
def _act(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return 0.5 * x * (1.0 + torch.erf(x * 0.7071067811865476))


def _act_grad(x, act):
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-x))
        return p * (1.0 + x * (1.0 - p))
    if act == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x))
        return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * x * x)
    return 0.5 * (1.0 + torch.erf(x * 0.7071067811865476)) + x * torch.exp(-0.5 * x * x) * 0.3989422804014327


def _plain(s):
    c = s["case"]
    if c["op"] == "glu":
        x = s["X"].float()
        gate, up = x @ s["Wg"].float(), x @ s["Wu"].float()
        h = (_act(gate, c["act"]) * up).half()
        return {"H": h, "G": gate.half(), "U": up.half()} if c["save"] else {"H": h}
    if c["op"] == "glu_backward":
        gate, up, dh = s["G"].float(), s["U"].float(), s["dH"].float()
        dg = dh * up * _act_grad(gate, c["act"])
        du = dh * _act(gate, c["act"])
        xt = s["X"].float().t()
        dx = dg @ s["Wg"].float().t() + du @ s["Wu"].float().t()
        return {"dX": dx.half(), "dWg": (xt @ dg).half(), "dWu": (xt @ du).half()}
    if c["op"] == "quantize":
        x = s["X"].float()
        amax = x.abs().amax(dim=1, keepdim=True)
        q = torch.round(x * 127.0 / torch.where(amax > 0, amax, torch.ones_like(amax)))
        scale = amax / 127.0
        return {"values": q * scale, "scale": scale[:, 0]}
    acc = s["A"].float() @ s["B"].float().t()
    acc = acc * s["sa"][:, None] * s["sb"][None, :]
    if s["bias"] is not None:
        acc = acc + s["bias"].float()
    return {"C": acc.half() if c["out"] == "f16" else acc}


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    import pax_b200

    c = s["case"]
    if c["op"] == "glu":
        if c["save"]:
            h, gate, up = pax_b200.glu(s["X"], s["Wg"], s["Wu"], activation=c["act"], save=True)
            return {"H": h, "G": gate, "U": up}
        return {"H": pax_b200.glu(s["X"], s["Wg"], s["Wu"], activation=c["act"])}
    if c["op"] == "glu_backward":
        dx, dwg, dwu = pax_b200.glu_backward(s["dH"], s["X"], s["Wg"], s["Wu"], s["G"], s["U"], activation=c["act"])
        return {"dX": dx, "dWg": dwg, "dWu": dwu}
    if c["op"] == "quantize":
        # the codes are given as the values they stand for, which costs one more pass than the operator itself
        q, scale = pax_b200.quantize_rows(s["X"])
        return {"values": q * scale[:, None], "scale": scale}
    return {"C": pax_b200.gemm_i8(s["A"], s["B"], s["sa"], s["sb"], bias=s["bias"],
                                  out_dtype=torch.float16 if c["out"] == "f16" else torch.float32)}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work and exact values
def work(case):
    c = case
    if c["op"] == "glu":
        outs = 3 if c["save"] else 1
        return {"bytes": 2 * (c["m"] * c["d"] + 2 * c["d"] * c["f"] + outs * c["m"] * c["f"]), "flops": 4 * c["m"] * c["d"] * c["f"]}
    if c["op"] == "glu_backward":
        # reads dH, G, U, X, Wg, Wu; writes dX, dWg, dWu
        return {"bytes": 2 * (3 * c["m"] * c["f"] + 2 * c["m"] * c["d"] + 4 * c["d"] * c["f"]), "flops": 8 * c["m"] * c["d"] * c["f"]}
    if c["op"] == "quantize":
        return {"bytes": 3 * c["m"] * c["k"] + 4 * c["m"], "flops": 2 * c["m"] * c["k"]}
    out = 2 if c["out"] == "f16" else 4
    return {"bytes": c["k"] * (c["m"] + c["n"]) + out * c["m"] * c["n"] + 4 * (c["m"] + c["n"]) + (2 * c["n"] if c["bias"] else 0),
            "flops": 2 * c["m"] * c["n"] * c["k"]}


def _act64(x, act):
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu_tanh":
        return x * torch.sigmoid(2.0 * (2.0 / torch.pi) ** 0.5 * (x + 0.044715 * x.pow(3)))
    return x * 0.5 * torch.erfc(-x / 2.0 ** 0.5)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "glu":
        gate = torch.matmul(s["X"].double(), s["Wg"].double())
        up = torch.matmul(s["X"].double(), s["Wu"].double())
        out = {"H": _act64(gate, c["act"]) * up}
        return {**out, "G": gate, "U": up} if c["save"] else out
    if c["op"] == "glu_backward":
        gate = s["G"].double().requires_grad_(True)
        up = s["U"].double().requires_grad_(True)
        dg, du = torch.autograd.grad(_act64(gate, c["act"]) * up, (gate, up), s["dH"].double())
        x = s["X"].double()
        dx = torch.matmul(torch.cat([dg, du], 1), torch.cat([s["Wg"], s["Wu"]], 1).double().mT)
        return {"dX": dx, "dWg": torch.matmul(x.mT, dg), "dWu": torch.matmul(x.mT, du)}
    if c["op"] == "quantize":
        x = s["X"].double()
        scale = x.abs().max(dim=1).values / 127.0
        top = (scale * 127.0).clamp_min(1e-300)
        # a quotient of 127 times one 11-bit number by another is never within 2^-20 of a tie without being one
        q = torch.round(torch.round(x * 127.0 / top[:, None] * 2.0 ** 20) / 2.0 ** 20)
        return {"values": q * scale[:, None], "scale": scale}
    acc = torch.matmul(s["A"].double(), s["B"].double().mT)
    acc = acc * torch.outer(s["sa"].double(), s["sb"].double())
    if s["bias"] is not None:
        acc = acc + s["bias"].double()
    return {"C": acc}

"""Operators of a gated feed-forward block whose weights stay quantised in memory, as cases that can be timed and compared.

A case is a dict of plain values; its ``op`` says which operator it is:

  gated   h = act(x Wg^T + bg) * (x Wu^T + bu), Wg and Wu as ``QuantizedLinear`` packs them: what a decode step or a prompt calls
  train   the same with gradients for x and the biases: forward and backward; what the backward needs of the forward is kept in
          the activations' type, or with ``saved`` "8bit" in 8 bits
  grad    dx = dy W of one packed weight: the gradient that a frozen quantised layer passes on
  store   activations to 8 bits, and back: what a program keeps for a later backward pass

Weights: ``rows`` x ``cols`` codes, (w = code * scale, symmetric) with one fp16 scale for every ``group`` codes of the flattened
matrix; 4 and 2 bits packed low bits first with code + qmax, 8 bits one signed code a byte.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}
BLOCK = 64                     # values that share a scale in 8-bit storage


def _case(op, m, n, k, dtype, bits=4, group=128, act="silu", bias=False, saved="full"):
    """n x k weights (store: rows of n values) on m rows of activations."""
    return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bits": bits, "group": group, "act": act, "bias": bias, "saved": saved}


def listed():
    return [
        # one token through a 7B-shape block: what a decode step waits for
        dict(_case("gated", 1, 11008, 4096, "float16"), name="gated 7B, 1 row"),
        # the smallest call: a draft model's block at one token, launch and host time show
        dict(_case("gated", 1, 704, 512, "bfloat16", group=64), name="gated small, 1 row"),
        # a model kept at eight bits with finer scales, fp32 activations, a few rows, an output width of no round size
        dict(_case("gated", 5, 3001, 2752, "float32", bits=8, group=64, act="gelu", bias=True), name="gated 8-bit fp32, 5 rows"),
        # some two dozen sequences decoded together
        dict(_case("gated", 24, 11008, 4096, "bfloat16"), name="gated 7B, 24 rows"),
        # a prompt
        dict(_case("gated", 777, 11008, 4096, "float16", bias=True), name="gated 7B, prompt"),
        # a long prompt through the widest block: gate and up of a 70B-shape model
        dict(_case("gated", 2048, 28672, 8192, "bfloat16"), name="gated 70B, prompt"),
        # one block of a 7B-shape model while adapters around it are trained
        dict(_case("train", 2048, 11008, 4096, "bfloat16"), name="train 7B block"),
        # a smaller block with biases, short of memory: finer scales, sizes off every power of two
        dict(_case("train", 777, 2736, 1024, "float16", group=64, act="gelu", bias=True, saved="8bit"), name="train small, 8-bit kept"),
        # the gradient of a batch through one frozen projection
        dict(_case("grad", 512, 11008, 4096, "float16"), name="grad 7B layer"),
        # the same of a few rows through byte codes
        dict(_case("grad", 19, 4001, 2816, "bfloat16", bits=8, group=64), name="grad 8-bit, 19 rows"),
        # a 7B-shape block's intermediate activations of a batch
        dict(_case("store", 2048, 11008, 0, "bfloat16"), name="store 7B"),
        # a handful of rows of no round width
        dict(_case("store", 33, 1003, 0, "float32"), name="store small"),
    ]


def _log(rng, lo, hi):
    """An integer from lo to hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: one row to 2048, blocks of a hundred to 28672 rows and 256 to 8192 columns (training: the
    7B shape at most), each type, code width, group and activation, sizes off every power of two among them."""
    op = rng.choice(["gated", "gated", "gated", "gated", "train", "train", "grad", "grad", "store"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "store":
        return _case(op, _log(rng, 1, 2048), _log(rng, 64, 28672), 0, rng.choice(["float16", "bfloat16", "float32"]))
    bits, group = rng.choice([4, 4, 4, 4, 2, 8]), rng.choice([128, 128, 128, 64, 32])
    step = max(group, 128 if bits == 2 else 64)
    wide = op == "gated"
    n = _log(rng, 100, 28672 if wide else 11008)
    k = step * _log(rng, max(1, 256 // step), (8192 if wide else 4096) // step)
    few = rng.random() < (0.5 if op == "gated" else 0.2)
    m = rng.randint(1, 32) if few else _log(rng, 33, 2048)
    saved = rng.choice(["full", "8bit"]) if op == "train" else "full"
    if m <= 16 and saved == "full" and rng.random() < 0.2:
        dtype = "float32"
    return _case(op, m, n, k, dtype, bits, group, rng.choice(["silu", "silu", "gelu"]), rng.random() < 0.3 and op != "grad", saved)


def _weight(case, gen):
    """Packed codes and fp16 scales of one Gaussian matrix, quantised symmetrically to the largest magnitude of each group."""
    n, k, bits = case["n"], case["k"], case["bits"]
    qmax = (1 << (bits - 1)) - 1
    w = torch.randn(n * k // case["group"], case["group"], generator=gen, device="cuda") * 0.02
    scale = (w.abs().amax(1, keepdim=True) / qmax).to(torch.float16)
    q = torch.round(w / scale.float()).clamp_(-qmax, qmax).to(torch.int8).view(n, k)
    if bits == 8:
        return q, scale.flatten()
    u = (q + qmax).to(torch.uint8)
    if bits == 4:
        return u[:, 0::2] | (u[:, 1::2] << 4), scale.flatten()
    return u[:, 0::4] | (u[:, 1::4] << 2) | (u[:, 2::4] << 4) | (u[:, 3::4] << 6), scale.flatten()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]
    state = {"case": case}
    if op == "store":
        # activations: a bell with some channels far larger than the rest
        loud = torch.where(torch.rand(case["n"], generator=gen, device="cuda") < 0.01, 20.0, 1.0)
        state["x"] = (torch.randn(case["m"], case["n"], generator=gen, device="cuda") * loud).to(dt)
        return state
    state["gate"], state["gate_scales"] = _weight(case, gen)
    if op == "grad":
        state["dy"] = (torch.randn(case["m"], case["n"], generator=gen, device="cuda") * 1e-3).to(dt)
        return state
    state["up"], state["up_scales"] = _weight(case, gen)
    state["x"] = torch.randn(case["m"], case["k"], generator=gen, device="cuda").to(dt)
    state["gate_bias"] = (torch.randn(case["n"], generator=gen, device="cuda") * 0.1).to(dt) if case["bias"] else None
    state["up_bias"] = (torch.randn(case["n"], generator=gen, device="cuda") * 0.1).to(dt) if case["bias"] else None
    if op == "train":
        state["dh"] = (torch.randn(case["m"], case["n"], generator=gen, device="cuda") * 1e-3).to(dt)
        for name in ("x", "gate_bias", "up_bias"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# -- plain forms ----------------------------------------------------------------

def _dense(packed, scales, case):
    """The weight in 32 bits."""
    bits, qmax = case["bits"], (1 << (case["bits"] - 1)) - 1
    if bits == 4:
        q = torch.stack([packed & 15, packed >> 4], -1).reshape(case["n"], case["k"]).float() - qmax
    elif bits == 2:
        q = torch.stack([(packed >> s) & 3 for s in (0, 2, 4, 6)], -1).reshape(case["n"], case["k"]).float() - qmax
    else:
        q = packed.float()
    return (q.view(-1, case["group"]) * scales.float()[:, None]).view(case["n"], case["k"])


def _stored(x):
    """Rows in 32 bits as the values that their 8-bit form stands for: blocks of 64 of a row, code = round(127 x / largest)."""
    m, n = x.shape
    pad = -n % BLOCK
    b = torch.cat([x, x.new_zeros(m, pad)], 1).view(m, -1, BLOCK)
    most = b.abs().amax(-1, keepdim=True)
    top = torch.full_like(most, 127.0)                 # (a tensor: torch multiplies by the inverse of a number, which moves ties)
    codes = torch.round(b * top / torch.where(most > 0, most, 1.0))
    return (codes * (most / top)).view(m, -1)[:, :n]


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    c = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * c, c + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_gated(s):
    case, x = s["case"], s["x"].detach().float()
    wg, wu = _dense(s["gate"], s["gate_scales"], case), _dense(s["up"], s["up_scales"], case)
    g, u = x @ wg.T, x @ wu.T
    if case["bias"]:
        g, u = g + s["gate_bias"].detach().float(), u + s["up_bias"].detach().float()
    return wg, wu, g, u


def _plain(s):
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "store":
        return _stored(s["x"].float()).to(dt)
    if op == "grad":
        return (s["dy"].float() @ _dense(s["gate"], s["gate_scales"], case)).to(dt)
    wg, wu, g, u = _plain_gated(s)
    h = (_act(g, case["act"])[0] * u).to(dt)
    if op == "gated":
        return h
    if case["saved"] == "8bit":
        g, u = _stored(g), _stored(u)
    a, slope = _act(g, case["act"])
    dh = s["dh"].float()
    dg, du = dh * u * slope, dh * a
    out = [h, (dg @ wg + du @ wu).to(dt)]
    return out + [dg.sum(0).to(dt), du.sum(0).to(dt)] if case["bias"] else out


# -- the framework's calls --------------------------------------------------------

def _own(s):
    from eoq_quantization_b200 import gated

    case = s["case"]
    op, weight = case["op"], (case["n"], case["k"], case["bits"], case["group"])
    if op == "store":
        return gated.store_8bit(s["x"]).dequantize()
    if op == "grad":
        return gated.packed_input_grad(s["gate"], s["gate_scales"], *weight, s["dy"])
    h = gated.gated_packed(s["gate"], s["gate_scales"], s["up"], s["up_scales"], *weight, s["x"], s["gate_bias"], s["up_bias"],
                           activation=case["act"], saved=case["saved"])
    if op == "gated":
        return h
    leaves = [s["x"]] + ([s["gate_bias"], s["up_bias"]] if case["bias"] else [])
    return [h.detach(), *torch.autograd.grad(h, leaves, s["dh"])]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    m, n, k, e = case["m"], case["n"], case["k"], BYTES[case["dtype"]]
    if case["op"] == "store":
        return {"bytes": 2 * m * n * e, "flops": 4 * m * n}
    weight = n * k * case["bits"] // 8 + 2 * n * k // case["group"]
    if case["op"] == "grad":
        return {"bytes": weight + m * (n + k) * e, "flops": 2 * m * n * k}
    bias = 2 * n * e if case["bias"] else 0
    if case["op"] == "gated":
        return {"bytes": 2 * weight + m * (n + k) * e + bias, "flops": 4 * m * n * k}
    return {"bytes": 2 * weight + 2 * m * (n + k) * e + 2 * bias, "flops": 8 * m * n * k}


# -- in 64 bits, from the definition -----------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        f64 = torch.float64

        def matrix(packed, scales):
            if case["bits"] == 8:
                codes = packed.to(f64)
            else:
                per, top = 8 // case["bits"], 2 ** case["bits"]
                codes = torch.empty(case["n"], case["k"], dtype=f64, device="cuda")
                rest = packed.to(torch.int32)
                for j in range(per):
                    codes[:, j::per] = (rest % top).to(f64) - (top // 2 - 1)
                    rest = rest // top
            return codes * scales.to(f64).repeat_interleave(case["group"]).view(case["n"], case["k"])

        def eight(v):
            out = torch.empty_like(v)
            for at in range(0, v.shape[1], BLOCK):
                part = v[:, at:at + BLOCK]
                largest = part.abs().max(dim=1, keepdim=True).values
                out[:, at:at + BLOCK] = torch.round(127 * part / largest.clamp_min(1e-300)) * largest / 127
            return out

        if case["op"] == "store":
            return eight(s["x"].to(f64))
        wg = matrix(s["gate"], s["gate_scales"])
        if case["op"] == "grad":
            return s["dy"].to(f64) @ wg
        wu, x = matrix(s["up"], s["up_scales"]), s["x"].detach().to(f64)
        g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
        if case["bias"]:
            g += s["gate_bias"].detach().to(f64)
            u += s["up_bias"].detach().to(f64)
        if case["act"] == "silu":
            value, slope = (lambda t: t * torch.sigmoid(t)), (lambda t: torch.sigmoid(t) + t * torch.sigmoid(t) * torch.sigmoid(-t))
        else:
            normal = torch.distributions.Normal(torch.zeros((), dtype=f64, device="cuda"), torch.ones((), dtype=f64, device="cuda"))
            value, slope = (lambda t: t * normal.cdf(t)), (lambda t: normal.cdf(t) + t * torch.exp(normal.log_prob(t)))
        h = value(g) * u
        if case["op"] == "gated":
            return h
        if case["saved"] == "8bit":
            g, u = eight(g), eight(u)
        dh = s["dh"].to(f64)
        dg, du = dh * u * slope(g), dh * value(g)
        back = [h, torch.matmul(dg, wg) + torch.matmul(du, wu)]
        return back + [dg.sum(dim=0), du.sum(dim=0)] if case["bias"] else back

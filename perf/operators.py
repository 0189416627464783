"""Cases of the int8 operators with a scale for each token and channel, and their plain forms.

The operators (``sigcomp_b200.int8``):

* ``quantize_tokens`` / ``dequantize_tokens``: a row of activations held in 8 bits with one scale.
  ``s = fl(max|x| / 127)``, ``r = fl(127 / max|x|)`` (fl: rounded to 32 bits; the maximum at least
  2**-100) and ``q = rint(x * r)``, the product taken exactly and ties going to the even number;
  the row stands for ``q * s``.
* ``int8_linear``: ``y[i, j] = relu((sum_k q[i, k] w[j, k]) * s[i] * t[j] + b[j])`` with int8 rows
  ``q`` and ``w``, their scales ``s`` (token) and ``t`` (channel), and a result in 16 or 32 bits.
  Rows given as floats are quantised first, as by ``quantize_tokens``.
* ``int8_linear_requant``: the same product, whose rows come back quantised: with a scale for each
  token, or with one given scale (``rint(y / scale)`` saturated), the form an entropy model's
  logits have.

Every sum of products is a whole number and exact, so a token's result depends neither on the rows
beside it nor on how the work is split: coding a batch and decoding token by token agree.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
# a maximum below this quantises like this one, so that 127 / max stays finite
SMALLEST = 2.0 ** -100


def listed():
    return [
        # one decoding step's window of embeddings, 64 positions of 128
        {"name": "values-token", "op": "values", "rows": 1, "k": 8192, "type": "bf16", "pad": 0},
        # a compress group's hidden activations, held in 8 bits between layers
        {"name": "values-batch", "op": "values", "rows": 262144, "k": 512, "type": "fp16", "pad": 0},
        # the first layer of an entropy model for a single token
        {"name": "linear-token", "op": "linear", "rows": 1, "k": 8192, "n": 512, "type": "bf16", "relu": True,
         "bias": True, "pad": 0},
        # a square projection for a handful of streams decoded in step
        {"name": "linear-few", "op": "linear", "rows": 24, "k": 4096, "n": 4096, "type": "fp16", "relu": False,
         "bias": False, "pad": 0},
        # a ragged calibration batch in 32 bits, rows cut from a wider buffer
        {"name": "linear-odd", "op": "linear", "rows": 1001, "k": 1000, "n": 777, "type": "fp32", "relu": False,
         "bias": True, "pad": 3},
        # the first layer over a compress group: 64 K windows of 8,192 inputs
        {"name": "product-batch", "op": "product", "rows": 65536, "k": 8192, "n": 512, "type": "bf16", "relu": True,
         "bias": True},
        # a square product, as large models have it
        {"name": "product-square", "op": "product", "rows": 4096, "k": 4096, "n": 4096, "type": "bf16",
         "relu": False, "bias": False},
        # a hidden layer over a compress group, int8 in and int8 out
        {"name": "requant-batch", "op": "requant", "rows": 262144, "k": 512, "n": 512, "relu": True, "bias": True,
         "static": False},
        # a hidden layer for a few streams decoded in step
        {"name": "requant-few", "op": "requant", "rows": 16, "k": 512, "n": 512, "relu": True, "bias": True,
         "static": False},
        # a wider layer over an odd number of rows
        {"name": "requant-wide", "op": "requant", "rows": 2001, "k": 1536, "n": 2304, "relu": False, "bias": True,
         "static": False},
        # three layers in a row, the step of one stream and of a full batch of 20,480 chunks
        {"name": "mlp-token", "op": "mlp", "rows": 1, "k": 8192, "n": 512, "out": 256, "type": "bf16"},
        {"name": "mlp-batch", "op": "mlp", "rows": 20480, "k": 8192, "n": 512, "out": 256, "type": "bf16"},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["values", "linear", "linear", "product", "product", "requant", "requant", "mlp"])
    rows, k = _log(rng, 1, 262144), _log(rng, 1, 8192)
    if rng.random() < 0.5:
        k = min(8192, 64 * math.ceil(k / 64))
    rows = max(1, min(rows, (1 << 27) // k))
    case = {"op": op, "rows": rows, "k": k}
    if op != "values":
        n = min(_log(rng, 1, 8192), max(1, (1 << 27) // rows))
        if rng.random() < 0.5:
            n = 16 * math.ceil(n / 16)
        # no more products than the largest listed case has
        case["rows"] = max(1, min(rows, 65536 * 8192 * 512 // (k * n)))
        case["n"] = n
    if op in ("values", "linear"):
        case["pad"] = rng.choice([0, 0, 1, 8, 24])
    if op == "mlp":
        case["out"] = _log(rng, 1, 1024)
        case["n"] = n = min(case["n"], 2048)
        case["rows"] = max(1, min(case["rows"], 65536 * 8192 * 512 // (n * (k + n + case["out"]))))
    else:
        if op in ("linear", "product", "requant"):
            case["relu"], case["bias"] = rng.random() < 0.5, rng.random() < 0.7
        if op == "requant":
            case["static"] = rng.random() < 0.3
    if op != "requant":
        case["type"] = rng.choice(["bf16", "fp16", "fp32"]) if op != "mlp" else rng.choice(["bf16", "fp16"])
    return case


# ---- inputs -----------------------------------------------------------------------------------

def _int8_rows(gen, rows, cols, spread):
    """int8 rows of a bell shape within +-127; rows start 16 bytes apart or a multiple of that, as
    ``quantize_tokens`` lays them out."""
    q = torch.zeros((rows, -(-cols // 16) * 16), dtype=torch.int8, device="cuda")[:, :cols]
    step = max(1, (1 << 26) // cols)
    for i in range(0, rows, step):
        part = torch.empty((min(step, rows - i), cols), dtype=torch.float16, device="cuda")
        q[i:i + step] = part.normal_(0, spread, generator=gen).round_().clamp_(-127, 127)
    return q


def _float_rows(gen, rows, cols, kind, pad):
    """Activations: a magnitude for each token, a few strong channels, one token of zeros."""
    x = torch.empty((rows, cols + pad), dtype=TYPES[kind], device="cuda").normal_(0, 1, generator=gen)[:, :cols]
    x *= torch.empty((rows, 1), device="cuda").normal_(0, 1, generator=gen).exp_().to(x.dtype)
    x[:, 3::97] *= 6
    if rows > 2:
        x[rows // 2] = 0
    return x


def _layer(gen, n, k, bias):
    """int8 weights, a scale for each channel that keeps results of order one, and a bias."""
    w = _int8_rows(gen, n, k, 36.0)
    t = torch.empty(n, device="cuda").uniform_(0.5, 1.5, generator=gen) * (3.0 / (36.0 * math.sqrt(k)))
    return w, t, torch.empty(n, device="cuda").normal_(0, 0.5, generator=gen) if bias else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, rows, k = case["op"], case["rows"], case["k"]
    state = {"case": dict(case)}
    if op in ("values", "linear", "mlp"):
        state["x"] = _float_rows(gen, rows, k, case["type"], case.get("pad", 0))
    else:
        state["q"] = _int8_rows(gen, rows, k, 40.0)
        state["s"] = torch.empty(rows, device="cuda").uniform_(0.2, 3.0, generator=gen) / 127
    if op != "values":
        state["layer"] = _layer(gen, case["n"], k, case.get("bias", True))
    if op == "mlp":
        state["hidden"] = _layer(gen, case["n"], case["n"], True)
        state["last"] = _layer(gen, case["out"], case["n"], True)
    if case.get("static"):
        state["scale"] = 0.06
    return state


# ---- the plain forms --------------------------------------------------------------------------

def _quantize(x):
    top = x.float().abs().amax(dim=1).clamp_min(SMALLEST)
    # a tensor of 127, since a division by or of a plain number is done with a rounded reciprocal
    most = torch.full_like(top, 127)
    # the product of two 32-bit numbers is exact in 64, so only rint() rounds
    q = (x.double() * (most / top).double()[:, None]).round()
    return q.to(torch.int8), top / most


def _dequantize(q, s, kind):
    return (q.float() * s[:, None]).to(kind)


def _linear(q, s, w, t, b, relu):
    """The result in 32 bits: whole sums in 64 (32 lose them from 2**24 on), rounded once, times the
    token's scale, then times the channel's plus the bias with one rounding."""
    total = (q.double() @ w.double().t()).float()
    y = (total * s[:, None]).double() * t.double()
    y = (y if b is None else y + b.double()).float()
    return y.relu() if relu else y


def _plain(state):
    case, kind = state["case"], TYPES.get(state["case"].get("type"), torch.bfloat16)
    op = case["op"]
    if op in ("values", "linear", "mlp"):
        q, s = _quantize(state["x"])
    else:
        q, s = state["q"], state["s"]
    if op == "values":
        return {"values": _dequantize(q, s, kind), "scales": s}
    if op == "mlp":
        q, s = _quantize(_linear(q, s, *state["layer"], True))
        q, s = _quantize(_linear(q, s, *state["hidden"], True))
        return _linear(q, s, *state["last"], False).to(kind)
    y = _linear(q, s, *state["layer"], case["relu"])
    if op != "requant":
        return y.to(kind)
    if case["static"]:
        s = torch.full((1,), state["scale"], device="cuda")
        return _dequantize((y / s).round().clamp_(-128, 127), s, kind)
    q, s = _quantize(y)
    return {"values": _dequantize(q, s, kind), "scales": s}


def run(state):
    if not own:
        return _plain(state)
    from sigcomp_b200.int8 import dequantize_tokens, int8_linear, int8_linear_requant, quantize_tokens
    case = state["case"]
    op = case["op"]
    if op == "values":
        q, s = quantize_tokens(state["x"])
        return {"values": dequantize_tokens(q, s, dtype=state["x"].dtype), "scales": s}
    if op == "linear":
        return int8_linear(state["x"], *state["layer"], relu=case["relu"])
    if op == "product":
        return int8_linear(state["q"], *state["layer"], x_scales=state["s"], relu=case["relu"],
                           dtype=TYPES[case["type"]])
    if op == "mlp":
        q, s = quantize_tokens(state["x"])
        q, s = int8_linear_requant(q, s, *state["layer"], relu=True)
        q, s = int8_linear_requant(q, s, *state["hidden"], relu=True)
        return int8_linear(q, *state["last"], x_scales=s, dtype=TYPES[case["type"]])
    if case["static"]:
        q = int8_linear_requant(state["q"], state["s"], *state["layer"], relu=case["relu"],
                                output_scale=state["scale"])
        return dequantize_tokens(q, state["scale"], dtype=torch.bfloat16)
    q, s = int8_linear_requant(state["q"], state["s"], *state["layer"], relu=case["relu"])
    return {"values": dequantize_tokens(q, s, dtype=torch.bfloat16), "scales": s}


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    op, rows, k = case["op"], case["rows"], case["k"]
    e = SIZES.get(case.get("type"), 2)
    if op == "values":
        return {"bytes": rows * (2 * k * e + 4), "flops": 0}
    n = case["n"]
    layers = [(k, n, case.get("bias", True))]
    if op == "mlp":
        layers += [(n, n, True), (n, case["out"], True)]
    weights = sum(b * (a + 4 + 4 * bias) for a, b, bias in layers)
    rows_in = k * e if op in ("linear", "mlp") else k + 4
    rows_out = layers[-1][1] * e + (4 if op == "requant" and not case["static"] else 0)
    return {"bytes": rows * (rows_in + rows_out) + weights, "flops": 2 * rows * sum(a * b for a, b, _ in layers)}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _held(x):
    """(whole numbers, scale, reciprocal) of rows in 64 bits; scale and reciprocal are 32-bit numbers
    by definition."""
    top = torch.linalg.vector_norm(x, ord=math.inf, dim=-1, keepdim=True)
    top = torch.where(top < SMALLEST, torch.full_like(top, SMALLEST), top)
    s, r = (top / 127).float().double(), (127 / top).float().double()
    return torch.round(x * r), s


def _affine(q, s, w, t, b, relu):
    y = torch.einsum("ik,jk->ij", q, w.to(torch.float64)) * (s * t.to(torch.float64))
    if b is not None:
        y = y + b.to(torch.float64)
    return torch.where(y < 0, torch.zeros_like(y), y) if relu else y


def _exact_rows(state, i, j):
    case = state["case"]
    op = case["op"]
    if op in ("values", "linear", "mlp"):
        q, s = _held(state["x"][i:j].to(torch.float64))
    else:
        q, s = state["q"][i:j].to(torch.float64), state["s"][i:j, None].to(torch.float64)
    if op == "values":
        return {"values": q * s, "scales": s[:, 0]}
    if op == "mlp":
        q, s = _held(_affine(q, s, *state["layer"], True))
        q, s = _held(_affine(q, s, *state["hidden"], True))
        return _affine(q, s, *state["last"], False)
    y = _affine(q, s, *state["layer"], case["relu"])
    if op != "requant":
        return y
    if case["static"]:
        return torch.round(y / state["scale"]).clamp(-128, 127) * state["scale"]
    q, s = _held(y)
    return {"values": q * s, "scales": s[:, 0]}


def exact(case, seed):
    state = prepare(case, seed)
    step = max(1, (1 << 26) // max(case["k"], case.get("n", 1)))
    parts = [_exact_rows(state, i, min(i + step, case["rows"])) for i in range(0, case["rows"], step)]
    if isinstance(parts[0], dict):
        return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    return torch.cat(parts)

"""What the products in 8-bit integers are measured on: one call of an operator, with the inputs that a step of a model brings to it.

Weights are held as integers in -127..127 with one scale for each output channel; activations are rounded to such integers row by
row, within the call, with one scale for each row (token): the row's largest magnitude / 127.  The product of the integers is exact,
and one multiplication by both scales makes the result.  Kinds of case:

  linear    rows in 16 or 32 bits -> rounded -> times the weights: a projection
  norm      32-bit rows of the residual stream -> RMS norm -> rounded -> times the weights: a layer's input projection
  swiglu    rows -> rounded -> times the gate's and the up projection's weights -> silu(gate) * up: the front of a feed-forward
  experts   router logits and rows -> every row's chosen experts, gated feed-forwards of two products with the activation rounded
            between them: the result of every (row, choice) pair

The plain form and exact() are written from these definitions.
"""
import math

import torch

own = False


def _linear(name, rows, k, n, x="bfloat16", out="bfloat16", bias=False):
    case = dict(kind="linear", rows=rows, k=k, n=n, x=x, out=out, bias=bias)
    return dict(case, name=name) if name else case


def _norm(name, rows, k, n):
    case = dict(kind="norm", rows=rows, k=k, n=n)
    return dict(case, name=name) if name else case


def _swiglu(name, rows, k, f):
    case = dict(kind="swiglu", rows=rows, k=k, f=f)
    return dict(case, name=name) if name else case


def _experts(name, rows, k, f, experts, top, weight_on="output"):
    case = dict(kind="experts", rows=rows, k=k, f=f, experts=experts, top=top, weight_on=weight_on)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one sequence decodes: a narrow projection, the smallest call
        _linear("linear-1", 1, 2048, 2048),
        # a batch of 24 decodes: the projection back from a wide feed-forward
        _linear("linear-24", 24, 8192, 2560),
        # short prompts, rows and columns that fill no tile, a 32-bit result with a bias
        _linear("linear-333", 333, 2560, 1537, x="float32", out="float32", bias=True),
        # a long prompt through the widest projection: the largest call
        _linear("linear-8192", 8192, 2560, 16384),
        # five sequences decode: a layer's input projection from the residual stream
        _norm("norm-5", 5, 2048, 8240),
        # a prompt of 2,048 tokens
        _norm("norm-2048", 2048, 2048, 8240),
        # one sequence decodes: gate and up
        _swiglu("swiglu-1", 1, 2048, 4096),
        # prompts together, an odd number of rows
        _swiglu("swiglu-1031", 1031, 2560, 8192),
        # one sequence decodes: four experts of 32
        _experts("experts-1", 1, 2048, 1024, 32, 4),
        # a batch decodes: nearly every expert, a few rows each
        _experts("experts-37", 37, 2048, 1024, 32, 4, "input"),
        # many small experts, a prompt that leaves ragged groups
        _experts("experts-777", 777, 2048, 688, 64, 6, "input"),
        # long prompts, hundreds of rows an expert
        _experts("experts-4096", 4096, 2048, 1024, 32, 4),
    ]


_MOST = 2 * 8192 * 2560 * 16384          # operations of the largest listed case


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "swiglu", "experts", "experts"])
    rows = _log_int(rng, 1, 8192)
    k = 16 * _log_int(rng, 16, 512)
    if kind == "experts":
        experts, rows = rng.choice([4, 8, 16, 32, 64, 128]), _log_int(rng, 1, 4096)
        top = rng.randint(1, min(8, experts))
        k, f = 16 * rng.randint(32, 160), 8 * rng.randint(32, 256)
        while experts * k * f > 1 << 28:
            experts //= 2
        top = min(top, experts)
        while 6 * rows * top * k * f > _MOST // 4:
            rows //= 2
        return _experts(None, rows, k, f, experts, top, rng.choice(["input", "output"]))
    n = _log_int(rng, 128, 16384)
    if rng.random() < 0.25:
        k -= rng.randint(1, 15)          # rows of odd lengths
    while 2 * rows * k * n > _MOST:
        rows //= 2
    if kind == "norm":
        return _norm(None, rows, k, n)
    if kind == "swiglu":
        return _swiglu(None, rows, k, max(64, 8 * (n // 16)))
    return _linear(None, rows, k, n, rng.choice(["bfloat16", "float32"]), rng.choice(["bfloat16", "float32"]), rng.random() < 0.4)


# ---- inputs ------------------------------------------------------------------------------------------
_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rows(g, rows, k, dtype):
    """Activations as a model's are: columns of unequal size, a few of them many times the others."""
    x = torch.empty(rows, k, device="cuda").normal_(generator=g)
    size = torch.empty(k, device="cuda").normal_(0.0, 0.5, generator=g).exp_()
    outliers = torch.rand(k, generator=g, device="cuda") < 0.004
    return (x * torch.where(outliers, size * 8.0, size)).to(dtype)


def _weights(g, *shape):
    """(integers, a scale per output channel) of N(0, 0.02) weights, rows starting on 16-byte boundaries."""
    n, k = math.prod(shape[:-1]), shape[-1]
    q = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    scale = torch.empty(n, device="cuda")
    for at in range(0, n, 16384):
        w = torch.empty(min(16384, n - at), k, device="cuda").normal_(0.0, 0.02, generator=g)
        s = w.abs().amax(1) / 127.0
        q[at:at + 16384, :k] = torch.round(w / s[:, None]).clamp_(-127, 127).to(torch.int8)
        scale[at:at + 16384] = s
    return q.view(*shape[:-1], -1)[..., :k], scale.view(shape[:-1])


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case)
    if case["kind"] == "linear":
        s["x"] = _rows(g, case["rows"], case["k"], _TYPES[case["x"]])
        s["w"], s["w_scale"] = _weights(g, case["n"], case["k"])
        s["bias"] = torch.empty(case["n"], device="cuda").normal_(generator=g) if case["bias"] else None
    elif case["kind"] == "norm":
        s["x"] = _rows(g, case["rows"], case["k"], torch.float32)
        s["norm"] = torch.empty(case["k"], device="cuda").normal_(1.0, 0.1, generator=g)
        s["w"], s["w_scale"] = _weights(g, case["n"], case["k"])
    elif case["kind"] == "swiglu":
        s["x"] = _rows(g, case["rows"], case["k"], torch.bfloat16)
        s["w"], s["w_scale"] = _weights(g, 2 * case["f"], case["k"])             # the gate's rows, then the up projection's
    else:
        e, f, k = case["experts"], case["f"], case["k"]
        s["x"] = _rows(g, case["rows"], k, torch.bfloat16)
        # some experts are chosen several times as often as others
        s["logits"] = torch.empty(case["rows"], e, device="cuda").normal_(generator=g) + torch.empty(e, device="cuda").normal_(0.0, 0.5, generator=g)
        s["gate_up"], s["gate_up_scale"] = _weights(g, e, 2 * f, k)
        s["down"], s["down_scale"] = _weights(g, e, k, f)
        # room for an expert's rows in the plain form: those of the most chosen one
        s["most"] = int(torch.bincount(s["logits"].topk(case["top"]).indices.flatten(), minlength=e).max())
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def _int8(x):
    """The integers and the scales of rows of 32-bit values."""
    largest = x.abs().amax(-1, keepdim=True)
    scale = largest / largest.new_full((), 127.0)                               # (a quotient: by a number torch would multiply by 1 / 127)
    return torch.where(scale > 0, torch.round(x / scale), 0.0), scale


def _product(x, w, w_scale):
    q, scale = _int8(x)
    return (q @ w.float().transpose(-1, -2)) * scale * w_scale.unsqueeze(-2)


def _gated(y):
    gate, up = y.chunk(2, -1)
    return gate * torch.sigmoid(gate) * up


def _plain(s):
    case, x = s["case"], s["x"].float()
    if case["kind"] == "linear":
        y = _product(x, s["w"], s["w_scale"])
        return (y if s["bias"] is None else y + s["bias"]).to(_TYPES[case["out"]])
    if case["kind"] == "norm":
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * s["norm"]
        return _product(x, s["w"], s["w_scale"]).to(torch.bfloat16)
    if case["kind"] == "swiglu":
        return _gated(_product(x, s["w"], s["w_scale"])).to(torch.bfloat16)
    rows, top, e = case["rows"], case["top"], case["experts"]
    best = s["logits"].topk(top)
    weight = torch.softmax(best.values, -1).flatten()
    expert = best.indices.flatten()                                             # of every (row, choice) pair
    order = torch.argsort(expert, stable=True)
    start = torch.searchsorted(expert[order], torch.arange(e, device="cuda"))
    place = torch.empty_like(order)
    place[order] = torch.arange(rows * top, device="cuda")
    place = place - start[expert]                                               # which of its expert's rows a pair is
    grouped = x.new_zeros(e, s["most"], x.shape[1])
    grouped[expert, place] = x.repeat_interleave(top, 0)
    y = _product(grouped, s["gate_up"], s["gate_up_scale"])
    if case["weight_on"] == "input":
        shares = x.new_zeros(e, s["most"], 1)
        shares[expert, place, 0] = weight
        y = y * shares
    y = _product(_gated(y), s["down"], s["down_scale"])[expert, place]
    if case["weight_on"] == "output":
        y = y * weight[:, None]
    return y.view(rows, top, -1).to(torch.bfloat16)


def _own(s):
    from tinyllama_c_b200 import ops
    case, x = s["case"], s["x"]
    if case["kind"] == "linear":
        out = torch.empty(case["rows"], case["n"], dtype=_TYPES[case["out"]], device="cuda")
        ops.linear_int8(x, s["w"], s["w_scale"], out, colbias=s["bias"])
    elif case["kind"] == "norm":
        out = torch.empty(case["rows"], case["n"], dtype=torch.bfloat16, device="cuda")
        q, scale = ops.rmsnorm_int8(x, s["norm"], 1e-5)
        ops.linear_int8(q, s["w"], s["w_scale"], out, a_scale=scale)
    elif case["kind"] == "swiglu":
        out = torch.empty(case["rows"], case["f"], dtype=torch.bfloat16, device="cuda")
        ops.linear_swiglu_int8(x, s["w"], s["w_scale"], out)
    else:
        out = torch.empty(case["rows"], case["top"], case["k"], dtype=torch.bfloat16, device="cuda")
        routing = ops.moe_route(s["logits"], case["experts"], case["top"], weights="softmax")
        ops.moe_experts_int8(x, s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"], routing, case["top"], out,
                             weight_on=case["weight_on"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = dict(bfloat16=2, float32=4)
    m, k = case["rows"], case["k"]
    if case["kind"] == "experts":
        e, f, top = case["experts"], case["f"], case["top"]
        used = e * (1.0 - (1.0 - 1.0 / e) ** (m * top))                         # experts that some row chooses
        return {"bytes": 2 * m * k + 4 * m * e + used * (3 * f * k + 4 * (2 * f + k)) + 2 * m * top * k, "flops": 6 * m * top * k * f}
    n = 2 * case["f"] if case["kind"] == "swiglu" else case["n"]
    x = size[case["x"]] if case["kind"] == "linear" else 4 if case["kind"] == "norm" else 2
    out = size[case["out"]] * n if case["kind"] == "linear" else 2 * n if case["kind"] == "norm" else n
    return {"bytes": x * m * k + n * k + 4 * n + out * m, "flops": 2 * m * k * n}


# ---- in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()

    def product(rows, w, w_scale):
        largest = rows.abs().max(dim=1).values
        step = largest / 127
        q = torch.round(rows / torch.where(step == 0, torch.ones_like(step), step)[:, None])
        return torch.mm(q, w.double().t()).mul_(step[:, None]).mul_(w_scale.double()[None, :])

    def silu_times(y):
        half = y.shape[1] // 2
        return y[:, :half] / (1 + torch.exp(-y[:, :half])) * y[:, half:]

    if case["kind"] == "linear":
        y = product(x, s["w"], s["w_scale"])
        return y if s["bias"] is None else y + s["bias"].double()
    if case["kind"] == "norm":
        x = x * torch.rsqrt((x * x).sum(1, keepdim=True) / x.shape[1] + 1e-5) * s["norm"].double()
        return product(x, s["w"], s["w_scale"])
    if case["kind"] == "swiglu":
        return silu_times(product(x, s["w"], s["w_scale"]))
    # expert by expert, the rows that chose it
    logits = s["logits"].double()
    ranked = torch.sort(logits, dim=1, descending=True, stable=True)
    picked, values = ranked.indices[:, :case["top"]], ranked.values[:, :case["top"]]
    share = torch.exp(values - values[:, :1])
    share = share / share.sum(1, keepdim=True)
    y = torch.zeros(case["rows"], case["top"], case["k"], dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        row, choice = torch.nonzero(picked == e, as_tuple=True)
        if not len(row):
            continue
        gu = product(x[row], s["gate_up"][e], s["gate_up_scale"][e])
        weight = share[row, choice][:, None]
        if case["weight_on"] == "input":
            gu = gu * weight
        result = product(silu_times(gu), s["down"][e], s["down_scale"][e])
        y[row, choice] = result if case["weight_on"] == "input" else result * weight
    return y

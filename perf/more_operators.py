"""What a decoder's training step needs between its table and its losses, and the optimizer of its matrices, as measurable cases.

A case is a dict; "op" says which operator one pass goes through:

  layerNorm      rows less their mean, over their deviation, times a weight, plus a bias
  layerNormGrad  the gradient of its input, weight and bias
  rotary         heads turned by their token's position ("inverse": back, which is the gradient)
  orthogonalize  Newton-Schulz products that bring the singular values of matrices near 1
  muon           one step of that optimizer: momentum, orthogonalised update, decay
"""
import math

import torch

own = False

TORCH = {"float": torch.float32, "half": torch.float16, "long": torch.int64, "double": torch.float64}
SIZE = {"float": 4, "half": 2}
EPS = 1e-5                       # of the norms
NS = (3.4445, -4.7750, 2.0315)   # of the odd polynomial that a Newton-Schulz step is
NS_STEPS, NS_EPS = 5, 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.1
GRAD_SCALE = 1.0 / 128           # the gradients come from a loss times 128


def listed():
    return [
        # the newest tokens of 24 sequences that are being generated: launch latency
        {"name": "layernorm-decode-24", "op": "layerNorm", "type": "half", "rows": 24, "dim": 2048},
        # a training batch of 8 sequences of 2049 tokens
        {"name": "layernorm-batch-16k", "op": "layerNorm", "type": "half", "rows": 16392, "dim": 2048},
        # a micro-batch of a small model, its weights' gradients added to those of the ones before it; rows off the 16-byte grid
        {"name": "layernorm-grad-add-odd", "op": "layerNormGrad", "type": "float", "rows": 1500, "dim": 513, "accumulate": True},
        # a training batch of a larger model
        {"name": "layernorm-grad-16k", "op": "layerNormGrad", "type": "half", "rows": 16392, "dim": 4096, "accumulate": False},
        # the newest tokens' queries and keys, far along a context that was made 8 times longer
        {"name": "rotary-decode-24", "op": "rotary", "type": "half", "tokens": 24, "heads": 40, "behind": 8, "dim": 128, "turned": 128,
         "context": 131072, "factor": 8.0, "interleaved": False, "inverse": False},
        # the same heads of a training batch, within a fused projection whose values lie behind them
        {"name": "rotary-batch-16k", "op": "rotary", "type": "half", "tokens": 16392, "heads": 40, "behind": 8, "dim": 128, "turned": 128,
         "context": 4096, "factor": 1.0, "interleaved": False, "inverse": False},
        # the gradient of a small model's queries: pairs side by side, half of an odd head turned
        {"name": "rotary-inverse-odd", "op": "rotary", "type": "float", "tokens": 1500, "heads": 9, "behind": 0, "dim": 101, "turned": 50,
         "context": 2048, "factor": 1.0, "interleaved": True, "inverse": True},
        # each head's matrix of a small model on its own
        {"name": "orthogonalize-heads", "op": "orthogonalize", "type": "float", "batch": 12, "rows": 65, "cols": 513},
        # a large model's matrix, taller than wide
        {"name": "orthogonalize-half-tall", "op": "orthogonalize", "type": "half", "batch": 1, "rows": 8192, "cols": 2048},
        # a square one in float
        {"name": "orthogonalize-float-4k", "op": "orthogonalize", "type": "float", "batch": 1, "rows": 4096, "cols": 4096},
        # the step of a small model: some tens of small odd matrices
        {"name": "muon-small", "op": "muon", "type": "float", "layers": 2, "width": 65, "master": False},
        # the step of a large one in half precision with float copies of the parameters
        {"name": "muon-half-150m", "op": "muon", "type": "half", "layers": 12, "width": 1024, "master": True},
    ]


def _log(rng, low, high):
    """A whole number between low and high, even over its logarithm; two times in three as it falls, else a multiple of 8 or 64."""
    n = min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))
    if rng.random() < 2 / 3:
        return n
    step = 64 if n >= 256 else 8
    return min(high, max(low, n // step * step))


def draw(rng):
    op = rng.choice(("layerNorm", "layerNormGrad", "rotary", "orthogonalize", "muon"))
    case = {"op": op, "type": rng.choice(("float", "half"))}
    if op in ("layerNorm", "layerNormGrad"):
        case["dim"] = _log(rng, 16, 16384)
        case["rows"] = _log(rng, 1, min(65536, (1 << 26) // case["dim"]))
        if op == "layerNormGrad":
            case["accumulate"] = rng.choice((False, True))
    elif op == "rotary":
        case["dim"] = _log(rng, 16, 256)
        case["turned"] = rng.choice((case["dim"] // 2 * 2, case["dim"] // 4 * 2))
        case["heads"], case["behind"] = _log(rng, 1, 64), rng.choice((0, 0, 1, 8))
        case["tokens"] = _log(rng, 1, min(32768, (1 << 26) // (case["dim"] * case["heads"])))
        case["context"] = _log(rng, 1024, 1 << 20)
        case["factor"] = rng.choice((1.0, 4.0, 32.0))
        case["interleaved"], case["inverse"] = rng.choice((False, True)), rng.choice((False, True))
    elif op == "orthogonalize":
        case["rows"], case["cols"] = _log(rng, 16, 4096), _log(rng, 16, 4096)
        case["batch"] = _log(rng, 1, max(1, min(64, (1 << 22) // (case["rows"] * case["cols"]))))
    else:
        case["layers"], case["width"] = rng.randint(1, 8), _log(rng, 16, 800)
        case["master"] = case["type"] == "half" and rng.random() < 0.5
    return case


def _groups(case):
    """(rows, cols, how many) of a decoder's matrices, equal ones together: queries, keys, values and outputs; into and out of the middle layer."""
    w, n = case["width"], case["layers"]
    return [(w, w, 4 * n), (4 * w, w, n), (w, 4 * w, n)]


def _places(case):
    """(offset, stride, rows, cols, count) of each group in one allocation, and the allocation's size; a matrix begins at a multiple of 64."""
    at, places = 0, []
    for rows, cols, count in _groups(case):
        stride = -(-rows * cols // 64) * 64
        places.append((at, stride, rows, cols, count))
        at += stride * count
    return places, at


# ------------------------------------------------------------------------- operands --
class _Alias(object):
    """What torch needs to see an engine tensor's memory without a copy; keeps the tensor alive."""

    def __init__(self, t):
        self.tensor = t
        self.__cuda_array_interface__ = {
            "shape": t.shape, "strides": None, "data": (t.data_ptr(), False), "version": 2,
            "typestr": {"float": "<f4", "half": "<f2", "long": "<i8", "double": "<f8"}[t.kind]}


class _Operands(object):
    """The tensors that a program holds: torch's, or the engine's with torch's views of the same memory."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))
        self.handle, self.tensor = {}, {}

    def put(self, name, kind, values):
        """`values` as the operand `name`."""
        if own:
            import cutorch_amd as thc
            self.handle[name] = thc.Tensor(kind).resize(tuple(values.shape))
            t = torch.as_tensor(_Alias(self.handle[name]), device="cuda")
            t.copy_(values)
        else:
            t = values.to(TORCH[kind])
        self.tensor[name] = t
        return t

    def room(self, name, kind, *shape):
        """Room for the output `name`. The plain forms make theirs themselves."""
        if own:
            import cutorch_amd as thc
            self.handle[name] = thc.Tensor(kind).resize(shape)
            self.tensor[name] = torch.as_tensor(_Alias(self.handle[name]), device="cuda").zero_()

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def lists(self, case):
        """Each matrix as a tensor of its own, and the step that a program keeps."""
        if own:
            import cutorch_amd as thc
            parts = {name: [t.view_as_strided(at + i * stride, (rows, cols), (cols, 1)) for at, stride, rows, cols, count in _places(case)[0]
                            for i in range(count)] for name, t in self.handle.items()}
            self.optimizer = thc.Muon(parts["param"], parts["grad"], master=parts.get("master"), momentum=parts["momentum"], lr=LR, beta=BETA,
                                      weight_decay=DECAY, steps=NS_STEPS, eps=NS_EPS)


def _prepare_norm(o, case):
    rows, dim, kind = case["rows"], case["dim"], case["type"]
    size = torch.exp(0.5 * o.normal(dim))                              # some channels are larger than others, each has its offset
    o.put("input", kind, o.normal(rows, dim) * size + 0.3 * o.normal(dim))
    o.put("weight", kind, 1 + 0.2 * o.normal(dim))
    if case["op"] == "layerNorm":
        o.put("bias", kind, 0.1 * o.normal(dim))
        o.room("output", kind, rows, dim)
        return
    o.put("gradOutput", kind, o.normal(rows, dim))
    o.room("gradInput", kind, rows, dim)
    for name in ("gradWeight", "gradBias"):
        o.put(name, kind, math.sqrt(rows) * o.normal(dim) if case["accumulate"] else torch.zeros(dim, device="cuda"))


def _prepare_rotary(o, case):
    tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
    x = o.put("input", case["type"], o.normal(tokens, heads + case["behind"], dim))
    o.tensor["input"] = x[:, :heads]
    if own:
        h = o.handle["input"]
        o.handle["input"] = h.narrow(1, 0, heads)
    # sequences of up to 2048 tokens, each somewhere along the context
    first = torch.randint(0, case["context"], (tokens // 2048 + 1,), generator=o.g, device="cuda")
    at = torch.arange(tokens, device="cuda")
    o.put("positions", "long", (first[at // 2048] + at % 2048) % case["context"])
    o.put("frequencies", "double", _frequencies(case))
    o.scale = 1 + 0.1 * math.log(case["factor"])                       # what longer contexts take the logits down by is given back
    o.room("output", case["type"], tokens, heads, dim)


def _frequencies(case):
    """Radians per position: those that turn seldom within the first context are slowed down by the factor, in part between 1 and 32 turns."""
    half, factor = case["turned"] // 2, case["factor"]
    f = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(1, half))
    turns = f * (case["context"] / factor / (2 * math.pi))
    kept = ((turns - 1) / 31).clamp(0, 1)
    return f * (kept + (1 - kept) / factor)


def _prepare_muon(o, case):
    places, total = _places(case)
    grad, momentum = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for at, stride, rows, cols, count in places:
        # some strong directions that last from step to step, and noise
        left, right = o.normal(count, rows, 8), o.normal(count, 8, cols)
        lasting = (left * torch.logspace(0, -1.5, 8, device="cuda")) @ right * 0.02
        for flat, share in ((grad, 1.0), (momentum, 12.0)):
            m = torch.as_strided(flat, (count, rows, cols), (stride, cols, 1), at)
            m.copy_(share * lasting + share ** 0.5 * 0.01 * o.normal(count, rows, cols))
    o.put("grad", case["type"], grad / GRAD_SCALE / 16)
    o.put("momentum", "float", momentum / 16)
    p = torch.zeros(total, device="cuda")
    for at, stride, rows, cols, count in places:
        torch.as_strided(p, (count, rows, cols), (stride, cols, 1), at).copy_(0.02 * o.normal(count, rows, cols))
    o.put("param", case["type"], p)
    if case["master"]:
        o.put("master", "float", p)
    o.lists(case)


def prepare(case, seed):
    o = _Operands(seed)
    o.case = case
    if case["op"] in ("layerNorm", "layerNormGrad"):
        _prepare_norm(o, case)
    elif case["op"] == "rotary":
        _prepare_rotary(o, case)
    elif case["op"] == "muon":
        _prepare_muon(o, case)
    else:
        shape = (case["batch"], case["rows"], case["cols"])
        strong = (o.normal(shape[0], shape[1], 8) * torch.logspace(0, -1.5, 8, device="cuda")) @ o.normal(shape[0], 8, shape[2])
        o.put("input", case["type"], 0.05 * strong + 0.02 * o.normal(*shape))
        o.room("output", case["type"], *shape)
    return o


# ---------------------------------------------------------------------- plain forms --
def _standard(x):
    """Rows less their mean over their deviation, and one over that."""
    x = x.float()
    x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    return x * r, r


def _plain_norm(t):
    x = _standard(t["input"])[0]
    return (x * t["weight"].float() + t["bias"].float()).to(t["input"].dtype)


def _plain_norm_grad(case, t):
    x, r = _standard(t["input"])
    g = t["gradOutput"].float()
    gw = g * t["weight"].float()
    grad = r * (gw - gw.mean(1, keepdim=True) - x * (gw * x).mean(1, keepdim=True))
    weight, bias = (g * x).sum(0), g.sum(0)
    if case["accumulate"]:
        weight, bias = weight + t["gradWeight"].float(), bias + t["gradBias"].float()
    t["gradWeight"].copy_(weight)
    t["gradBias"].copy_(bias)
    return {"gradInput": grad.to(t["input"].dtype), "gradWeight": t["gradWeight"], "gradBias": t["gradBias"]}


def _plain_rotary(case, t, scale):
    angle = t["positions"].double()[:, None, None] * t["frequencies"]
    cos, sin = (torch.cos(angle) * scale).float(), (torch.sin(angle) * (-scale if case["inverse"] else scale)).float()
    x, n = t["input"].float(), case["turned"]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if case["interleaved"] else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., n:]), -1).to(t["input"].dtype)


def _plain_orthogonalize(x):
    """Of a batch of matrices in float."""
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = (x / (x.square().sum((1, 2), keepdim=True).sqrt() + NS_EPS)).contiguous()
    for _ in range(NS_STEPS):
        a = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = NS[0] * x + torch.bmm(NS[1] * a + NS[2] * torch.bmm(a, a), x)
    return x.transpose(1, 2) if tall else x


def _plain_muon(case, t):
    g = t["grad"].float() * GRAD_SCALE
    momentum = t["momentum"] * BETA + g
    t["momentum"].copy_(momentum)
    update = g + momentum * BETA
    p = (t["master"] if case["master"] else t["param"]).float() * (1 - LR * DECAY)
    for at, stride, rows, cols, count in _places(case)[0]:
        shape = (count, rows, cols), (stride, cols, 1), at
        torch.as_strided(p, *shape).sub_(LR * math.sqrt(max(1.0, rows / cols)) * _plain_orthogonalize(torch.as_strided(update, *shape)))
    t["param"].copy_(p)
    out = {"param": t["param"], "momentum": t["momentum"]}
    if case["master"]:
        t["master"].copy_(p)
        out["master"] = t["master"]
    return out


def _plain(o):
    case, t = o.case, o.tensor
    if case["op"] == "layerNorm":
        return _plain_norm(t)
    if case["op"] == "layerNormGrad":
        return _plain_norm_grad(case, t)
    if case["op"] == "rotary":
        return _plain_rotary(case, t, o.scale)
    if case["op"] == "orthogonalize":
        return _plain_orthogonalize(t["input"].float()).to(t["input"].dtype, memory_format=torch.contiguous_format)
    return _plain_muon(case, t)


# --------------------------------------------------------------------------- a pass --
def run(o):
    if not own:
        return _plain(o)
    case, h, t = o.case, o.handle, o.tensor
    op = case["op"]
    if op == "layerNorm":
        h["output"].layer_norm(h["input"], h["weight"], h["bias"], EPS)
        return t["output"]
    if op == "layerNormGrad":
        h["gradInput"].layer_norm_grad(h["gradWeight"], h["gradBias"], h["input"], h["gradOutput"], h["weight"], EPS, accumulate=case["accumulate"])
        return {"gradInput": t["gradInput"], "gradWeight": t["gradWeight"], "gradBias": t["gradBias"]}
    if op == "rotary":
        h["output"].rotary(h["input"], h["positions"], h["frequencies"], o.scale, interleaved=case["interleaved"], inverse=case["inverse"])
        return t["output"]
    if op == "orthogonalize":
        h["output"].orthogonalize(h["input"], NS_STEPS, NS_EPS)
        return t["output"]
    o.optimizer.step(GRAD_SCALE)
    out = {"param": t["param"], "momentum": t["momentum"]}
    if case["master"]:
        out["master"] = t["master"]
    return out


# ------------------------------------------------------------------------- measures --
def work(case):
    op, e = case["op"], SIZE[case["type"]]
    if op == "layerNorm":
        n, dim = case["rows"] * case["dim"], case["dim"]
        return {"bytes": e * (2 * n + 2 * dim), "flops": 8 * n}
    if op == "layerNormGrad":
        n, dim = case["rows"] * case["dim"], case["dim"]
        return {"bytes": e * (3 * n + dim * (5 if case["accumulate"] else 3)), "flops": 18 * n}
    if op == "rotary":
        rows = case["tokens"] * case["heads"]
        return {"bytes": 2 * e * rows * case["dim"] + 8 * case["tokens"] + 4 * case["turned"], "flops": 3 * rows * case["turned"]}
    groups = [(case["rows"], case["cols"], case["batch"])] if op == "orthogonalize" else _groups(case)
    elements = sum(r * c * n for r, c, n in groups)
    # two of a step's three products are symmetric
    flops = sum(n * NS_STEPS * min(r, c) ** 2 * (3 * max(r, c) + min(r, c)) for r, c, n in groups)
    if op == "orthogonalize":
        return {"bytes": 2 * e * elements, "flops": flops}
    return {"bytes": elements * (8 + e + (e + 8 if case["master"] else 2 * e)), "flops": flops}


# -------------------------------------------------------------------------- 64 bits --
def exact(case, seed):
    o = prepare(case, seed)
    t, op = o.tensor, case["op"]
    if op == "layerNorm":
        var, mean = torch.var_mean(t["input"].double(), 1, correction=0, keepdim=True)
        return (t["input"].double() - mean) / torch.sqrt(var + EPS) * t["weight"].double() + t["bias"].double()
    if op == "layerNormGrad":
        return _exact_norm_grad(case, t)
    if op == "rotary":
        return _exact_rotary(case, t, o.scale)
    if op == "orthogonalize":
        return torch.stack([_exact_orthogonal(x.double()) for x in t["input"]])
    out = {name: torch.zeros(t["param"].shape, dtype=torch.float64, device="cuda") for name in ("param", "momentum")}
    source = t["master" if case["master"] else "param"]
    for at, stride, rows, cols, count in _places(case)[0]:
        for i in range(count):
            s = slice(at + i * stride, at + i * stride + rows * cols)
            g = t["grad"][s].double() * GRAD_SCALE
            m = BETA * t["momentum"][s].double() + g
            out["momentum"][s] = m
            q = _exact_orthogonal((g + BETA * m).view(rows, cols)).reshape(-1)
            out["param"][s] = (1 - LR * DECAY) * source[s].double() - LR * max(1.0, rows / cols) ** 0.5 * q
    if case["master"]:
        out["master"] = out["param"]
    return out


def _exact_norm_grad(case, t):
    """By the formula of each row's Jacobian: what the mean and the deviation take from the gradient is its part along the ones and along x."""
    x, g = t["input"].double(), t["gradOutput"].double()
    dim = case["dim"]
    away = x - x.sum(1, keepdim=True) / dim
    deviation = torch.sqrt(away.pow(2).sum(1, keepdim=True) / dim + EPS)
    gw = g * t["weight"].double()
    along = (gw * away).sum(1, keepdim=True) / (dim * deviation ** 2)
    out = {"gradInput": (gw - gw.sum(1, keepdim=True) / dim - along * away) / deviation,
           "gradWeight": (g * (away / deviation)).sum(0), "gradBias": g.sum(0)}
    if case["accumulate"]:
        out["gradWeight"] = out["gradWeight"] + t["gradWeight"].double()
        out["gradBias"] = out["gradBias"] + t["gradBias"].double()
    return out


def _exact_rotary(case, t, scale):
    """As a product of complex numbers."""
    x, n = t["input"].double(), case["turned"]
    angle = torch.outer(t["positions"].double(), t["frequencies"])[:, None]
    turn = torch.polar(torch.full_like(angle, scale), -angle if case["inverse"] else angle)
    out = x.clone()
    first = slice(0, n, 2) if case["interleaved"] else slice(0, n // 2)
    second = slice(1, n, 2) if case["interleaved"] else slice(n // 2, n)
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_orthogonal(x):
    """The steps' product as a matrix on the left (or right) of the first one, from that one's square alone."""
    x = x / (torch.linalg.norm(x) + NS_EPS)
    tall = x.shape[0] > x.shape[1]
    square = x.T @ x if tall else x @ x.T
    one = torch.eye(square.shape[0], dtype=torch.float64, device=x.device)
    total = one
    for _ in range(NS_STEPS):
        a = total @ square @ total
        total = (NS[0] * one + a @ (NS[1] * one + NS[2] * a)) @ total
    return x @ total if tall else total @ x

"""The training operators of a language model, as measurable cases.

A case is a dict; "op" says which operator one pass goes through:

  embedding      rows of a table by token, times a factor
  embeddingGrad  the gradient of that table: the rows of the output's gradient, summed by token
  tokenLogProb   log-probability of each position's token under its row of logits
  policyLoss     clipped policy loss with a KL term: losses, log-probabilities and the gradient of the logits
  adamW          one AdamW step of many tensors, states in 32 bits
  adamW8         the same with states in 8 bits, and the states as the values that they stand for

Tokens are 1-based and about evenly spread over the logarithm of their number, so that the commonest one makes up
some percent of a batch, as in text.
"""
import math

import torch

own = False

TORCH = {"float": torch.float32, "half": torch.float16, "byte": torch.uint8, "char": torch.int8, "long": torch.int64}
SIZE = {"float": 4, "half": 2}
BLOCK = 256                      # elements that share a scale in 8-bit states
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.2, 0.05
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.95, 1e-8, 0.1
FIRST_STEP = 100                 # of the steps that are timed: a run that is under way
GRAD_SCALE = 1.0 / 128           # the gradients come from a loss times 128


def listed():
    return [
        # the newest tokens of 16 sequences that are being generated: launch latency
        {"name": "embedding-decode-16", "op": "embedding", "type": "half", "tokens": 16, "dim": 2048, "vocab": 32000},
        # a training batch of 8 sequences of 2049 tokens
        {"name": "embedding-batch-16k", "op": "embedding", "type": "half", "tokens": 16392, "dim": 2048, "vocab": 32000},
        # a micro-batch whose gradient is added to that of the ones before it; odd row length, rows off the 16-byte grid
        {"name": "embedding-grad-add-odd", "op": "embeddingGrad", "type": "float", "tokens": 1500, "dim": 513, "vocab": 10007,
         "padding": 0, "accumulate": True},
        # a training batch's gradient of a large table, written whole: rows without a token are zeroed
        {"name": "embedding-grad-32k", "op": "embeddingGrad", "type": "half", "tokens": 32768, "dim": 2048, "vocab": 50000,
         "padding": 1, "accumulate": False},
        # scoring the newest tokens of a few sequences: few long rows
        {"name": "logprob-decode-24", "op": "tokenLogProb", "type": "half", "rows": 24, "vocab": 128000},
        # a batch scored by the reference model
        {"name": "logprob-batch-4k", "op": "tokenLogProb", "type": "float", "rows": 4096, "vocab": 50001},
        # a small model's update: short rows in float
        {"name": "policy-small-float", "op": "policyLoss", "type": "float", "rows": 96, "vocab": 1000, "reference": True},
        # a whole batch with a large odd vocabulary: every row starts at another place of the 16-byte grid
        {"name": "policy-batch-half-odd", "op": "policyLoss", "type": "half", "rows": 4096, "vocab": 100001, "reference": True},
        # the step of a small model: some tens of tensors of a few hundred or thousand elements
        {"name": "adamw-small", "op": "adamW", "type": "float", "layers": 2, "width": 65, "vocab": 256, "master": False},
        # the step of a large one in half precision with float copies of the parameters
        {"name": "adamw-half-200m", "op": "adamW", "type": "half", "layers": 12, "width": 1024, "vocab": 50000, "master": True},
        # 8-bit states, odd sizes: every tensor ends inside a block of the scales
        {"name": "adamw8-odd", "op": "adamW8", "type": "float", "layers": 4, "width": 257, "vocab": 5003, "master": False},
        # 8-bit states of a large model
        {"name": "adamw8-180m", "op": "adamW8", "type": "float", "layers": 12, "width": 1024, "vocab": 32000, "master": False},
    ]


def _log(rng, low, high):
    """A whole number between low and high, even over its logarithm; two times in three as it falls, else a multiple of 8 or 64."""
    n = min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))
    if rng.random() < 2 / 3:
        return n
    step = 64 if n >= 256 else 8
    return min(high, max(low, n // step * step))


def draw(rng):
    op = rng.choice(("embedding", "embeddingGrad", "tokenLogProb", "policyLoss", "adamW", "adamW8"))
    kind = rng.choice(("float", "half"))
    if op in ("embedding", "embeddingGrad"):
        dim = _log(rng, 16, 8192)
        vocab = _log(rng, 100, min(262144, (1 << 28) // dim))
        case = {"op": op, "type": kind, "tokens": _log(rng, 1, min(131072, (1 << 27) // dim)), "dim": dim, "vocab": vocab}
        if op == "embeddingGrad":
            case["padding"] = rng.choice((0, 1, vocab))
            case["accumulate"] = rng.choice((False, True))
        return case
    if op in ("tokenLogProb", "policyLoss"):
        vocab = _log(rng, 64, 262144)
        case = {"op": op, "type": kind, "rows": _log(rng, 1, min(16384, (1 << 28) // vocab)), "vocab": vocab}
        if op == "policyLoss":
            case["reference"] = rng.choice((False, True))
        return case
    width = _log(rng, 16, 1024)
    return {"op": op, "type": kind, "layers": rng.randint(1, 12), "width": width, "vocab": _log(rng, 100, 32000),
            "master": kind == "half" and rng.random() < 0.5}


def _shapes(case):
    """The parameters of a decoder of this size: the table, then each layer's matrices, biases and norms."""
    w = case["width"]
    layer = [(w,), (w,), (3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
    return [(case["vocab"], w)] + layer * case["layers"] + [(w,), (w,)]


def _places(case):
    """(offset, shape) of each parameter in one allocation, and the allocation's size: each begins at a multiple of BLOCK."""
    at, places = 0, []
    for shape in _shapes(case):
        places.append((at, shape))
        at += -(-math.prod(shape) // BLOCK) * BLOCK
    return places, at


# ------------------------------------------------------------------------- operands --
class _Alias(object):
    """What torch needs to see an engine tensor's memory without a copy; keeps the tensor alive."""

    def __init__(self, t):
        self.tensor = t
        self.__cuda_array_interface__ = {
            "shape": t.shape, "strides": None, "data": (t.data_ptr(), False), "version": 2,
            "typestr": {"float": "<f4", "half": "<f2", "long": "<i8", "byte": "|u1", "char": "|i1"}[t.kind]}


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
        """Room for the output `name`, zeros at first: what lies between the tensors stays so. The plain forms make theirs themselves."""
        if own:
            import cutorch_amd as thc
            self.handle[name] = thc.Tensor(kind).resize(shape)
            self.tensor[name] = torch.as_tensor(_Alias(self.handle[name]), device="cuda").zero_()

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=dtype)

    def even(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def tokens(self, n, vocab):
        t = torch.exp(self.even(n) * math.log(vocab + 1)).floor().long()
        return t.clamp_(1, vocab)


def _prepare_logits(o, case):
    rows, vocab = case["rows"], case["vocab"]
    tokens = torch.randint(1, vocab + 1, (rows,), generator=o.g, device="cuda")
    x = o.normal(rows, vocab, dtype=TORCH[case["type"]]).mul_(2)
    at = (tokens - 1)[:, None]
    x.scatter_add_(1, at, torch.full_like(at, 7, dtype=x.dtype))      # what was sampled was likely
    x = o.put("logits", case["type"], x)
    o.put("tokens", "long", tokens)
    return x, at


def _prepare_policy(o, case):
    rows = case["rows"]
    x, at = _prepare_logits(o, case)
    now = torch.empty(rows, device="cuda")
    for i in range(0, rows, 512):
        part = x[i:i + 512].double()
        now[i:i + 512] = (part.gather(1, at[i:i + 512])[:, 0] - part.logsumexp(1)).float()
    # the policy has moved by about a fifth since the tokens were sampled, in steps that keep clear of the clip's edges
    o.put("old", "float", now + torch.round(o.normal(rows) * 10) * 0.02 + 0.005)
    o.put("advantage", "float", o.normal(rows))
    if case["reference"]:
        o.put("reference", "float", now + 0.3 * o.normal(rows))
    kept = (o.even(rows) >= 0.1).float()                               # a tenth is padding
    kept[0] = 1
    o.put("weight", "float", kept / kept.sum().clamp_min(1))
    o.room("loss", "float", rows)
    o.room("logProb", "float", rows)
    o.room("gradLogits", case["type"], rows, case["vocab"])


def _prepare_adamw(o, case):
    places, total = _places(case)
    inside = torch.zeros(total, device="cuda")                         # 0 between the tensors
    size = torch.zeros(total, device="cuda")                           # gradients differ between tensors
    for k, (at, shape) in enumerate(places):
        n = math.prod(shape)
        inside[at:at + n] = 1
        size[at:at + n] = 0.002 * (1 + k % 7)
    size *= inside
    p = 0.02 * o.normal(total) * inside
    o.put("param", case["type"], p)
    if case["master"]:
        o.put("master", "float", p)
    o.put("grad", case["type"], o.normal(total) * size / GRAD_SCALE)
    mean, square = 0.3 * o.normal(total) * size, (0.25 + 1.5 * o.even(total)) * size * size
    if case["op"] == "adamW":
        o.put("mean", "float", mean)
        o.put("square", "float", square)
    else:
        for name, kind, (codes, scales) in (("mean", "char", _encode_mean(mean)), ("square", "byte", _encode_square(square))):
            o.put(name, kind, codes)
            o.put(name + "Scale", "float", scales)
            o.room(name + "Value", "float", total)
    if own:
        import cutorch_amd as thc
        parts = {}
        for name, t in o.handle.items():
            if name.endswith("Scale"):
                parts[name] = [t.narrow(0, at // BLOCK, -(-math.prod(shape) // BLOCK)) for at, shape in places]
            else:
                parts[name] = [t.view_as_strided(at, shape, [math.prod(shape[d + 1:]) for d in range(len(shape))]) for at, shape in places]
        scales = {"mean_scale": parts["meanScale"], "square_scale": parts["squareScale"]} if case["op"] == "adamW8" else {}
        o.optimizer = thc.AdamW(parts["param"], parts["grad"], master=parts.get("master"), lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS,
                                weight_decay=DECAY, mean=parts["mean"], square=parts["square"], step=FIRST_STEP, **scales)
        o.values = (parts.get("meanValue"), parts.get("squareValue"))


def prepare(case, seed):
    o = _Operands(seed)
    o.case, o.step = case, FIRST_STEP
    op, kind = case["op"], case["type"]
    if op in ("embedding", "embeddingGrad"):
        n, dim, vocab = case["tokens"], case["dim"], case["vocab"]
        o.put("tokens", "long", o.tokens(n, vocab))
        if op == "embedding":
            o.put("weight", kind, 0.02 * o.normal(vocab, dim))
            o.room("output", kind, n, dim)
        else:
            o.put("gradOutput", kind, o.normal(n, dim))
            o.put("gradWeight", kind, o.normal(vocab, dim) if case["accumulate"] else torch.zeros(vocab, dim, device="cuda"))
    elif op == "tokenLogProb":
        _prepare_logits(o, case)
        o.room("logProb", "float", case["rows"])
    elif op == "policyLoss":
        _prepare_policy(o, case)
    else:
        _prepare_adamw(o, case)
    return o


# ---------------------------------------------------------------------- plain forms --
def _factor(case):
    return math.sqrt(case["dim"])


def _plain_embedding(case, weight, tokens):
    return (weight[tokens - 1].float() * _factor(case)).to(weight.dtype)


def _plain_embedding_grad(case, grad, tokens, grad_out):
    total = torch.zeros(grad.shape, device=grad.device)
    rows = torch.where((tokens == case["padding"])[:, None], 0.0, grad_out.float())
    total.index_add_(0, tokens - 1, rows)
    total = total * _factor(case)
    grad.copy_(grad.float() + total if case["accumulate"] else total)
    return grad


def _log_softmax_parts(logits, tokens):
    x = logits.float()
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    return e, total, (x.gather(1, (tokens - 1)[:, None]) - torch.log(total))[:, 0]


def _plain_policy(case, t):
    e, total, now = _log_softmax_parts(t["logits"], t["tokens"])
    kept = t["weight"] != 0
    ratio = torch.exp(now - t["old"])
    gain, held = ratio * t["advantage"], ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * t["advantage"]
    loss = -torch.minimum(gain, held)
    slope = torch.where(gain <= held, -gain, 0.0)
    if case["reference"]:
        away = t["reference"] - now
        loss = loss + KL * (torch.exp(away) - away - 1)
        slope = slope + KL * (1 - torch.exp(away))
    loss = torch.where(kept, t["weight"] * loss, 0.0)
    slope = torch.where(kept, t["weight"] * slope, 0.0) * case["rows"]          # the loss is scaled by the number of rows
    grad = e * (-slope[:, None] / total)
    at = (t["tokens"] - 1)[:, None]
    grad.scatter_(1, at, grad.gather(1, at) + slope[:, None])
    grad = torch.where(kept[:, None], grad, 0.0)
    return {"loss": loss, "logProb": torch.where(kept, now, 0.0), "gradLogits": grad.to(t["logits"].dtype)}


def _encode_mean(mean):
    """Sign and 7 bits of each value's square root over its block's largest; the largest magnitude of each block."""
    top = mean.abs().view(-1, BLOCK).amax(1)
    share = (mean.abs().view(-1, BLOCK) * _inverse(top)[:, None]).view(-1)
    return (torch.sign(mean) * torch.round(torch.sqrt(share) * 127)).to(torch.int8), top


def _encode_square(square):
    """8 bits of each value's fourth root over its block's largest, at least 1 where the value is not zero; each block's largest."""
    top = square.view(-1, BLOCK).amax(1)
    share = (square.view(-1, BLOCK) * _inverse(top)[:, None]).view(-1)
    code = torch.round(torch.sqrt(torch.sqrt(share)) * 255)
    return torch.where(share > 0, code.clamp_min(1), code).to(torch.uint8), top


def _inverse(top):
    return torch.where(top > 0, torch.reciprocal(top), torch.zeros_like(top))


def _decode_mean(codes, top, dtype=torch.float32):
    t = codes.to(dtype) * (1 / 127)
    return ((t * t.abs()).view(-1, BLOCK) * top.to(dtype)[:, None]).view(-1)


def _decode_square(codes, top, dtype=torch.float32):
    t = codes.to(dtype) * (1 / 255)
    t = t * t
    return ((t * t).view(-1, BLOCK) * top.to(dtype)[:, None]).view(-1)


def _adamw(p, g, mean, square, step):
    """The step's formulas in the type of its operands, one elementary operation at a time."""
    g = g * GRAD_SCALE
    mean = mean * BETA1 + g * (1 - BETA1)
    square = square * BETA2 + (g * g) * (1 - BETA2)
    root = torch.sqrt(square) * (1 / math.sqrt(1 - BETA2 ** step)) + EPS
    return p * (1 - LR * DECAY) - (mean / root) * (LR / (1 - BETA1 ** step)), mean, square


def _plain_adamw(case, t, step):
    source = t["master"] if case["master"] else t["param"]
    eight = case["op"] == "adamW8"
    mean = _decode_mean(t["mean"], t["meanScale"]) if eight else t["mean"]
    square = _decode_square(t["square"], t["squareScale"]) if eight else t["square"]
    p, mean, square = _adamw(source.float(), t["grad"].float(), mean, square, step)
    t["param"].copy_(p)
    out = {"param": t["param"]}
    if case["master"]:
        t["master"].copy_(p)
        out["master"] = t["master"]
    if not eight:
        t["mean"].copy_(mean)
        t["square"].copy_(square)
        return {**out, "mean": t["mean"], "square": t["square"]}
    codes, top = _encode_mean(mean)
    t["mean"].copy_(codes)
    t["meanScale"].copy_(top)
    codes, top = _encode_square(square)
    t["square"].copy_(codes)
    t["squareScale"].copy_(top)
    return {**out, "mean": _decode_mean(t["mean"], t["meanScale"]), "square": _decode_square(t["square"], t["squareScale"])}


def _plain(o):
    case, t = o.case, o.tensor
    if case["op"] == "embedding":
        return _plain_embedding(case, t["weight"], t["tokens"])
    if case["op"] == "embeddingGrad":
        return _plain_embedding_grad(case, t["gradWeight"], t["tokens"], t["gradOutput"])
    if case["op"] == "tokenLogProb":
        return _log_softmax_parts(t["logits"], t["tokens"])[2]
    if case["op"] == "policyLoss":
        return _plain_policy(case, t)
    o.step += 1
    return _plain_adamw(case, t, o.step)


# --------------------------------------------------------------------------- a pass --
def run(o):
    if not own:
        return _plain(o)
    case, h, t = o.case, o.handle, o.tensor
    op = case["op"]
    if op == "embedding":
        h["output"].embedding(h["weight"], h["tokens"], _factor(case))
        return t["output"]
    if op == "embeddingGrad":
        h["gradWeight"].embedding_grad(h["tokens"], h["gradOutput"], _factor(case), padding=case["padding"], accumulate=case["accumulate"])
        return t["gradWeight"]
    if op == "tokenLogProb":
        h["logProb"].token_log_prob(h["logits"], h["tokens"])
        return t["logProb"]
    if op == "policyLoss":
        h["loss"].policy_loss(h["logProb"], h["gradLogits"], h["logits"], h["tokens"], h["old"], h["advantage"],
                              reference=h.get("reference"), weight=h["weight"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                              kl=KL, grad_scale=case["rows"])
        return {"loss": t["loss"], "logProb": t["logProb"], "gradLogits": t["gradLogits"]}
    o.optimizer.step(GRAD_SCALE)
    out = {"param": t["param"]}
    if case["master"]:
        out["master"] = t["master"]
    if op == "adamW":
        return {**out, "mean": t["mean"], "square": t["square"]}
    o.optimizer.moments(*o.values)
    return {**out, "mean": t["meanValue"], "square": t["squareValue"]}


# ------------------------------------------------------------------------- measures --
def work(case):
    op, e = case["op"], SIZE[case["type"]]
    if op == "embedding":
        n, dim = case["tokens"], case["dim"]
        return {"bytes": 8 * n + e * dim * (_distinct(n, case["vocab"]) + n), "flops": n * dim}
    if op == "embeddingGrad":
        n, dim, vocab = case["tokens"], case["dim"], case["vocab"]
        written = 2 * _distinct(n, vocab) if case["accumulate"] else vocab
        return {"bytes": 8 * n + e * dim * (n + written), "flops": n * dim}
    if op == "tokenLogProb":
        return {"bytes": case["rows"] * (case["vocab"] * e + 12), "flops": 4 * case["rows"] * case["vocab"]}
    if op == "policyLoss":       # nine rows of ten are read, all are written
        rows = case["rows"]
        return {"bytes": rows * (1.9 * case["vocab"] * e + 28 + 4 * case["reference"]), "flops": 7 * rows * case["vocab"]}
    n = sum(math.prod(s) for s in _shapes(case))
    params = e + (e + 8 if case["master"] else 2 * e)
    states = 16 if op == "adamW" else 2 * 2 * (1 + 4 / BLOCK) + 8
    return {"bytes": n * (params + states), "flops": (14 if op == "adamW" else 30) * n}


def _distinct(n, vocab):
    """How many different ones n tokens hold, by their distribution."""
    full = math.log(vocab + 1)
    edges = sorted({int(round(math.exp(full * i / 400))) for i in range(401)} | {1, vocab + 1})
    return sum((b - a) * -math.expm1(n * math.log1p(-min(1 - 1e-12, math.log(b / a) / full / (b - a)))) for a, b in zip(edges, edges[1:]))


# -------------------------------------------------------------------------- 64 bits --
def exact(case, seed):
    o = prepare(case, seed)
    t, op = o.tensor, case["op"]
    if op == "embedding":
        return torch.index_select(t["weight"], 0, t["tokens"] - 1).double() * _factor(case)
    if op == "embeddingGrad":
        used = t["tokens"] != case["padding"]
        rows, group = torch.unique(t["tokens"][used] - 1, return_inverse=True)
        sums = torch.zeros(len(rows), case["dim"], dtype=torch.float64, device="cuda").index_add_(0, group, t["gradOutput"][used].double())
        total = t["gradWeight"].double() if case["accumulate"] else torch.zeros(t["gradWeight"].shape, dtype=torch.float64, device="cuda")
        total[rows] += sums * _factor(case)
        return total
    if op == "tokenLogProb":
        return torch.cat([torch.log_softmax(x.double(), 1).gather(1, (a - 1)[:, None])[:, 0]
                          for x, a in zip(t["logits"].split(1024), t["tokens"].split(1024))])
    if op == "policyLoss":
        return _exact_policy(case, t)
    eight = op == "adamW8"
    mean = _decode_mean(t["mean"], t["meanScale"], torch.float64) if eight else t["mean"].double()
    square = _decode_square(t["square"], t["squareScale"], torch.float64) if eight else t["square"].double()
    g, step = t["grad"].double() * GRAD_SCALE, FIRST_STEP + 1
    mean = BETA1 * mean + (1 - BETA1) * g
    square = BETA2 * square + (1 - BETA2) * g ** 2
    corrected = (mean / (1 - BETA1 ** step)) / ((square / (1 - BETA2 ** step)).sqrt() + EPS)
    source = t["master" if case["master"] else "param"].double()
    p = source - LR * (DECAY * source + corrected)
    out = {"param": p, "mean": mean, "square": square}
    if case["master"]:
        out["master"] = p
    if eight:
        out["mean"], out["square"] = _held(mean, 127, 2), _held(square, 255, 4)
    return out


def _held(x, top_code, power):
    """x as 8 bits hold it: blocks of codes whose `power` is the share of the block's largest magnitude."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    share = torch.where(top > 0, x.abs() / top, 0.0)
    code = torch.round(share ** (1 / power) * top_code)
    if power == 4:
        code = torch.where(share > 0, code.clamp_min(1), code)
    return (torch.sign(x) * top * (code / top_code) ** power).view(-1)


def _exact_policy(case, t):
    at = (t["tokens"] - 1)[:, None]
    used, weight, advantage = t["weight"] != 0, t["weight"].double(), t["advantage"].double()
    loss, logp, grad = [], [], []
    for i in range(0, case["rows"], 512):
        s = slice(i, i + 512)
        probability = torch.softmax(t["logits"][s].double(), 1)
        now = torch.log(probability.gather(1, at[s])[:, 0])
        r = torch.exp(now - t["old"][s].double())
        free, clipped = r * advantage[s], torch.clamp(r, 1 - CLIP_LOW, 1 + CLIP_HIGH) * advantage[s]
        value, slope = torch.maximum(-free, -clipped), -free * (free <= clipped)
        if case["reference"]:
            q = torch.exp(t["reference"][s].double() - now)
            value, slope = value + KL * (q - torch.log(q) - 1), slope + KL * (1 - q)
        chosen = torch.zeros_like(probability).scatter_(1, at[s], 1.0)
        w = weight[s]
        loss.append(value * w)
        logp.append(now * used[s])
        grad.append((chosen - probability) * (slope * w * case["rows"])[:, None])
    return {"loss": torch.cat(loss), "logProb": torch.cat(logp), "gradLogits": torch.cat(grad)}

"""A decoder layer's projections in 8 bits, and the sampled token: what is measured, in plain form and through the library.

Between the residual stream and the answer a serving loop uses four operators: the residual's addition with the
root-mean-square norm, whose result leaves in 8 bits with a scale for each 128 columns; the product of such rows with
weights that have a scale for each block of 128 x 128; the other rows that enter a product (the gated activation, the
attention's output), brought to the same form; and the choice of a token from its logits with temperature, top-k, top-p
and min-p from given random numbers.

``own = False`` runs each operator as elementary torch operations in 32 bits (in 64 where a choice hangs on a border),
``own = True`` as a program that uses the library calls it. ``exact`` computes the same outputs in 64 bits from the
definitions.

Layouts: rows [rows, width]; their scales [blocks of 128 columns, rows]; weights [n, k] with scales [blocks of n,
blocks of k]; logits [rows, vocabulary], each row's settings in tensors of one entry a row.
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
BLOCK = 128
LARGEST = 448.0  # of e4m3
TINY = 2.0 ** -126
EPSILON = 1e-6


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # decode of one sequence: q, k and v of one token (hidden 4096, 32 + 2 x 8 heads of 128)
        {"name": "product one token", "op": "product", "type": "bf16", "m": 1, "n": 6144, "k": 4096},
        # decode of sixteen sequences: gate and up (2 x 12288)
        {"name": "product batch", "op": "product", "type": "bf16", "m": 16, "n": 24576, "k": 4096},
        # one prompt of an odd length: down
        {"name": "product ragged prompt", "op": "product", "type": "fp16", "m": 777, "n": 4096, "k": 12288},
        # packed prompts: gate and up
        {"name": "product prompts", "op": "product", "type": "bf16", "m": 8192, "n": 24576, "k": 4096},
        # decode of one sequence
        {"name": "norm one token", "op": "norm", "type": "bf16", "rows": 1, "width": 4096},
        # packed prompts
        {"name": "norm prompts", "op": "norm", "type": "bf16", "rows": 8192, "width": 4096},
        # decode of sixteen sequences: the gated activation before down
        {"name": "activation batch", "op": "activation", "type": "bf16", "rows": 16, "width": 12288, "gated": True},
        # packed prompts: the gated activation
        {"name": "activation prompts", "op": "activation", "type": "fp16", "rows": 8192, "width": 12288, "gated": True},
        # one prompt of an odd length: the attention's output before its projection
        {"name": "attention output", "op": "activation", "type": "bf16", "rows": 2047, "width": 4096, "gated": False},
        # one chat: the next token
        {"name": "sample one", "op": "sample", "type": "bf16", "rows": 1, "vocabulary": 151936, "mix": 1},
        # sixteen users, each with settings of their own
        {"name": "sample batch", "op": "sample", "type": "bf16", "rows": 16, "vocabulary": 151936, "mix": 2},
        # every node of sixteen drafted trees
        {"name": "sample trees", "op": "sample", "type": "fp16", "rows": 1024, "vocabulary": 151936, "mix": 3},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["product", "product", "product", "norm", "activation", "sample", "sample"])
    case = {"op": op, "type": rng.choice(["bf16", "fp16"])}
    if op == "product":
        n, k = rng.choice([(6144, 4096), (4096, 4096), (24576, 4096), (4096, 12288), (4096, 1024), (1024, 2048), (151936, 1024),
                           (_log(rng, 16, 16384), 16 * _log(rng, 4, 768)), (_log(rng, 16, 16384), 16 * _log(rng, 4, 768)),
                           (_log(rng, 16, 16384), 16 * _log(rng, 4, 768))])
        return case | {"m": _log(rng, 1, min(8192, 8192 * 24576 * 4096 // (n * k))), "n": n, "k": k}
    if op == "sample":
        vocabulary = rng.choice([151936, 4096, _log(rng, 17, 262144)])
        return case | {"rows": _log(rng, 1, min(1024, 1024 * 151936 // vocabulary)), "vocabulary": vocabulary,
                       "mix": rng.randrange(1 << 30)}
    most, gated = (8192 * 12288, rng.random() < 0.6) if op == "activation" else (8192 * 4096, None)
    width = rng.choice([4096, 12288, 1024, 16 * _log(rng, 4, 1024)])
    case |= {"rows": _log(rng, 1, min(8192, most // width)), "width": width}
    return case if gated is None else case | {"gated": gated}


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * _blocks(k) * (m + _blocks(n)) + 2 * m * n, "flops": 2 * m * n * k}
    rows = case["rows"]
    if case["op"] == "sample":
        return {"bytes": rows * (2 * case["vocabulary"] + 28), "flops": rows * case["vocabulary"]}
    width = case["width"]
    quantised = rows * (width + 4 * _blocks(width))
    if case["op"] == "norm":
        return {"bytes": rows * width * 6 + 2 * width + quantised, "flops": 8 * rows * width}
    return {"bytes": rows * width * (4 if case["gated"] else 2) + quantised, "flops": rows * width * (8 if case["gated"] else 3)}


# ----------------------------------------------------------------- inputs ----

def _settings(case):
    """Each row's temperature, top-k, top-p and min-p, as users mix them: part of the case, not of the seed."""
    r = random.Random(case["mix"])
    if case["rows"] == 1:  # an ordinary chat's
        return [(r.choice([0.6, 0.7, 1.0]), r.choice([20, 50]), r.choice([0.8, 0.95]), 0.0)]
    return [(r.choice([0.0, 0.6, 0.7, 1.0, 1.0, 1.5]), r.choice([0, 0, 1, 20, 50, 1000]), r.choice([1.0, 1.0, 0.95, 0.8, 0.5]),
             r.choice([0.0, 0.0, 0.05, 0.2])) for _ in range(case["rows"])]


def _logits(g, case):
    """A broad mass of tokens, a few likely ones a row, and in some rows a grammar's mask."""
    rows, vocabulary = case["rows"], case["vocabulary"]
    logits = torch.empty(rows, vocabulary, dtype=TYPES[case["type"]], device="cuda")
    for part in logits.split(128):
        x = torch.randn(part.shape, device="cuda", generator=g) * 2.0
        likely = torch.rand(part.shape, device="cuda", generator=g) < 40 / vocabulary
        part.copy_(x + 12.0 * torch.rand(part.shape, device="cuda", generator=g) * likely)
    for row in range(0, rows, 7):  # a mask that leaves about a tenth
        if row % 2:
            logits[row, torch.rand(vocabulary, device="cuda", generator=g) > 0.1] = -math.inf
            logits[row, vocabulary // 2] = 1.0
    return logits


def _weights(g, n, k):
    """Normal weights, each block of 128 x 128 scaled to its largest value."""
    w = torch.empty(n, k, dtype=E4M3, device="cuda")
    scales = torch.empty(_blocks(n), _blocks(k), device="cuda")
    for begin in range(0, n, 8192):
        rows = min(8192, n - begin)
        x = torch.zeros(BLOCK * _blocks(rows), BLOCK * _blocks(k), device="cuda")
        x[:rows, :k] = torch.randn(rows, k, device="cuda", generator=g) * 0.02
        x = x.view(_blocks(rows), BLOCK, _blocks(k), BLOCK)
        s = x.abs().amax((1, 3)) / LARGEST
        scales[begin // BLOCK:begin // BLOCK + len(s)] = s
        w[begin:begin + rows] = (x / s[:, None, :, None]).view(-1, BLOCK * _blocks(k))[:rows, :k].to(E4M3)
    return w, scales


def _stream(g, rows, width, dtype):
    """Activations as a layer has them: some columns far larger than the others."""
    x = torch.randn(rows, width, device="cuda", generator=g)
    x[:, ::97] *= 20.0
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, s = TYPES[case["type"]], {"case": case, "op": case["op"]}
    empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    if case["op"] == "product":
        a, a_scales = _quantise(_stream(g, case["m"], case["k"], torch.float32))
        w, w_scales = _weights(g, case["n"], case["k"])
        return s | {"a": a, "a_scales": a_scales, "w": w, "w_scales": w_scales, "out": empty(case["m"], case["n"], dtype=dtype)}
    rows = case["rows"]
    if case["op"] == "sample":
        settings = [torch.tensor(x, device="cuda") for x in zip(*_settings(case))]
        names = ("temperature", "top_k", "top_p", "min_p")
        s |= dict(zip(names, (x.int() if name == "top_k" else x.float() for name, x in zip(names, settings))))
        return s | {"logits": _logits(g, case), "u": torch.rand(rows, device="cuda", generator=g),
                    "tokens": empty(rows, dtype=torch.int32), "logprobs": empty(rows)}
    width = case["width"]
    s |= {"q": empty(rows, width, dtype=E4M3), "scales": empty(_blocks(width), rows)}
    if case["op"] == "norm":
        return s | {"x": _stream(g, rows, width, dtype), "residual": _stream(g, rows, width, dtype) * 4, "total": empty(rows, width, dtype=dtype),
                    "weight": (1.0 + 0.2 * torch.randn(width, device="cuda", generator=g)).to(dtype)}
    return s | {"x": _stream(g, rows, width * (2 if case["gated"] else 1), dtype)}


# ------------------------------------------------------------- plain forms ----

def _grouped(y):
    """[rows, blocks, 128] of rows whose last block may be short, with zeros behind it."""
    rows, width = y.shape
    if width % BLOCK:
        y = torch.cat([y, torch.zeros(rows, BLOCK - width % BLOCK, dtype=y.dtype, device=y.device)], 1)
    return y.view(rows, -1, BLOCK)


def _quantise(y):
    """Rows in 8 bits and their scales: the largest value of each 128 columns becomes 448."""
    rows, width = y.shape
    y = _grouped(y)
    scales = (y.abs().amax(-1) / LARGEST).clamp_(min=TINY)
    q = (y / scales[..., None]).clamp_(-LARGEST, LARGEST).to(E4M3).view(rows, -1)[:, :width]
    return q.contiguous(), scales.t().contiguous()


def _product(s):
    k, n = s["case"]["k"], s["case"]["n"]
    a = (_grouped(s["a"].float()) * s["a_scales"].t()[..., None]).view(len(s["a"]), -1)[:, :k]
    w = s["w"].float()
    w *= s["w_scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return (a @ w.t()).to(s["out"].dtype)


def _norm(s):
    total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    t = total.float()
    y = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPSILON) * s["weight"].float()
    return total, *_quantise(y)


def _activation(s):
    if not s["case"]["gated"]:
        return _quantise(s["x"].float())
    gate, up = s["x"].float().chunk(2, 1)
    return _quantise(gate / (1.0 + torch.exp(-gate)) * up)


def _sample(s):
    """Tokens in the order of their logits, of equal ones the lowest id first. In 64 bits: a token hangs on where u falls
    between the sums of up to all of them."""
    logits, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    greedy = (s["temperature"] == 0)[:, None]
    x = (logits.double() - logits[:, :1].double()) / torch.where(greedy, 1.0, s["temperature"][:, None]).double()
    rank = torch.arange(x.shape[1], device="cuda")
    limit = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1])[:, None]
    limit = torch.where(greedy, 1, limit)
    weight = torch.where(rank < limit, x.exp(), 0.0)
    sums = weight.cumsum(1)
    before = torch.cat([torch.zeros_like(sums[:, :1]), sums[:, :-1]], 1)
    keep = (before < s["top_p"][:, None].double() * sums[:, -1:]) & (weight >= s["min_p"][:, None].double()) & (weight > 0)
    keep[:, 0] = True
    kept = keep.sum(1, keepdim=True)
    total = sums.gather(1, kept - 1)
    at = torch.minimum(((sums <= s["u"][:, None].double() * total) & keep).sum(1, keepdim=True), kept - 1)
    return order.gather(1, at)[:, 0].int(), (x.gather(1, at) - total.log())[:, 0].float()


def run(s):
    """One pass."""
    if not own:
        return {"product": _product, "norm": _norm, "activation": _activation, "sample": _sample}[s["op"]](s)
    from xpu_playground_b200 import kernels
    if s["op"] == "product":
        return kernels.fp8_gemm(s["a"], s["a_scales"], s["w"], s["w_scales"], out=s["out"])
    if s["op"] == "norm":
        return kernels.fp8_rms_norm(s["x"], s["weight"], s["residual"], EPSILON, total=s["total"], q=s["q"], scales=s["scales"])
    if s["op"] == "activation":
        call = kernels.fp8_silu_multiply if s["case"]["gated"] else kernels.fp8_quantize
        return call(s["x"], q=s["q"], scales=s["scales"])
    return kernels.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], tokens=s["tokens"],
                          logprobs=s["logprobs"])


# ---------------------------------------------------------------- in 64 bits ----

def _eight_bits64(y):
    """What the 8 bits stand for before they are rounded, and the scales, block by block."""
    q, scales = torch.empty_like(y), []
    for begin in range(0, y.shape[1], BLOCK):
        part = y[:, begin:begin + BLOCK]
        top = part.abs().max(1).values / LARGEST
        scales.append(torch.where(top < TINY, torch.full_like(top, TINY), top))
        q[:, begin:begin + BLOCK] = part / scales[-1][:, None]
    return q, torch.stack(scales)


def _choice64(logits, temperature, top_k, top_p, min_p, u):
    """One row: token and logarithm of its probability."""
    order = np.argsort(-logits, kind="stable")
    if temperature == 0:
        return int(order[0]), 0.0
    z = (logits[order] - logits[order[0]]) / temperature
    if top_k > 0:
        z = z[:top_k]
    p = np.exp(z)
    mass = np.cumsum(p)
    many = int(np.searchsorted(mass, top_p * mass[-1], side="left")) + 1  # the shortest beginning that has top_p
    many = max(1, min(many, int((p >= min_p).sum()), int((p > 0).sum())))
    at = min(int(np.searchsorted(mass[:many], u * mass[many - 1], side="right")), many - 1)
    return int(order[at]), float(z[at] - np.log(mass[many - 1]))


def exact(case, seed):
    if case["op"] == "sample" and case["rows"] * case["vocabulary"] > 20_000_000:
        return None  # sorting so many rows one by one takes too long
    s = prepare(case, seed)
    if case["op"] == "product":
        out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for g, begin in enumerate(range(0, case["k"], BLOCK)):
            sums = s["a"][:, begin:begin + BLOCK].double() @ s["w"][:, begin:begin + BLOCK].double().t()
            columns = s["w_scales"][:, g].double()[torch.arange(case["n"], device="cuda") // BLOCK]
            out += sums * s["a_scales"][g].double()[:, None] * columns
        return out
    if case["op"] == "norm":
        total = s["x"].double() + s["residual"].double()
        t = total.to(s["x"].dtype).double()  # the stream is held in its type
        y = t / ((t * t).sum(1, keepdim=True) / case["width"] + EPSILON).sqrt() * s["weight"].double()
        return total, *_eight_bits64(y)
    if case["op"] == "activation":
        if not case["gated"]:
            return _eight_bits64(s["x"].double())
        width = case["width"]
        return _eight_bits64(s["x"][:, :width].double() * torch.sigmoid(s["x"][:, :width].double()) * s["x"][:, width:].double())
    logits = s["logits"].double().cpu().numpy()
    rows = [_choice64(logits[i], *(float(s[x][i]) if x != "top_k" else int(s[x][i])
                                   for x in ("temperature", "top_k", "top_p", "min_p", "u"))) for i in range(case["rows"])]
    return (torch.tensor([t for t, _ in rows], dtype=torch.int32, device="cuda"),
            torch.tensor([p for _, p in rows], dtype=torch.float64, device="cuda"))

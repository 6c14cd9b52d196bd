"""Measured operators of the quantised model beside the prover: the activations of a row in 8 bits, the 8-bit product
(scaled, as whole sums, or as field elements for the witness), and what a row of logits says about the token that was given.

`listed()` gives the fixed cases, `draw(rng)` more of the same ranges, `prepare(case, seed)` a case's inputs on the GPU,
`run(state)` one pass, `work(case)` the bytes and operations that a pass cannot do without, `exact(case, seed)` the outputs
from the definitions in 64 bits.  With `own` false a pass runs in elementary torch operations, with `own` true through the
package's entry points.

A case is a dict with a "kind":

  quantize   rows of activations (or of a weight, one row a channel) to int8 with one scale a row
  product    int8 x int8 with a scale a token and a scale a channel; "layout" says how the (k, n) weight lies in memory:
             "kn" row-major, "nk" the transposed view of a weight stored by output channel
  witness    the same product as whole numbers: int32 sums, or field elements as a commitment takes them
  logprobs   log probability of each row's token, the row's entropy, its "top" likeliest tokens
"""
import math

import torch

own = False
DEV = "cuda"
P = (1 << 64) - (1 << 32) + 1                     # the field of the witness
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int32": torch.int32, "field": torch.uint64}


def listed():
    return [
        # the activation of one token before a projection: a launch and its latency
        dict(name="quantize 1x4096 bf16", kind="quantize", m=1, k=4096, dtype="bf16", pitch=4096),
        # the activations of a 1000-token prompt before the down projection
        dict(name="quantize 1000x11008 bf16", kind="quantize", m=1000, k=11008, dtype="bf16", pitch=11008),
        # an MLP weight by output channel, from 32-bit values
        dict(name="quantize 11008x4096 fp32", kind="quantize", m=11008, k=4096, dtype="fp32", pitch=4096),
        # one token through the up projection, weight stored by output channel
        dict(name="product 1x4096x11008", kind="product", m=1, k=4096, n=11008, layout="nk", dtype="bf16"),
        # sixteen sequences answering together through the down projection, weight as the prover holds it
        dict(name="product 16x11008x4096", kind="product", m=16, k=11008, n=4096, layout="kn", dtype="fp16"),
        # sizes that no tile divides, rows that start on odd bytes
        dict(name="product 333x1001x515", kind="product", m=333, k=1001, n=515, layout="kn", dtype="fp32"),
        # a 1000-token prompt through the up projection
        dict(name="product 1000x4096x11008", kind="product", m=1000, k=4096, n=11008, layout="nk", dtype="bf16"),
        # four thousand tokens through an expert's 5120 x 8192 weight
        dict(name="product 4096x5120x8192", kind="product", m=4096, k=5120, n=8192, layout="nk", dtype="bf16"),
        # the witness of the up projection, committed as field elements
        dict(name="witness 1000x4096x11008", kind="witness", m=1000, k=4096, n=11008, layout="kn", dtype="field"),
        # one answered token, twenty alternatives
        dict(name="logprobs 1x32000 fp32", kind="logprobs", rows=1, vocab=32000, dtype="fp32", top=20, temperature=1.0, masked="no", pitch=32000),
        # a batch of answers over a large vocabulary of odd size in padded rows, part of it not allowed
        dict(name="logprobs 64x202045 fp16", kind="logprobs", rows=64, vocab=202045, dtype="fp16", top=20, temperature=0.7, masked="inf", pitch=202048),
        # the answers of a whole batch under review
        dict(name="logprobs 4096x32000 bf16", kind="logprobs", rows=4096, vocab=32000, dtype="bf16", top=5, temperature=1.0, masked="no", pitch=32000),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm; two thirds of them are left as they fall, the others are
    taken down to a multiple of 16."""
    v = min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    return max(lo, v // 16 * 16) if rng.random() < 0.35 else v


def draw(rng):
    kind = rng.choice(("quantize", "product", "product", "product", "witness", "logprobs", "logprobs"))
    if kind == "quantize":
        m, k = _spread(rng, 1, 11008), _spread(rng, 64, 16384)
        m = min(m, 45_000_000 // k)
        return dict(kind=kind, m=m, k=k, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), pitch=k + rng.choice((0, 0, 8, 5)))
    if kind == "logprobs":
        vocab = _spread(rng, 500, 262144)
        rows = _spread(rng, 1, 4096)
        rows = max(1, min(rows, 131_000_000 // vocab // 2))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=rng.choice(("bf16", "fp16", "fp32")), top=rng.choice((0, 1, 5, 8, 20)),
                    temperature=rng.choice((1.0, 1.0, 0.7, 1.5)), masked=rng.choice(("no", "no", "inf", "lowest")),
                    pitch=vocab + rng.choice((0, 0, 16, 3)))
    m, k, n = _spread(rng, 1, 4096), _spread(rng, 32, 11008), _spread(rng, 16, 11008)
    m = max(1, min(m, 170_000_000_000 // (k * n)))
    dtype = rng.choice(("bf16", "fp16", "fp32")) if kind == "product" else rng.choice(("field", "field", "int32"))
    return dict(kind=kind, m=m, k=k, n=n, layout=rng.choice(("nk", "kn")), dtype=dtype)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _pitched(t, pitch):
    """`t` as the leading columns of a buffer with `pitch` columns."""
    if pitch == t.size(1):
        return t
    buf = torch.zeros(t.size(0), pitch, dtype=t.dtype, device=t.device)
    buf[:, : t.size(1)] = t
    return buf[:, : t.size(1)]


def _int8(gen, *shape):
    """Quantised values: a bell that uses most of the range, its tails cut at +-127."""
    return (torch.randn(shape, generator=gen, device=DEV) * 36).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    kind = case["kind"]
    if kind == "quantize":
        x = torch.randn(case["m"], case["k"], generator=gen, device=DEV)
        x *= torch.exp(torch.randn(case["m"], 1, generator=gen, device=DEV))           # rows of different size
        if case["m"] > 8:
            x[case["m"] // 2] = 0                                                       # a row of padding
        return dict(case=case, x=_pitched(x.to(DTYPES[case["dtype"]]), case["pitch"]))
    if kind in ("product", "witness"):
        m, k, n = case["m"], case["k"], case["n"]
        a = _int8(gen, m, k)
        b = _int8(gen, n, k).t() if case["layout"] == "nk" else _int8(gen, k, n)
        s = dict(case=case, a=a, b=b)
        if kind == "product":
            s["sa"] = torch.rand(m, generator=gen, device=DEV) * 0.05 + 0.005
            s["sb"] = torch.rand(n, generator=gen, device=DEV) * 0.002 + 0.0002
        return s
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device=DEV) * 2.5
    likely = torch.randint(0, vocab, (rows, 12), generator=gen, device=DEV)
    x.scatter_add_(1, likely, torch.rand(rows, 12, generator=gen, device=DEV) * 14)     # a few likely tokens
    tokens = likely[:, 0].clone()
    x = x.to(DTYPES[case["dtype"]])
    if case["masked"] != "no":                                                          # tokens that are not allowed
        low = -math.inf if case["masked"] == "inf" else torch.finfo(x.dtype).min
        off = torch.rand(rows, vocab, generator=gen, device=DEV) < 0.3
        off.scatter_(1, tokens[:, None], False)
        x.masked_fill_(off, low)
    if rows > 8:
        tokens[rows // 3] = -1                                                          # a position without a token
    return dict(case=case, x=_pitched(x, case["pitch"]), tokens=tokens)


# ---- one pass ---------------------------------------------------------------------------------------------------
def _plain_quantize(x):
    """q = 127 x / (largest magnitude of the row), rounded half to even; scale = largest magnitude / 127.  The quotient
    in 64 bits, since a value next to a border would fall on it in 32."""
    x = x.double()
    big = x.abs().amax(1, keepdim=True)
    q = torch.where(big > 0, 127 * x / torch.where(big > 0, big, 1.0), 0.0).round()
    return q.to(torch.int8), (big[:, 0] / 127).float()


def _plain_product(a, b, sa, sb, dtype):
    """The sums reach 2^31, so they are made in 64 bits."""
    acc = a.double() @ b.double()
    if sa is None:
        acc = acc.to(torch.int64)
        return acc.to(torch.int32) if dtype == torch.int32 else torch.where(acc < 0, acc + (P - (1 << 64)), acc)
    return (acc.float() * sa[:, None] * sb).to(dtype)


def _plain_logprobs(x, tokens, top, temperature):
    x = x.float()
    z = (x - x.amax(1, keepdim=True)) / temperature
    e = z.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    given = z.gather(1, tokens.clamp(min=0)[:, None]) - log_total
    logprob = torch.where(tokens < 0, 0.0, given[:, 0])
    entropy = log_total[:, 0] - (e * z.clamp(min=-1e4)).sum(1) / total[:, 0]
    order = x.sort(dim=1, descending=True, stable=True)[1][:, :top]
    likely = z.gather(1, order) - log_total
    order = torch.where(likely == -math.inf, -1, order)
    return logprob, entropy, likely, order


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from verinf_b200 import int8, logprobs
        if kind == "quantize":
            return int8.int8_quantize_rows(state["x"])
        if kind == "product":
            return int8.int8_matmul(state["a"], state["b"], state["sa"], state["sb"], dtype=DTYPES[case["dtype"]])
        if kind == "witness":
            y = int8.int8_matmul(state["a"], state["b"], dtype=DTYPES[case["dtype"]])
            return y.view(torch.int64) if y.dtype == torch.uint64 else y
        return tuple(logprobs.token_logprobs(state["x"], state["tokens"], top=case["top"], temperature=case["temperature"]))
    if kind == "quantize":
        return _plain_quantize(state["x"])
    if kind in ("product", "witness"):
        return _plain_product(state["a"], state["b"], state.get("sa"), state.get("sb"), DTYPES[case["dtype"]])
    return _plain_logprobs(state["x"], state["tokens"], case["top"], case["temperature"])


# ---- work and definition -----------------------------------------------------------------------------------------
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "int32": 4, "field": 8}


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        mk = case["m"] * case["k"]
        return {"bytes": mk * (_SIZE[case["dtype"]] + 1) + 4 * case["m"], "flops": 3 * mk}      # |x| and max, product, rounding
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        # a row once, its token, log probability and entropy, its list; per entry a maximum, a difference, an exponential,
        # a sum and a weighted sum
        return {"bytes": n * _SIZE[case["dtype"]] + case["rows"] * (8 + 4 + 4 + 12 * case["top"]), "flops": 6 * n}
    m, k, n = case["m"], case["k"], case["n"]
    scales = 4 * (m + n) if kind == "product" else 0
    return {"bytes": m * k + k * n + m * n * _SIZE[case["dtype"]] + scales, "flops": 2 * m * k * n}


def _exact_sums(a, b):
    """int64 sums, slice by slice: 256 products of at most 2^14 stay whole in fp32."""
    acc = torch.zeros(a.size(0), b.size(1), dtype=torch.int64, device=DEV)
    for k in range(0, a.size(1), 256):
        acc += (a[:, k:k + 256].float() @ b[k:k + 256].float()).to(torch.int64)
    return acc


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x = s["x"].double()
        most = x.abs().max(1).values
        # whole numbers nearest to 127 x / most, ties to even: the remainder decides between the two neighbours
        big = torch.where(most == 0, 1.0, most)[:, None]
        low = torch.floor(127 * x / big)
        rest = 2 * (127 * x - low * big) / big
        up = (rest > 1) | ((rest == 1) & (low % 2 != 0))
        return (low + up).to(torch.int8), most / 127
    if kind in ("product", "witness"):
        acc = _exact_sums(s["a"], s["b"])
        if kind == "product":
            return acc.double() * s["sa"].double()[:, None] * s["sb"].double()[None, :]
        if case["dtype"] == "int32":
            return acc.to(torch.int32)
        return acc + (acc < 0).to(torch.int64) * (P - (1 << 64))
    logp = torch.log_softmax(s["x"].double() / case["temperature"], 1)
    tokens = s["tokens"]
    given = logp[torch.arange(len(tokens), device=DEV), tokens.clamp(min=0)]
    given = given * (tokens >= 0)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    taken = s["x"].double().clone()
    ids = torch.empty(len(tokens), case["top"], dtype=torch.int64, device=DEV)
    place = torch.arange(case["vocab"], device=DEV)
    for j in range(case["top"]):
        best = taken.max(1, keepdim=True).values
        ids[:, j] = torch.where(taken == best, place, case["vocab"]).min(1).values       # the lowest index among equals
        taken.scatter_(1, ids[:, j:j + 1], -math.inf)
    top = logp.gather(1, ids)
    return given, entropy, top, torch.where(top == -math.inf, -1, ids)

"""Performance cases of the 8-bit projections and of the log probabilities
(cq35.quantize_rows, norm_quantize, gated_quantize, int8_linear,
token_logprobs): what a round of batched serving runs before, between and
behind the paged-cache operators. `run` computes a case either in plain torch
operations or through the library's operators.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "catena-models_amd"))

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # a decode round's attention contexts before the output projection, 35B head counts
        dict(op="quantize", name="quantize: 16 rows of 4096", rows=16, channels=4096, type="bf16"),
        # the same of a large prompt round
        dict(op="quantize", name="quantize: 8192 rows of 4096", rows=8192, channels=4096, type="bf16"),
        # one token between two blocks of a layer: latency alone
        dict(op="norm", name="norm: 1 row of 2048", rows=1, channels=2048, type="bf16", residual=True),
        # a large prompt round, residual stream in and out
        dict(op="norm", name="norm: 8192 rows of 2048", rows=8192, channels=2048, type="bf16", residual=True),
        # a decode round with drafts at the 0.8B feed-forward width
        dict(op="gated", name="gated: 37 rows of 3584", rows=37, channels=3584, type="bf16"),
        # a large prompt round at the 2B feed-forward width
        dict(op="gated", name="gated: 8192 rows of 6144", rows=8192, channels=6144, type="bf16"),
        # one token through the 2B gate and up projections: the weights' bytes
        dict(op="linear", name="linear: 1 x 2048 to 12288", rows=1, channels=2048, outputs=12288, type="bf16"),
        # a mixed round through the 35B query, gate, key and value projections
        dict(op="linear", name="linear: 300 x 2048 to 9216", rows=300, channels=2048, outputs=9216, type="bf16"),
        # a large prompt round through the 2B gate and up projections
        dict(op="linear", name="linear: 8192 x 2048 to 12288", rows=8192, channels=2048, outputs=12288, type="bf16"),
        # one answered token with its alternatives
        dict(op="logprobs", name="logprobs: 1 row, top 8", rows=1, vocab=248320, given=1, top=8, type="bf16"),
        # a decode round that reports 20 alternatives, logits in 32 bits
        dict(op="logprobs", name="logprobs: 64 rows F32, top 20", rows=64, vocab=248320, given=1, top=20, type="f32"),
        # a prompt's tokens scored
        dict(op="logprobs", name="logprobs: 1000 rows scored", rows=1000, vocab=248320, given=1, top=1, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["quantize", "norm", "gated", "linear", "linear", "logprobs"])
    kind = rng.choice(["bf16", "bf16", "f32"])
    if op in ("quantize", "norm", "gated"):
        channels = 16 * _log(rng, 4, 1024)
        most = 8192 * 6144 // (channels * (2 if kind == "f32" else 1))
        case = dict(op=op, rows=_log(rng, 1, min(16384, most)), channels=channels, type=kind)
        return dict(case, residual=rng.random() < 0.7) if op == "norm" else case
    if op == "linear":
        channels = 16 * _log(rng, 8, 512)
        if rng.random() < 0.15:  # a vocabulary head
            return dict(op=op, rows=rng.randint(1, 64), channels=16 * _log(rng, 16, 128), outputs=248320, type=kind)
        outputs = _log(rng, 33, 16384)
        most = 8192 * 2048 * 12288 // (channels * outputs)
        return dict(op=op, rows=_log(rng, 1, min(8192, most)), channels=channels, outputs=outputs, type=kind)
    vocab = _log(rng, 1000, 248320)
    most = 1000 * 248320 // (vocab * (2 if kind == "f32" else 1))
    return dict(op=op, rows=_log(rng, 1, min(2000, most)), vocab=vocab, given=rng.choice([1, 1, 1, 4]),
                top=rng.choice([0, 1, 5, 20, 32]), type=kind)


# ------------------------------------------------------------------ inputs


def _normal(gen, shape, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=gen)


def _activations(gen, rows, channels):
    """Rows as a model makes them: a few channels are far larger than the others."""
    x = _normal(gen, (rows, channels))
    loud = torch.rand(channels, device="cuda", generator=gen) < 0.01
    return x * torch.where(loud, 8.0, 1.0)


def _int8(gen, rows, channels, std):
    """An 8-bit matrix and its scales, as quantised rows of normal values look."""
    amax = std * (3.5 + 0.5 * torch.rand(rows, device="cuda", generator=gen))
    x = torch.empty(rows, channels, dtype=torch.float16, device="cuda").normal_(0.0, 1.0, generator=gen)
    q = (x * (127.0 * std / amax[:, None]).half()).round().clamp(-127, 127).to(torch.int8)
    return q, amax / 127.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, dtype = case["op"], case["rows"], TYPES[case["type"]]
    s = dict(op=op, dtype=dtype)
    if op == "quantize":
        s["x"] = _activations(gen, rows, case["channels"]).to(dtype)
    elif op == "norm":
        s["x"] = _normal(gen, (rows, case["channels"])).to(dtype)
        s["residual"] = _activations(gen, rows, case["channels"]).to(dtype) if case["residual"] else None
        s["weight"] = _normal(gen, (case["channels"],), 0.02, 1.0)
        s["eps"] = 1e-6
    elif op == "gated":
        # the projection's result: gate and up behind each other in each row
        both = _normal(gen, (rows, 2 * case["channels"])).to(dtype)
        s["gate"], s["up"] = both[:, :case["channels"]], both[:, case["channels"]:]
    elif op == "linear":
        s["x"], s["w"] = _int8(gen, rows, case["channels"], 1.0), _int8(gen, case["outputs"], case["channels"], 0.02)
    else:
        x = torch.empty(rows, case["vocab"], dtype=dtype, device="cuda").normal_(0.0, 2.5, generator=gen)
        # likely tokens of each row, and tokens that a grammar or a filter rules out
        at = torch.randint(case["vocab"], (rows, 6), device="cuda", generator=gen)
        x.scatter_(1, at, _normal(gen, (rows, 6), 2.0, 12.0).to(dtype))
        s["tokens"] = torch.cat([at[:, :1], torch.randint(case["vocab"], (rows, 3), device="cuda", generator=gen)], 1)[:, :case["given"]].contiguous()
        out = torch.randint(case["vocab"], (rows, case["vocab"] // 50), device="cuda", generator=gen)
        s["logits"] = x.scatter_(1, out, float("-inf"))
        s["top"] = case["top"]
    return s


# ------------------------------------------------------------- plain forms


def _values(data, scale):
    """What 8-bit rows stand for."""
    out = torch.empty(data.shape, dtype=torch.bfloat16, device=data.device)
    return torch.mul(data, scale[:, None], out=out)


def _plain_rows(y):
    amax = y.abs().amax(-1)
    q = torch.round(y * (127.0 / amax)[:, None]).to(torch.int8)
    return q, amax / 127.0


def _plain_quantize(s):
    q, scale = _plain_rows(s["x"].float())
    return _values(q, scale), scale


def _plain_norm(s):
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["dtype"])
    x = h.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * s["weight"]
    q, scale = _plain_rows(y)
    return _values(q, scale), scale, h


def _plain_gated(s):
    gate = s["gate"].float()
    q, scale = _plain_rows(gate / (1.0 + torch.exp(-gate)) * s["up"].float())
    return _values(q, scale), scale


def _plain_linear(s):
    (x, sx), (w, sw) = s["x"], s["w"]
    sums = torch.matmul(x.float(), w.float().t())
    return (sums * sx[:, None] * sw).to(s["dtype"])


def _plain_logprobs(s):
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - (e * torch.where(e > 0, d, 0.0)).sum(-1, keepdim=True) / total
    # a key for each entry, larger for larger logits and, among equal ones, for lower indices
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -2147483648 - bits, bits)
    keys = order * 4294967296 + (4294967295 - torch.arange(x.shape[1], device=x.device))
    best = keys.topk(s["top"], -1).values
    tokens = 4294967295 - (best & 4294967295)
    return (d.gather(1, s["tokens"]) - log_total, entropy[:, 0], tokens, d.gather(1, tokens) - log_total)


def run(state):
    s = state
    op = s["op"]
    if own:
        import cq35
        if op == "quantize":
            q = cq35.quantize_rows(s["x"])
            return _values(q.data, q.scale), q.scale
        if op == "norm":
            q = cq35.norm_quantize(s["x"], s["weight"], residual=s["residual"], eps=s["eps"])
            return _values(q.data, q.scale), q.scale, q.summed
        if op == "gated":
            q = cq35.gated_quantize(s["gate"], s["up"])
            return _values(q.data, q.scale), q.scale
        if op == "linear":
            return cq35.int8_linear(s["x"], s["w"], dtype=s["dtype"])
        p = cq35.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        return p.logprobs, p.entropy, p.top_tokens, p.top_logprobs
    return {"quantize": _plain_quantize, "norm": _plain_norm, "gated": _plain_gated, "linear": _plain_linear,
            "logprobs": _plain_logprobs}[op](s)


def work(case):
    rows, b = case["rows"], BYTES[case["type"]]
    if case["op"] == "linear":
        K, N = case["channels"], case["outputs"]
        return {"bytes": (rows + N) * (K + 4) + rows * N * b, "flops": 2 * rows * N * K}
    if case["op"] == "logprobs":
        return {"bytes": rows * (case["vocab"] * b + 12 * case["given"] + 4 + 12 * case["top"]), "flops": 6 * rows * case["vocab"]}
    C = case["channels"]
    if case["op"] == "quantize":
        return {"bytes": rows * (C * b + C + 4), "flops": 3 * rows * C}
    if case["op"] == "gated":
        return {"bytes": rows * (2 * C * b + C + 4), "flops": 8 * rows * C}
    streams = 3 if case["residual"] else 1  # input, residual and sum, or the input alone
    return {"bytes": rows * (streams * C * b + C + 4) + 4 * C, "flops": 7 * rows * C}


# ------------------------------------------------------------ in 64 bits


def _exact_rows(y):
    scale = y.abs().max(-1).values / 127
    return (y / scale.unsqueeze(-1)).round() * scale.unsqueeze(-1), scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_rows(s["x"].double())
    if op == "norm":
        h = s["x"].double()
        if s["residual"] is not None:  # the sum of two values of 32 bits or fewer, to the stream's type
            h = (h + s["residual"].double()).to(s["dtype"]).double()
        variance = h.square().sum(-1) / h.shape[-1]
        return (*_exact_rows(h / (variance + s["eps"]).sqrt().unsqueeze(-1) * s["weight"].double()), h)
    if op == "gated":
        gate = s["gate"].double()
        return _exact_rows(gate * torch.sigmoid(gate) * s["up"].double())
    if op == "linear":
        (x, sx), (w, sw) = s["x"], s["w"]
        return (x.double() * sx.double().unsqueeze(1)) @ (w.double() * sw.double().unsqueeze(1)).t().contiguous()
    logits = s["logits"].double()
    normaliser = torch.logsumexp(logits, -1, keepdim=True)
    logits -= normaliser
    given = logits.gather(1, s["tokens"])
    best = logits.topk(s["top"], -1).values
    p = logits.exp()
    entropy = -(p * logits.masked_fill_(p == 0, 0.0)).sum(-1)
    return given, entropy, None, best

"""Measured cases of the operators on a language model's logits (montecarlo_amd.logits): the score of given tokens with
entropy and top alternatives, its gradient, the draw of tokens, and the keys of whole passwords.

``run`` computes them in plain torch (``own`` false) or through the framework (``own`` true) on what ``prepare`` made."""
import math

import torch

own = False

SKIP, OUTSIDE = -2, -1
LOG2E = 1.4426950408889634
IMPOSSIBLE = 1022.0
LOWEST = torch.finfo(torch.float32).min
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a password typed at a prompt: its dozen symbols scored at once, with what the model expected instead
        {"name": "score_one_password", "op": "score", "batch": 1, "length": 12, "vocab": 97, "dtype": "fp32", "entropy": True, "top": 5, "temperature": 1.0},
        # a test set of 65536 passwords under a character model (printable ASCII, start and end), padded to 16
        {"name": "score_test_set_chars", "op": "score", "batch": 65536, "length": 16, "vocab": 97, "dtype": "bf16", "entropy": True, "top": 0, "temperature": 1.0},
        # a test set under a sub-word model, with ten alternatives for each place
        {"name": "score_test_set_subwords", "op": "score", "batch": 512, "length": 16, "vocab": 32768, "dtype": "bf16", "entropy": True, "top": 10, "temperature": 1.0},
        # a wide vocabulary of odd size in full precision, many alternatives: the largest
        {"name": "score_wide_vocabulary", "op": "score", "batch": 683, "length": 3, "vocab": 131073, "dtype": "fp32", "entropy": True, "top": 32, "temperature": 1.3},
        # a training step of a byte model on padded passwords
        {"name": "gradient_bytes", "op": "gradient", "batch": 8192, "length": 31, "vocab": 257, "dtype": "bf16", "entropy": False, "temperature": 1.0},
        # a training step of a sub-word model with an entropy bonus, odd vocabulary
        {"name": "gradient_subwords", "op": "gradient", "batch": 256, "length": 16, "vocab": 50001, "dtype": "bf16", "entropy": True, "temperature": 1.0},
        # a small full-precision training step
        {"name": "gradient_full_precision", "op": "gradient", "batch": 37, "length": 21, "vocab": 8192, "dtype": "fp32", "entropy": False, "temperature": 1.0},
        # one step of an interactive generator: few rows, a wide vocabulary
        {"name": "draw_few_wide", "op": "draw", "rows": 8, "vocab": 131072, "dtype": "fp32", "temperature": 1.0, "live": 1.0},
        # one step of a million samples in flight under a character model
        {"name": "draw_million_chars", "op": "draw", "rows": 1048576, "vocab": 97, "dtype": "fp16", "temperature": 1.0, "live": 1.0},
        # a late step of samples under a sub-word model, a quarter of them ended, sharpened
        {"name": "draw_subwords_late", "op": "draw", "rows": 4096, "vocab": 32768, "dtype": "bf16", "temperature": 0.8, "live": 0.75},
        # the keys of one small batch of samples
        {"name": "keys_small_padded", "op": "keys", "batch": 1000, "length": 24, "packed": False},
        # the keys of a large test set, packed
        {"name": "keys_test_set_packed", "op": "keys", "batch": 2000003, "length": 24, "packed": True},
    ]


def draw(rng):
    op = rng.choice(["score", "score", "gradient", "gradient", "draw", "draw", "keys"])
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    if op == "keys":
        return {"op": op, "batch": log(3, 2000000), "length": log(1, 24), "packed": rng.random() < 0.5}
    vocab = log(32, 131072)
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    most = min(1 << 20, (1 << (27 if op == "score" else 26)) // vocab)
    rows = log(1, max(2, most))
    temperature = rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 3)])
    if op == "draw":
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "live": rng.choice([1.0, 0.8])}
    length = min(rows, log(1, 32))
    case = {"op": op, "batch": max(1, rows // length), "length": length, "vocab": vocab, "dtype": dtype, "entropy": rng.random() < 0.6, "temperature": temperature}
    if op == "score":
        case["top"] = rng.choice([0, 1, log(2, 32)])
    return case


def work(case):
    if case["op"] == "keys":
        n = case["batch"] * (case["length"] // 2 + 1)
        return {"bytes": 4 * n + 16 * case["batch"], "flops": n}
    if case["op"] == "draw":
        n = int(case["rows"] * case["live"]) * case["vocab"]
        return {"bytes": n * BYTES[case["dtype"]] + 17 * case["rows"], "flops": 4 * n}
    length, rows = case["length"], case["batch"] * case["length"]
    # the rows behind a password's end are not read (their gradient is written: zeros)
    read = int(rows * (max(1, length // 2) + length) / (2 * length)) * case["vocab"]
    if case["op"] == "gradient":
        return {"bytes": (read + rows * case["vocab"]) * BYTES[case["dtype"]] + 20 * rows, "flops": (12 if case["entropy"] else 9) * read}
    return {"bytes": read * BYTES[case["dtype"]] + (16 + 8 * case["top"]) * rows, "flops": (7 if case["entropy"] else 5) * read}


def _logits(shape, dtype, g):
    """Logits of a trained model's spread: noise of a few units, frequent tokens first, some tokens switched off, a few rows in
    which nothing is left and a few whose every token holds the lowest value."""
    x = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).mul_(2.5)
    vocab = shape[-1]
    x -= torch.log1p(torch.arange(vocab, device="cuda", dtype=torch.float32)) * 0.5
    x.masked_fill_(torch.rand(vocab, device="cuda", generator=g) < 0.02, -math.inf)
    rows = x.view(-1, vocab)
    if rows.shape[0] >= 64:
        rows[torch.randint(0, rows.shape[0], (1 + rows.shape[0] // 1024,), device="cuda", generator=g)] = -math.inf
        rows[torch.randint(0, rows.shape[0], (1 + rows.shape[0] // 1024,), device="cuda", generator=g)] = torch.finfo(dtype).min
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "keys":
        batch, length = case["batch"], case["length"]
        lengths = torch.randint(0, length + 1, (batch,), device="cuda", generator=g)
        n = int(lengths.sum()) if case["packed"] else batch * length
        ml2p = torch.empty(n, device="cuda", dtype=torch.float32).exponential_(0.3, generator=g)
        ml2p.masked_fill_(torch.rand(n, device="cuda", generator=g) < 0.001, math.inf)
        if not case["packed"]:
            return {"case": case, "ml2p": ml2p.view(batch, length), "lengths": lengths}
        offsets = torch.zeros(batch + 1, device="cuda", dtype=torch.int64)
        torch.cumsum(lengths, 0, out=offsets[1:])
        return {"case": case, "ml2p": ml2p, "offsets": offsets}
    vocab, dtype = case["vocab"], DTYPES[case["dtype"]]
    if op == "draw":
        rows = case["rows"]
        x = _logits((rows, vocab), dtype, g)
        u = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
        live = torch.rand(rows, device="cuda", generator=g) < case["live"] if case["live"] < 1.0 else None
        return {"case": case, "logits": x, "uniforms": u, "live": live}
    batch, length = case["batch"], case["length"]
    # a model's answer for a whole sequence: the logits at place i speak of token i + 1
    x = _logits((batch, length + 1, vocab), dtype, g)
    tokens = torch.empty((batch, length + 1), device="cuda", dtype=torch.int64)
    tokens[:, 1:] = torch.randint(0, vocab, (batch, length), device="cuda", generator=g)
    likely = x[:, :-1].argmax(-1)
    tokens[:, 1:] = torch.where(torch.rand((batch, length), device="cuda", generator=g) < 0.4, likely, tokens[:, 1:])
    tokens[:, 0] = 0
    tokens[torch.rand((batch, length + 1), device="cuda", generator=g) < 0.0005] = OUTSIDE
    end = torch.randint(max(1, length // 2), length + 1, (batch, 1), device="cuda", generator=g)
    tokens[torch.arange(length + 1, device="cuda")[None] > end] = SKIP
    state = {"case": case, "logits": x[:, :-1], "tokens": tokens[:, 1:]}
    if op == "gradient":
        n = batch * length
        state["weights"] = torch.rand((batch, length), device="cuda", generator=g) / n
        state["entropy_weights"] = (torch.rand((batch, length), device="cuda", generator=g) - 0.7) / n if case["entropy"] else None
    return state


def _softmax(x, temperature):
    """(y, w, Z) of every row: base-2 exponents below the largest logit, their powers and the powers' sum."""
    x = x.float()
    m = x.amax(-1, keepdim=True).clamp(min=LOWEST)
    y = (x - m) * (LOG2E / temperature)
    w = torch.exp2(y)
    return y, w, w.sum(-1)


def _score(y, w, z, tokens):
    """ml2p of the given tokens and the entropy."""
    vocab = y.shape[-1]
    empty, skipped = z == 0, tokens == SKIP
    inside = (tokens >= 0) & (tokens < vocab)
    at = y.gather(-1, tokens.clamp(0, vocab - 1)[..., None])[..., 0]
    ml2p = torch.where(inside & ~empty, torch.log2(z) - at, math.inf)
    ml2p = torch.where(torch.isnan(z), math.nan, ml2p).masked_fill(skipped, 0)
    entropy = torch.log2(z) - torch.where(w > 0, w * y, 0).sum(-1) / z
    return ml2p, entropy.masked_fill(empty | skipped, 0)


def _plain_score(s):
    case = s["case"]
    y, w, z = _softmax(s["logits"], case["temperature"])
    ml2p, entropy = _score(y, w, z, s["tokens"])
    out = {"ml2p": ml2p}
    if case["entropy"]:
        out["entropy"] = entropy
    k = case["top"]
    if k:
        # one whole number a token, larger for a larger logit and, among equals, for a lower index
        bits = (s["logits"].float() + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + torch.arange(y.shape[-1], 0, -1, device="cuda")
        ids = torch.topk(order, k, dim=-1).indices
        value = torch.log2(z)[..., None] - y.gather(-1, ids)
        gone = torch.isinf(value) | (z == 0)[..., None]
        none = gone | torch.isnan(z)[..., None]
        skipped = (s["tokens"] == SKIP)[..., None]
        out["top_tokens"] = torch.where(skipped, SKIP, torch.where(none, OUTSIDE, ids)).int()
        out["top_ml2p"] = value.masked_fill(gone, math.inf).masked_fill(skipped, 0)
    return out


def _plain_gradient(s):
    case, tokens = s["case"], s["tokens"]
    y, w, z = _softmax(s["logits"], case["temperature"])
    ml2p, entropy = _score(y, w, z, tokens)
    p = w / z[..., None]
    inside = (tokens >= 0) & (tokens < y.shape[-1])
    a = (s["weights"] * (LOG2E / case["temperature"]) * inside)[..., None]
    grad = a * p
    if case["entropy"]:
        b = (s["entropy_weights"] / case["temperature"])[..., None]
        grad -= b * torch.where(p > 0, p * (y - torch.log2(z)[..., None] + entropy[..., None]), 0)
    grad.scatter_add_(-1, tokens.clamp(0, y.shape[-1] - 1)[..., None], -a)
    grad = grad.masked_fill(((z == 0) | (tokens == SKIP))[..., None], 0)
    out = {"ml2p": ml2p, "grad": grad.to(s["logits"].dtype)}
    if case["entropy"]:
        out["entropy"] = entropy
    return out


def _plain_draw(s):
    case = s["case"]
    x = s["logits"].double()
    m = x.amax(-1, keepdim=True).clamp(min=LOWEST)
    y = (x - m) / case["temperature"]
    w = torch.exp(y)
    c = w.cumsum(-1)
    z = c[:, -1]
    at = (c <= (s["uniforms"] * z)[:, None]).sum(-1)
    at = torch.minimum(at, x.shape[-1] - 1 - (w > 0).flip(-1).int().argmax(-1))
    value = (torch.log(z) - y.gather(-1, at[:, None])[:, 0]) * LOG2E
    empty = z == 0
    tokens, value = at.masked_fill(empty, OUTSIDE), value.masked_fill(empty, math.inf)
    if s["live"] is not None:
        tokens, value = tokens.masked_fill(~s["live"], SKIP), value.masked_fill(~s["live"], 0)
    return {"tokens": tokens.int(), "ml2p": value.float()}


def _plain_keys(s):
    ml2p = s["ml2p"].double()
    if s["case"]["packed"]:
        lengths = s["offsets"].diff()
        owner = torch.repeat_interleave(torch.arange(lengths.numel(), device="cuda"), lengths, output_size=ml2p.numel())
        keys = torch.zeros(lengths.numel(), device="cuda", dtype=torch.float64).index_add_(0, owner, ml2p)
    else:
        there = torch.arange(ml2p.shape[1], device="cuda")[None] < s["lengths"][:, None]
        keys = torch.where(there, ml2p, 0).sum(-1)
    return {"keys": torch.where(torch.isinf(keys), IMPOSSIBLE, keys)}


def _own(s):
    from montecarlo_amd import logits as lg
    case = s["case"]
    if case["op"] == "score":
        r = lg.logits_score(s["logits"], s["tokens"], temperature=case["temperature"], entropy=case["entropy"], top=case["top"])
        return {k: v for k, v in r._asdict().items() if v is not None}
    if case["op"] == "gradient":
        r = lg.logits_gradient(s["logits"], s["tokens"], s["weights"], entropy_weights=s["entropy_weights"], temperature=case["temperature"])
        return {k: v for k, v in r._asdict().items() if v is not None}
    if case["op"] == "draw":
        return lg.logits_draw(s["logits"], s["uniforms"], temperature=case["temperature"], live=s["live"])._asdict()
    if case["packed"]:
        return {"keys": lg.logits_keys(s["ml2p"], offsets=s["offsets"])}
    return {"keys": lg.logits_keys(s["ml2p"], lengths=s["lengths"])}


def run(state):
    if own:
        return _own(state)
    return {"score": _plain_score, "gradient": _plain_gradient, "draw": _plain_draw, "keys": _plain_keys}[state["case"]["op"]](state)


def _exact_rows(x, temperature):
    """log p (natural) of every token in 64 bits, and whether the row has anything left."""
    left = (x > -math.inf).any(-1)
    x = x.double().masked_fill_(~left[..., None], 0)
    x = x.sub_(x.amax(-1, keepdim=True)).div_(temperature)  # (next to a lowest value the logarithm of the sum would be lost)
    return x.sub_(torch.logsumexp(x, -1)[..., None]).masked_fill_(~left[..., None], -math.inf), left


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "keys":
        ml2p = s["ml2p"].double()
        if case["packed"]:
            bad = torch.isinf(ml2p)
            edge = torch.zeros(ml2p.numel() + 1, device="cuda", dtype=torch.float64)
            torch.cumsum(ml2p.masked_fill(bad, 0), 0, out=edge[1:])
            hits = torch.zeros(ml2p.numel() + 1, device="cuda", dtype=torch.int64)
            torch.cumsum(bad, 0, out=hits[1:])
            return {"keys": edge[s["offsets"]].diff().masked_fill(hits[s["offsets"]].diff() > 0, IMPOSSIBLE)}
        place = torch.arange(case["length"], device="cuda").expand(case["batch"], -1)
        keys = ml2p.masked_fill(place >= s["lengths"][:, None], 0).sum(-1)
        return {"keys": keys.masked_fill(torch.isinf(keys), IMPOSSIBLE)}
    logp, left = _exact_rows(s["logits"], case["temperature"])
    vocab = logp.shape[-1]
    if case["op"] == "draw":
        c = torch.exp(logp).cumsum(-1)
        at = torch.searchsorted(c, (s["uniforms"] * c[:, -1])[:, None], right=True)[:, 0].clamp(max=vocab - 1)
        value = (-logp.gather(-1, at[:, None])[:, 0] / math.log(2)).masked_fill(~left, math.inf)
        at = at.masked_fill(~left, OUTSIDE)
        if s["live"] is not None:
            at, value = at.masked_fill(~s["live"], SKIP), value.masked_fill(~s["live"], 0)
        return {"tokens": at, "ml2p": value}
    tokens = s["tokens"]
    skipped, inside = tokens == SKIP, (tokens >= 0) & (tokens < vocab)
    picked = logp.gather(-1, tokens.clamp(0, vocab - 1)[..., None])[..., 0]
    ml2p = torch.where(inside, -picked / math.log(2), math.inf).masked_fill(skipped, 0)
    p = torch.exp(logp)
    entropy = torch.special.entr(p).sum(-1).masked_fill(skipped, 0) / math.log(2)
    out = {"ml2p": ml2p}
    if case["entropy"]:
        out["entropy"] = entropy
    if case["op"] == "score":
        if case["top"]:
            value = -torch.topk(logp, case["top"], dim=-1).values / math.log(2)
            out["top_tokens"] = None
            out["top_ml2p"] = value.masked_fill(skipped[..., None], 0)
        return out
    hit = torch.zeros_like(p).scatter_(-1, tokens.clamp(0, vocab - 1)[..., None], 1.0)
    a = (s["weights"].double() * inside / (math.log(2) * case["temperature"]))[..., None]
    grad = a * (p - hit)
    if case["entropy"]:
        b = (s["entropy_weights"].double() / case["temperature"])[..., None]
        grad += b * (torch.special.entr(p) / math.log(2) - p * entropy[..., None])
    out["grad"] = grad.masked_fill((skipped | ~left)[..., None], 0)
    return out

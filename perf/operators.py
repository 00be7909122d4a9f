"""Cases of the operators that train an embedding table: lookup with scaling
and its gradient, log probabilities with entropy and top alternatives and
their gradient, and the clipping of gradients by their global norm.

Each case names its operator (``op``) and its sizes. ``run`` computes it in
elementary torch operations where ``own`` is false and through
``ai_b200.train`` where it is true; ``exact`` computes it in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
PAD = 0  # the tokenizer's padding id: no row of its own, no gradient


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one query's tokens against a checkpoint's bf16 table: a search's latency
        {"name": "lookup_query", "op": "lookup", "tokens": 24, "vocab": 262144, "dim": 768,
         "table": "bfloat16", "dtype": "float32"},
        # the tokens of a batch of 256 x 512 from the widened table
        {"name": "lookup_batch", "op": "lookup", "tokens": 131072, "vocab": 262144, "dim": 768,
         "table": "float32", "dtype": "float32"},
        # a small model's table (vocabulary 2048) after a batch of 8 x 128, gradients in bf16
        {"name": "grad_small_table", "op": "grad", "tokens": 1024, "vocab": 2048, "dim": 768,
         "dtype": "bfloat16", "out": "float32"},
        # the whole table's gradient after a batch of 256 x 512
        {"name": "grad_batch", "op": "grad", "tokens": 131072, "vocab": 262144, "dim": 768,
         "dtype": "float32", "out": "float32"},
        # the rows that a few sentences touch of a table with 256 columns
        {"name": "rows_sentences", "op": "rows", "tokens": 333, "vocab": 262144, "dim": 256,
         "dtype": "float32", "out": "float32"},
        # the rows that 16 sequences of 2048 touch, gradients in bf16
        {"name": "rows_long", "op": "rows", "tokens": 32768, "vocab": 262144, "dim": 768,
         "dtype": "bfloat16", "out": "float32"},
        # one encoder layer's gradients: bf16 matrices, fp32 norms
        {"name": "clip_layer", "op": "clip", "layers": 1, "hidden": 768, "inter": 1152, "vocab": 0,
         "dtype": "mixed", "std": 0.01, "max_norm": 1.0},
        # every gradient of the 24-layer encoder and its table, in fp32
        {"name": "clip_model", "op": "clip", "layers": 24, "hidden": 768, "inter": 1152, "vocab": 262144,
         "dtype": "float32", "std": 0.001, "max_norm": 1.0},
        # one token's logits over the vocabulary, with 20 alternatives
        {"name": "logprobs_token", "op": "logprobs", "rows": 1, "width": 262144, "pad": 0, "dtype": "bfloat16",
         "scale": 1.0, "top": 20, "masked": False},
        # in-batch candidates of 8192 queries at temperature 0.05, the 8 hardest reported
        {"name": "logprobs_batch", "op": "logprobs", "rows": 8192, "width": 8192, "pad": 0, "dtype": "float32",
         "scale": 20.0, "top": 8, "masked": False},
        # a few rows of an odd width in bf16, with an entropy term and masked candidates
        {"name": "logprobs_grad_odd", "op": "logprobs_grad", "rows": 37, "width": 30011, "pad": 0,
         "dtype": "bfloat16", "scale": 1.0, "entropy": True, "masked": True},
        # the contrastive loss's gradient over the 8192 x 8192 similarities
        {"name": "logprobs_grad_batch", "op": "logprobs_grad", "rows": 8192, "width": 8192, "pad": 0,
         "dtype": "float32", "scale": 20.0, "entropy": False, "masked": False},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(["lookup", "grad", "rows", "clip", "logprobs", "logprobs_grad"])
    kind = rng.choice(["float32", "bfloat16", "float16"])
    if op in ("lookup", "grad", "rows"):
        dim = rng.choice([64, 256, 512, 768, 1024, _spread(rng, 8, 1024), _spread(rng, 8, 1024) | 1])
        vocab = _spread(rng, 500, 262144)
        tokens = _spread(rng, 1, 131072)
        case = {"op": op, "tokens": tokens, "vocab": vocab, "dim": dim, "dtype": kind}
        if op == "lookup":
            return {**case, "table": rng.choice(["float32", "bfloat16", "float16"])}
        return {**case, "out": rng.choice(["float32", kind])}
    if op == "clip":
        return {"op": op, "layers": rng.randint(1, 24), "hidden": _spread(rng, 32, 768), "inter": _spread(rng, 64, 1152),
                "vocab": rng.choice([0, _spread(rng, 500, 262144)]), "dtype": rng.choice(["float32", "bfloat16", "mixed"]),
                "std": 10.0 ** rng.uniform(-5, 0), "max_norm": rng.choice([0.5, 1.0, 10.0])}
    width = _spread(rng, 2, 262144)
    rows = _spread(rng, 1, max(1, min(16384, 67108864 // width)))
    case = {"op": op, "rows": rows, "width": width, "pad": rng.choice([0, 0, 1, (-width) % 8]), "dtype": kind,
            "scale": rng.choice([1.0, 10.0, 20.0, 50.0]), "masked": rng.random() < 0.5}
    if op == "logprobs":
        return {**case, "top": min(width, rng.choice([0, 1, 5, 8, 20, 64]))}
    return {**case, "entropy": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ids(case, g):
    """Token ids as texts have them: frequent ones low (density 1 / id), a
    BOS in every 128, one in sixteen of them padding."""
    n, vocab = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    ids = (vocab ** u).long().clamp_(1, vocab - 1)
    ids[::128] = 2
    ids[torch.rand(n, generator=g, device=DEV) < 1 / 16] = PAD
    return ids.int()


def _shapes(case):
    """The encoder's gradients: (shape, whether a norm's) in order."""
    h, f, d = case["hidden"], case["inter"], max(1, case["hidden"] // 3)
    got = [((case["vocab"], h), False)] if case["vocab"] else []
    for _ in range(case["layers"]):
        got += [((3 * d, h), False), ((d, h), False), ((d, h), False), ((h, 3 * d), False),
                ((f, h), False), ((f, h), False), ((h, f), False)]
        got += [((h,), True)] * 4 + [((d,), True)] * 2
    return got + [((h,), True)]


def _views(flat, shapes):
    got, at = [], 0
    for s in shapes:
        got.append(flat[at:at + math.prod(s)].view(s))
        at += math.prod(s)
    return got


def _logits(case, g):
    """Similarity rows (cosines, the pair's above the others' by 4 after the
    temperature, as in training) where a temperature is given, else logits;
    rows `pad` values apart from their width."""
    rows, width = case["rows"], case["width"]
    buf = torch.empty(rows, width + case["pad"], device=DEV, dtype=TYPES[case["dtype"]])
    spread = 768 ** -0.5 if case["scale"] > 1 else 2.5
    x = torch.randn(rows, width, generator=g, device=DEV).mul_(spread)
    t = torch.randint(0, width, (rows,), generator=g, device=DEV)
    x[torch.arange(rows, device=DEV), t] += 4.0 / case["scale"]
    if case["masked"]:  # one candidate in fifty is the query's own text; the last of several rows has none left
        x[torch.rand(rows, width, generator=g, device=DEV) < 0.02] = -math.inf
        if rows > 1:
            x[-1] = -math.inf
    buf.zero_()
    buf[:, :width] = x
    t[torch.rand(rows, generator=g, device=DEV) < 0.03] = -1  # rows without a pair
    return buf[:, :width], t.int()


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    state = {"case": case, "op": op}
    if op == "lookup":
        table = torch.randn(case["vocab"], case["dim"], generator=g, device=DEV).mul_(0.02).to(TYPES[case["table"]])
        return {**state, "table": table, "ids": _ids(case, g), "scale": case["dim"] ** 0.5, "dtype": TYPES[case["dtype"]]}
    if op in ("grad", "rows"):
        dy = torch.randn(case["tokens"], case["dim"], generator=g, device=DEV).mul_(1e-3).to(TYPES[case["dtype"]])
        return {**state, "dy": dy, "ids": _ids(case, g), "vocab": case["vocab"], "scale": case["dim"] ** 0.5,
                "dtype": TYPES[case["out"]]}
    if op == "clip":
        shapes = _shapes(case)
        wide = [s for s, norm in shapes if case["dtype"] == "float32" or (norm and case["dtype"] == "mixed")]
        thin = [s for s, norm in shapes if case["dtype"] == "bfloat16" or (not norm and case["dtype"] == "mixed")]
        state.update(grads=[], outs=[], flat={})
        for name, part in (("float32", wide), ("bfloat16", thin)):
            if part:
                n = sum(math.prod(s) for s in part)
                flat = torch.randn(n, generator=g, device=DEV).mul_(case["std"]).to(TYPES[name])
                out = torch.empty_like(flat)
                state["grads"] += _views(flat, part)
                state["outs"] += _views(out, part)
                state["flat"][name] = out
        state["max_norm"] = case["max_norm"]
        return state
    x, t = _logits(case, g)
    state.update(logits=x, targets=t, scale=case["scale"])
    if op == "logprobs":
        state["top"] = case["top"]
        return state
    # what the forward pass left: the log sums and the entropies, and the loss's share of each row
    kept = _plain_logprobs(x, t, case["scale"], 0)
    state.update(lse=kept["lse"], entropy=kept["entropy"],
                 dlogprob=torch.randn(case["rows"], generator=g, device=DEV) / case["rows"] - 1.0 / case["rows"],
                 dentropy=torch.full((case["rows"],), 0.01 / case["rows"], device=DEV) if case["entropy"] else None)
    return state


# ------------------------------------------------------------- plain forms
def _plain_lookup(s):
    ids = s["ids"].long()
    y = s["table"][ids].float() * s["scale"]
    return (y * (ids != PAD)[:, None]).to(s["dtype"])


def _plain_grad(s):
    ids = s["ids"].long()
    dy = s["dy"].float() * s["scale"] * (ids != PAD)[:, None]
    total = torch.zeros(s["vocab"], dy.shape[1], device=DEV).index_add_(0, ids, dy)
    return total.to(s["dtype"])


def _plain_rows(s):
    ids = s["ids"].long()
    n, kept = len(ids), ids != PAD
    met = torch.zeros(s["vocab"], dtype=torch.int64, device=DEV)
    met[ids] = 1
    met[PAD] = 0
    order = met.cumsum(0)  # a row's place among the rows met, from 1
    place = torch.where(kept, order[ids] - 1, n)
    rows = torch.zeros(n + 1, s["dy"].shape[1], device=DEV).index_add_(0, place, s["dy"].float() * s["scale"])
    row_ids = torch.full((n + 1,), -1, dtype=torch.int32, device=DEV)
    row_ids[place] = s["ids"]
    return {"ids": row_ids[:n], "rows": rows[:n].to(s["dtype"]), "count": order[-1:].int()}


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    c = torch.where(norm.isfinite() & (norm > s["max_norm"]), s["max_norm"] / norm, torch.ones_like(norm))
    done = [(g.float() * c).to(g.dtype).reshape(-1) for g in s["grads"]]
    kinds = {name: [d for d in done if d.dtype == TYPES[name]] for name in s["flat"]}
    return {"norm": norm, "grads": {name: torch.cat(part) for name, part in kinds.items()}}


def _plain_logprobs(logits, targets, scale, top):
    x = logits.float()
    m = x.amax(1, keepdim=True)
    empty = (m == -math.inf)[:, 0]
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    d = (x - m) * scale
    e = d.exp()
    s1 = e.sum(1)
    s2 = torch.where(e == 0, torch.zeros_like(e), e * d).sum(1)
    logs = s1.log()
    lse = m[:, 0] * scale + logs
    entropy = torch.where(empty, torch.zeros_like(s1), logs - s2 / s1)
    t = targets.long()
    logp = d.gather(1, t.clamp(min=0)[:, None])[:, 0] - logs
    logp = torch.where(empty, torch.full_like(logp, -math.inf), logp)
    out = {"logprob": torch.where(t < 0, torch.zeros_like(logp), logp), "entropy": entropy, "lse": lse}
    if top:
        value, index = x.sort(dim=1, descending=True, stable=True)
        value, index = (value[:, :top] - m) * scale - logs[:, None], index[:, :top]
        out["top_logprob"] = torch.where(empty[:, None], torch.full_like(value, -math.inf), value)
        out["top_index"] = index.int()
    return out


def _plain_logprobs_grad(s):
    x = s["logits"].float() * s["scale"]
    lse = s["lse"][:, None]
    logp = x - lse
    p = logp.exp()
    t = s["targets"].long()[:, None]
    hit = torch.arange(x.shape[1], device=DEV)[None, :] == t
    g = torch.where(t < 0, torch.zeros_like(lse), s["dlogprob"][:, None])
    dx = g * (hit.float() - p)
    if s["dentropy"] is not None:
        part = torch.where(p == 0, torch.zeros_like(p), p * (logp + s["entropy"][:, None]))
        dx = dx - s["dentropy"][:, None] * part
    dx = torch.where(lse == -math.inf, torch.zeros_like(dx), dx * s["scale"])
    return dx.to(s["logits"].dtype)


def _plain(s):
    op = s["op"]
    if op == "lookup":
        return _plain_lookup(s)
    if op == "grad":
        return _plain_grad(s)
    if op == "rows":
        return _plain_rows(s)
    if op == "clip":
        return _plain_clip(s)
    if op == "logprobs":
        return _plain_logprobs(s["logits"], s["targets"], s["scale"], s["top"])
    return _plain_logprobs_grad(s)


# ---------------------------------------------------------------- one pass
def run(state):
    s = state
    if not own:
        return _plain(s)
    from ai_b200 import train

    op = s["op"]
    if op == "lookup":
        return train.Embedding(s["table"], s["ids"], scale=s["scale"], padding=PAD, dtype=s["dtype"])
    if op == "grad":
        return train.EmbeddingGrad(s["dy"], s["ids"], s["vocab"], scale=s["scale"], padding=PAD, dtype=s["dtype"])
    if op == "rows":
        r = train.EmbeddingGradRows(s["dy"], s["ids"], s["vocab"], scale=s["scale"], padding=PAD, dtype=s["dtype"])
        return {"ids": r.Ids, "rows": r.Rows, "count": r.Count}
    if op == "clip":
        norm = train.ClipGradNorm(s["grads"], s["max_norm"], out=s["outs"])
        return {"norm": norm, "grads": s["flat"]}
    if op == "logprobs":
        r = train.LogProbs(s["logits"], s["targets"], scale=s["scale"], top=s["top"])
        out = {"logprob": r.LogProb, "entropy": r.Entropy, "lse": r.LogSum}
        if s["top"]:
            out.update(top_logprob=r.TopLogProb, top_index=r.TopIndex)
        return out
    return train.LogProbsGrad(s["logits"], s["targets"], s["lse"], s["dlogprob"], entropy=s["entropy"],
                              dentropy=s["dentropy"], scale=s["scale"])


# -------------------------------------------------------------------- work
def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    op = case["op"]
    if op in ("lookup", "grad", "rows"):
        n, d = case["tokens"], case["dim"]
        if op == "lookup":
            return {"bytes": n * (4 + d * (_size(case["table"]) + _size(case["dtype"]))), "flops": n * d}
        written = case["vocab"] if op == "grad" else n
        extra = 0 if op == "grad" else 4 * n + 4
        return {"bytes": n * (4 + d * _size(case["dtype"])) + written * d * _size(case["out"]) + extra, "flops": 2 * n * d}
    if op == "clip":
        total = sum(math.prod(s) * (4 if case["dtype"] == "float32" or (norm and case["dtype"] == "mixed") else 2)
                    for s, norm in _shapes(case))
        values = sum(math.prod(s) for s, _ in _shapes(case))
        return {"bytes": 2 * total + 4, "flops": 3 * values}
    rows, width, size = case["rows"], case["width"], _size(case["dtype"])
    if op == "logprobs":
        return {"bytes": rows * (width * size + 16 + 8 * case["top"]), "flops": 6 * rows * width}
    return {"bytes": rows * (2 * width * size + 12), "flops": 4 * rows * width}


# ----------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        w = s["table"].double()
        w[PAD] = 0
        return torch.nn.functional.embedding(s["ids"].long(), w) * s["scale"]
    if op in ("grad", "rows"):
        # tokens brought together by a sort; a run's sum is a difference of running totals
        ids, order = s["ids"].long().sort(stable=True)
        sums = s["dy"][order].double().cumsum(0)
        met, runs = ids.unique_consecutive(return_counts=True)
        end = runs.cumsum(0) - 1
        total = sums[end] * s["scale"]
        total[1:] -= sums[end[:-1]] * s["scale"]
        met, total = met[met != PAD], total[met != PAD]
        if op == "grad":
            out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device=DEV)
            out[met] = total
            return out
        rows = torch.zeros(len(ids), case["dim"], dtype=torch.float64, device=DEV)
        rows[:len(met)] = total
        return {"ids": None, "rows": rows, "count": None}
    if op == "clip":
        flat = {}
        for name in s["flat"]:
            flat[name] = torch.cat([g.reshape(-1) for g in s["grads"] if g.dtype == TYPES[name]]).double()
        norm = sum(torch.dot(f, f) for f in flat.values()) ** 0.5
        c = min(1.0, case["max_norm"] / float(norm))
        return {"norm": norm, "grads": {name: f * c for name, f in flat.items()}}
    z = s["logits"].double() * case["scale"]
    empty = torch.isinf(z).all(1)
    z[empty] = 0  # any finite row: these rows' values are put right below
    t = s["targets"].long()
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    h = torch.special.entr(p).sum(1)
    h[empty] = 0
    at = torch.arange(len(t), device=DEV)
    if op == "logprobs":
        picked = logp[at, t.clamp(min=0)]
        picked[empty] = -math.inf
        picked[t < 0] = 0
        lse = torch.logsumexp(z, 1)
        lse[empty] = -math.inf
        out = {"logprob": picked, "entropy": h, "lse": lse}
        if case["top"]:
            best = logp.topk(case["top"], dim=1).values
            best[empty] = -math.inf
            out.update(top_logprob=best, top_index=None)
        return out
    # the chain rule, from log p and the entropies
    one = torch.zeros_like(p)
    one[at[t >= 0], t[t >= 0]] = 1
    g = s["dlogprob"].double() * (t >= 0)
    dz = (one - p) * g[:, None]
    if s["dentropy"] is not None:
        dz += (torch.special.entr(p) - p * h[:, None]) * s["dentropy"].double()[:, None]
    dz[empty] = 0
    return dz * case["scale"]

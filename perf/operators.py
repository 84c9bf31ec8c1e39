"""The model-side operators around the collectives, as measured: the embedding lookup of a vocabulary
shard and its gradient by sorted tokens, the router of a mixture of experts and its gradient, and a
whole mixture-of-experts layer for a few tokens.

Where `own` is false, run() computes them in plain torch (32 bits, rounded once at the end); where it
is true, it makes the calls of torch_ccl_amd that a user makes.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _mccl():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    package = os.path.join(root, "torch-ccl_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import torch_ccl_amd
    return torch_ccl_amd


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _embedding(name, n, vocab, rows, first, hidden, dtype, scale):
    """n ids out of a vocabulary of `vocab`; the table holds `rows` of it, from id `first` on."""
    return {"name": name, "op": "embedding", "n": n, "vocab": vocab, "rows": rows, "first": first, "hidden": hidden,
            "dtype": dtype, "scale": scale}


def _grad(name, n, vocab, rows, first, hidden, dtype, out, accumulate, hot, scale):
    """The gradient of such a lookup: `hot` is the share of the tokens that are one and the same id."""
    return {"name": name, "op": "embedding_grad", "n": n, "vocab": vocab, "rows": rows, "first": first, "hidden": hidden,
            "dtype": dtype, "out": out, "accumulate": accumulate, "hot": hot, "scale": scale}


def _route(name, tokens, experts, topk, dtype, normalize, train, masked):
    """`train`: the gradient as well; `masked`: every so many-th expert is closed (-inf), 0 = none."""
    return {"name": name, "op": "moe_route", "tokens": tokens, "experts": experts, "topk": topk, "dtype": dtype,
            "normalize": normalize, "train": train, "masked": masked}


def _layer(name, tokens, topk, experts, local, first, hidden, inter, dtype, activation, padded):
    """`local` of `experts` experts, from `first` on, are this rank's; the last `padded` tokens are padding (expert -1)."""
    return {"name": name, "op": "moe_layer", "tokens": tokens, "topk": topk, "experts": experts, "local": local, "first": first,
            "hidden": hidden, "inter": inter, "dtype": dtype, "activation": activation, "padded": padded}


def listed():
    return [
        # one decode step of 8 requests on one of 8 vocabulary shards: latency
        _embedding("embed decode 8", 8, 32000, 4000, 12000, 4096, "bf16", 1.0),
        # a training batch of 8 x 4096 tokens over a whole table, rows of the dispatch workload, scaled by sqrt(hidden)
        _embedding("embed train 32768", 32768, 32000, 32000, 0, 7168, "bf16", math.sqrt(7168.0)),
        # a small model's step with rows that are no whole number of vectors
        _grad("grad small odd", 77, 1000, 1000, 0, 521, "f32", "f32", False, 0.1, 1.0),
        # a training batch over a whole table, a sixteenth of it one frequent token
        _grad("grad train 16384", 16384, 32000, 32000, 0, 4096, "bf16", "bf16", False, 0.0625, 64.0),
        # a micro-batch added into one of 8 vocabulary shards' fp32 gradient, a quarter of it padding
        _grad("grad shard accumulate", 32768, 128000, 16000, 0, 7168, "bf16", "f32", True, 0.25, 1.0),
        # the router of one decode step
        _route("route decode 16", 16, 256, 8, "f32", True, False, 0),
        # the router of the dispatch workload's batch on all 8 ranks, forward and gradient
        _route("route train 32768", 32768, 256, 8, "bf16", True, True, 0),
        # one token: every byte of 8 experts for one row
        _layer("layer 1 token", 1, 8, 64, 64, 0, 4096, 1024, "bf16", "silu", 0),
        # a decode batch of 8 requests, 3 of them padding
        _layer("layer 8 tokens", 8, 8, 128, 128, 0, 2048, 768, "bf16", "silu", 3),
        # a decode batch on one of 8 expert-parallel ranks of the dispatch workload's model
        _layer("layer 32 tokens shard", 32, 8, 256, 32, 64, 7168, 2048, "bf16", "silu", 0),
        # few wide experts and many tokens each
        _layer("layer 160 tokens wide", 160, 2, 8, 8, 0, 4096, 7168, "f16", "gelu", 0),
        # a small model with ragged sizes
        _layer("layer 5 tokens ragged", 5, 3, 34, 34, 0, 520, 200, "f16", "gelu", 0),
    ]


def _between(rng, lo, hi):
    """Spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding_grad", "embedding_grad", "moe_route", "moe_layer", "moe_layer", "moe_layer"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op in ("embedding", "embedding_grad"):
        n, hidden = _between(rng, 1, 32768), _between(rng, 64, 7168)
        vocab = _between(rng, 500, 60000)
        shards = rng.choice([1, 1, 2, 8])
        rows = (vocab + shards - 1) // shards
        first = rows * rng.randrange(shards)
        rows = max(1, min(rows, vocab - first))
        scale = rng.choice([1.0, 0.5, math.sqrt(hidden)])
        if op == "embedding":
            if dtype == "f32":
                n = (n + 1) // 2
            c = _embedding("", n, vocab, rows, first, hidden, dtype, scale)
        else:
            rows = max(1, min(rows, 2 ** 27 // hidden))
            c = _grad("", (n + 1) // 2, vocab, rows, first, hidden, dtype, rng.choice([dtype, "f32"]), rng.random() < 0.4,
                      rng.choice([0.0, 0.1, 0.5]), scale)
    elif op == "moe_route":
        experts = _between(rng, 4, 512)
        c = _route("", _between(rng, 1, 32768), experts, rng.randint(1, min(8, experts)), dtype, rng.random() < 0.5,
                   rng.random() < 0.6, rng.choice([0, 0, 3, 5]))
        c["tokens"] = min(c["tokens"], 2 ** 23 // experts)
    else:
        hidden, inter = 8 * _between(rng, 32, 896), 8 * _between(rng, 16, 512)
        experts = _between(rng, 4, 256)
        shards = rng.choice([1, 1, 2, 4])
        local = max(1, min(experts // shards, 2 ** 30 // (3 * hidden * inter)))
        first = rng.randrange(0, experts - local + 1)
        tokens = _between(rng, 1, 160)
        c = _layer("", tokens, rng.randint(1, min(8, experts)), experts, local, first, hidden, inter, rng.choice(["bf16", "f16"]),
                   rng.choice(["silu", "gelu"]), rng.choice([0, 0, tokens // 3]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _ids(case, g):
    """Token ids as text has them: the frequency of id v falls as 1 / (v + 1), and a share `hot` is one id of the shard."""
    n, vocab = case["n"], case["vocab"]
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).floor().to(torch.int64).clamp_(0, vocab - 1)
    hot = case.get("hot", 0.0)
    if hot:
        ids = torch.where(torch.rand(n, generator=g, device=DEV) < hot, torch.full_like(ids, case["first"] + case["rows"] // 2), ids)
    return ids


def _normal(shape, std, dtype, g):
    return torch.empty(shape, dtype=TYPES[dtype], device=DEV).normal_(0.0, std, generator=g)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "embedding":
        s["table"] = _normal((case["rows"], case["hidden"]), 0.02, case["dtype"], g)
        s["ids"] = _ids(case, g)
    elif case["op"] == "embedding_grad":
        s["ids"] = _ids(case, g)
        s["grad"] = _normal((case["n"], case["hidden"]), 1.0, case["dtype"], g)
        if case["accumulate"]:
            s["main"] = _normal((case["rows"], case["hidden"]), 1.0, case["out"], g)
    elif case["op"] == "moe_route":
        T, E, k = case["tokens"], case["experts"], case["topk"]
        s["logits"] = _normal((T, E), 1.0, case["dtype"], g)
        if case["masked"]:
            s["logits"][:, ::case["masked"]] = float("-inf")
        if case["train"]:
            s["grad_weights"] = _normal((T, k), 1.0, "f32", g)
    else:
        T, k, H, I = case["tokens"], case["topk"], case["hidden"], case["inter"]
        s["x"] = _normal((T, H), 1.0, case["dtype"], g)
        s["w_in"] = _normal((case["local"], 2 * I, H), 1.0 / math.sqrt(H), case["dtype"], g)
        s["w_out"] = _normal((case["local"], H, I), 1.0 / math.sqrt(I), case["dtype"], g)
        # experts differ in how often they are chosen
        logits = _normal((T, case["experts"]), 1.0, "f32", g) + _normal((1, case["experts"]), 0.5, "f32", g)
        top = torch.sort(logits, dim=1, descending=True, stable=True)
        s["ids"] = top.indices[:, :k].to(torch.int32).contiguous()
        s["weights"] = torch.softmax(top.values[:, :k], dim=1).contiguous()
        if case["padded"]:
            s["ids"][T - case["padded"]:] = -1
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _keys(ids, first, rows):
    r = ids - first
    return torch.where((r >= 0) & (r < rows), r, torch.full_like(r, rows))


def _plain_embedding(s, c):
    key = _keys(s["ids"], c["first"], c["rows"])
    inside = key < c["rows"]
    picked = s["table"][torch.where(inside, key, torch.zeros_like(key))].float() * c["scale"]
    return torch.where(inside[:, None], picked, torch.zeros_like(picked)).to(TYPES[c["dtype"]])


def _plain_grad(s, c):
    key = _keys(s["ids"], c["first"], c["rows"])
    in_order, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(in_order, torch.arange(c["rows"] + 1, device=DEV))
    total = torch.zeros(c["rows"] + 1, c["hidden"], dtype=torch.float32, device=DEV)
    total.index_add_(0, key, s["grad"].float())
    total = total[:-1] * c["scale"]
    if c["accumulate"]:
        s["main"].copy_(s["main"].float() + total)
        total = s["main"]
    return {"grad": total.to(TYPES[c["out"]]), "order": order, "offsets": offsets}


def _plain_route(s, c):
    logits = s["logits"].float()
    k, experts = c["topk"], c["experts"]
    values, places = torch.sort(logits, dim=1, descending=True, stable=True)
    values, ids = values[:, :k], places[:, :k]
    chosen = values > float("-inf")
    e = torch.exp(logits - values[:, :1])
    p = e / e.sum(dim=1, keepdim=True)
    w = torch.where(chosen, p.gather(1, ids), torch.zeros_like(values))
    if c["normalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    out = {"ids": torch.where(chosen, ids, torch.full_like(ids, -1)).to(torch.int32), "weights": w}
    if c["train"]:
        g = torch.where(chosen, s["grad_weights"], torch.zeros_like(w))
        mean = (g * w).sum(dim=1, keepdim=True)
        if c["normalize"]:
            d = torch.zeros_like(logits).scatter(1, ids, w * (g - mean))
        else:
            d = p * (torch.zeros_like(logits).scatter(1, ids, g) - mean)
        out["grad_logits"] = d.to(TYPES[c["dtype"]])
    return out


def _activate(v, name):
    return v * torch.sigmoid(v) if name == "silu" else 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _plain_layer(s, c):
    T, k, H, I = c["tokens"], c["topk"], c["hidden"], c["inter"]
    x, e = s["x"].float(), s["ids"].long() - c["first"]
    mine = (e >= 0) & (e < c["local"])
    e, w = torch.where(mine, e, torch.zeros_like(e)), torch.where(mine, s["weights"], torch.zeros_like(s["weights"]))
    if T * k <= c["local"]:  # few pairs: each with its own expert's weights
        gu = torch.matmul(s["w_in"][e.reshape(-1)].float(), x.repeat_interleave(k, dim=0)[:, :, None])[:, :, 0]
        h = _activate(gu[:, :I], c["activation"]) * gu[:, I:]
        y = torch.matmul(s["w_out"][e.reshape(-1)].float(), h[:, :, None])[:, :, 0]
        y = (y.view(T, k, H) * w[:, :, None]).sum(dim=1)
    else:  # many: every expert on every token, weighted by what the router gave it
        share = torch.zeros(T, c["local"], device=DEV).scatter_add(1, e, w)
        gu = torch.matmul(s["w_in"].float(), x.t().contiguous())
        h = _activate(gu[:, :I], c["activation"]) * gu[:, I:]
        y = torch.matmul(s["w_out"].float(), h)
        y = (y * share.t()[:, None, :]).sum(dim=0).t()
    return y.to(TYPES[c["dtype"]])


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"embedding": _plain_embedding, "embedding_grad": _plain_grad, "moe_route": _plain_route, "moe_layer": _plain_layer}[c["op"]](s, c)
    mccl = _mccl()
    if c["op"] == "embedding":
        return mccl.embedding(s["table"], s["ids"], scale=c["scale"], first_row=c["first"])
    if c["op"] == "embedding_grad":
        plan = mccl.sort_ids(s["ids"], c["rows"], first_row=c["first"])
        d = mccl.embedding_grad(s["grad"], plan, scale=c["scale"], dtype=TYPES[c["out"]], out=s.get("main"), accumulate=c["accumulate"])
        return {"grad": d, "order": plan[0], "offsets": plan[1]}
    if c["op"] == "moe_route":
        ids, weights = mccl.moe_route(s["logits"], c["topk"], normalize=c["normalize"])
        out = {"ids": ids, "weights": weights}
        if c["train"]:
            out["grad_logits"] = mccl.moe_route_grad(s["grad_weights"], s["logits"], ids, normalize=c["normalize"])
        return out
    return mccl.moe_layer(s["x"], s["w_in"], s["w_out"], s["ids"], s["weights"], first_expert=c["first"], activation=c["activation"])


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def _expected_rows(c):
    """(tokens of the shard, distinct rows of the shard among them), expected over the ids of _ids()."""
    v = torch.arange(c["first"], c["first"] + c["rows"], dtype=torch.float64)
    p = torch.log1p(1.0 / (v + 1.0)) / math.log(c["vocab"] + 1.0) * (1.0 - c.get("hot", 0.0))
    p[c["rows"] // 2] += c.get("hot", 0.0)
    return c["n"] * float(p.sum()), float((1.0 - (1.0 - p) ** c["n"]).sum())


def work(case):
    c, es = case, SIZE[case["dtype"]]
    if c["op"] == "embedding":
        inside, rows = _expected_rows(c)
        return {"bytes": c["n"] * 8 + rows * c["hidden"] * es + c["n"] * c["hidden"] * es, "flops": inside * c["hidden"]}
    if c["op"] == "embedding_grad":
        inside, rows = _expected_rows(c)
        moved = 2 * rows if c["accumulate"] else c["rows"]
        return {"bytes": c["n"] * 16 + 8 * (c["rows"] + 1) + inside * c["hidden"] * es + moved * c["hidden"] * SIZE[c["out"]],
                "flops": inside * c["hidden"]}
    if c["op"] == "moe_route":
        pairs, row = c["tokens"] * c["topk"], c["tokens"] * c["experts"] * es
        return {"bytes": row + 8 * pairs + (row + 4 * pairs if c["train"] else 0), "flops": 4 * c["tokens"] * c["experts"]}
    live = c["tokens"] - c["padded"]
    chosen = c["local"] * (1.0 - (1.0 - c["topk"] / c["experts"]) ** live)
    pairs = live * c["topk"] * c["local"] / c["experts"]
    weights = 3 * c["hidden"] * c["inter"]
    return {"bytes": chosen * weights * es + 2 * c["tokens"] * c["hidden"] * es + 8 * c["tokens"] * c["topk"], "flops": 2 * pairs * weights}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "embedding":
        out = torch.zeros(c["n"], c["hidden"], dtype=torch.float64, device=DEV)
        at = torch.nonzero((s["ids"] >= c["first"]) & (s["ids"] < c["first"] + c["rows"]))[:, 0]
        out[at] = s["table"].double()[s["ids"][at] - c["first"]] * c["scale"]
        return out
    if c["op"] == "embedding_grad":
        out = s["main"].double() if c["accumulate"] else torch.zeros(c["rows"], c["hidden"], dtype=torch.float64, device=DEV)
        at = torch.nonzero((s["ids"] >= c["first"]) & (s["ids"] < c["first"] + c["rows"]))[:, 0]
        out.index_add_(0, s["ids"][at] - c["first"], s["grad"][at].double(), alpha=c["scale"])
        return {"grad": out, "order": None, "offsets": None}
    if c["op"] == "moe_route":
        logits = s["logits"].double()
        # sorted by (value falling, index rising)
        ids = torch.argsort(-logits, dim=1, stable=True)[:, : c["topk"]]
        closed = torch.isinf(logits.gather(1, ids))
        p = torch.softmax(logits, dim=1)
        w = p.gather(1, ids)
        total = w.sum(dim=1, keepdim=True) if c["normalize"] else torch.ones_like(w[:, :1])
        out = {"ids": torch.where(closed, -1, ids).int(), "weights": w / total}
        if c["train"]:
            # through the function itself: the gradient of sum(g * weights) in the logits
            at = logits.clone().requires_grad_(True)
            q = torch.softmax(at, dim=1).gather(1, ids)
            q = q / q.sum(dim=1, keepdim=True) if c["normalize"] else q
            torch.sum(q * s["grad_weights"].double().masked_fill(closed, 0.0)).backward()
            out["grad_logits"] = at.grad
        return out
    out = torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device=DEV)
    I = c["inter"]
    for e in range(c["local"]):
        at = torch.nonzero(s["ids"] == c["first"] + e)
        if not len(at):
            continue
        both = s["x"][at[:, 0]].double() @ s["w_in"][e].double().t()
        gate, up = both[:, :I], both[:, I:]
        gate = gate / (1.0 + torch.exp(-gate)) if c["activation"] == "silu" else gate * 0.5 * torch.erfc(-gate / math.sqrt(2.0))
        y = (gate * up) @ s["w_out"][e].double().t()
        out.index_add_(0, at[:, 0], y * s["weights"][at[:, 0], at[:, 1]].double()[:, None])
    return out

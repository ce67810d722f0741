"""Performance cases of the operators at the two ends of a language model: the lookup of token
embeddings with its gradient, the selection of a beam search over beams and vocabulary, and the
reordering of states that follows it.

  listed()   named cases, each with what it stands for
  draw(rng)  one more case of the same ranges
  prepare / run / exact / work   see each function

`own` false: `run` computes the plain form, elementary torch operations in 32 or 64 bits.
`own` true: `run` calls spiky_amd's operators.

A case is a dict of plain values.  `op` selects the operator:

  embed      embed_tokens of [B, S] tokens of type `token` from a table [V, E] of type `weight` to
             type `out`; `scaled`: by sqrt(E); `padded`: a fifth of the tokens is -1, which has no
             row; `train` (forward + gradient of the table) or forward alone
  select     beam_select of the n best of K beams x V tokens for each of B searches; `masked`: a
             third of the vocabulary is -inf; `first`: only the first beam is alive; `done`: some
             beams have finished; `alpha`: the exponent of the lengths; `strided`: the logits are
             the last positions of a [B, K, 2, V] tensor
  reorder    reorder_states of `layers` tensors [B, K, H, L, D], of which the first `used` of L
             positions are taken along, to n beams
"""
import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


def listed():
    emb = dict(op="embed", weight="float32", out="float32", token="int64", scaled=False, padded=False, train=True)
    sel = dict(op="select", dtype="float32", masked=False, first=False, done=False, alpha=0.0, strided=False)
    reo = dict(op="reorder", dtype="bfloat16")
    return [
        # the byte-level transformer of this repository in training: B 32, S 256, E 256
        dict(emb, name="embed_bytes", B=32, S=256, V=256, E=256),
        # a few sequences, one new token each: latency counts
        dict(emb, name="embed_decode", B=4, S=1, V=50000, E=4096, weight="bfloat16", out="bfloat16", scaled=True,
             train=False),
        # sizes that are multiples of nothing, a padded batch
        dict(emb, name="embed_ragged", B=7, S=1143, V=10007, E=1001, weight="float16", out="float16", token="int32",
             padded=True, scaled=True),
        # a training step over a table in 32 bits whose rows go on in 16
        dict(emb, name="embed_mixed", B=8, S=2048, V=32000, E=2048, out="bfloat16"),
        # a large model's step and vocabulary
        dict(emb, name="embed_large", B=16, S=2048, V=152000, E=4096, weight="bfloat16", out="bfloat16"),
        # a byte-level model's search: latency counts
        dict(sel, name="select_bytes", B=1, K=4, V=256, n=4),
        # one request with a large vocabulary, its first step
        dict(sel, name="select_one", B=1, K=4, V=130000, n=8, dtype="bfloat16", masked=True, first=True),
        # odd sizes, the last positions of a longer block, finished beams and lengths
        dict(sel, name="select_ragged", B=5, K=3, V=50001, n=5, dtype="float16", done=True, alpha=0.7, strided=True),
        # a full batch of a server
        dict(sel, name="select_large", B=64, K=8, V=152000, n=16, dtype="bfloat16", masked=True, done=True, alpha=1.0),
        # the token histories of a few searches: latency counts
        dict(reo, name="reorder_histories", layers=1, B=4, K=4, n=4, H=1, L=512, used=512, D=1, dtype="int64"),
        # odd sizes, the first positions of longer caches
        dict(reo, name="reorder_ragged", layers=6, B=3, K=5, n=5, H=7, L=301, used=155, D=33, dtype="float16"),
        # the keys and values of a few layers at a long context
        dict(reo, name="reorder_large", layers=8, B=8, K=4, n=4, H=8, L=4096, used=3333, D=128),
    ]


# ---------------------------------------------------------------------- draws
def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width of a row: any whole number, or one of the usual multiples of 64."""
    d = _log(rng, lo, hi)
    return d if rng.random() < 0.5 else max(64, d // 64 * 64)


def draw(rng):
    op = rng.choice(["embed", "embed", "select", "select", "reorder"])
    floats = ["float32", "bfloat16", "float16"]
    while True:
        if op == "embed":
            weight = rng.choice(floats)
            c = dict(op=op, B=_log(rng, 1, 64), S=_log(rng, 1, 4096), V=_log(rng, 100, 260000), E=_width(rng, 16, 8192),
                     weight=weight, out=rng.choice(floats if weight == "float32" else [weight, "float32"]),
                     token=rng.choice(["int32", "int64"]), scaled=rng.random() < 0.4, padded=rng.random() < 0.3,
                     train=rng.random() < 0.7)
            if c["B"] * c["S"] <= 1 << 16 and c["B"] * c["S"] * c["E"] <= 1 << 26 and c["V"] * c["E"] <= 1 << 28:
                return c
        elif op == "select":
            K = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
            c = dict(op=op, B=_log(rng, 1, 128), K=K, V=_log(rng, 200, 260000), n=K if rng.random() < 0.4 else 2 * K,
                     dtype=rng.choice(floats), masked=rng.random() < 0.4, first=rng.random() < 0.2,
                     done=rng.random() < 0.4, alpha=rng.choice([0.0, 0.0, 0.7, 1.0]), strided=rng.random() < 0.3)
            c["done"] = c["done"] and not c["first"]
            if c["B"] * K * c["V"] <= 1 << (25 if c["dtype"] == "float32" else 26):
                return c
        else:
            K, L = rng.choice([1, 2, 3, 4, 5, 8, 16]), _log(rng, 1, 8192)
            c = dict(op=op, layers=_log(rng, 1, 40), B=_log(rng, 1, 32), K=K, n=K, H=rng.choice([1, 2, 7, 8, 16]), L=L,
                     used=max(1, int(L * rng.random())) if rng.random() < 0.6 else L, D=rng.choice([1, 33, 64, 128]),
                     dtype=rng.choice(floats + ["int32", "int64", "uint8"]))
            if c["layers"] * c["B"] * K * c["H"] * L * c["D"] <= 1 << 28:
                return c


# --------------------------------------------------------------------- inputs
def _type(name):
    return getattr(torch, name)


def _prepare_embed(c, gen):
    B, S, V, E = c["B"], c["S"], c["V"], c["E"]
    u = torch.rand(B, S, generator=gen, device=DEVICE, dtype=torch.float64)
    # tokens of a text: the frequency of the r-th most frequent goes as 1 / r; they lie anywhere in the table
    rank = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
    step = next(s for s in range(V * 5 // 8 | 1, 2 * V + 3) if math.gcd(s, V) == 1)
    tokens = rank * step % V
    if c["padded"]:
        tokens.masked_fill_(torch.rand(B, S, generator=gen, device=DEVICE) < 0.2, -1)
    w = torch.randn(V, E, generator=gen, device=DEVICE).mul_(0.05).to(_type(c["weight"]))
    s = {"tokens": tokens.to(_type(c["token"])), "weight": w, "scale": math.sqrt(E) if c["scaled"] else 1.0}
    if c["train"]:
        s["weight"].requires_grad_()
        s["dy"] = torch.randn(B, S, E, generator=gen, device=DEVICE).to(_type(c["out"]))
    return s


def _prepare_select(c, gen):
    B, K, V = c["B"], c["K"], c["V"]

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    x = torch.randn(B, K, 2 if c["strided"] else 1, V, generator=gen, device=DEVICE).mul_(4.0)[:, :, -1:]
    if c["masked"]:
        x.masked_fill_(uniform(V) < 0.33, -math.inf)
    if c["strided"]:
        whole = torch.zeros(B, K, 2, V, dtype=_type(c["dtype"]), device=DEVICE)
        whole[:, :, -1:] = x.to(whole.dtype)
        x = whole[:, :, -1:]
    s = {"logits": x.to(_type(c["dtype"]))[:, :, 0]}
    # the sums of the logarithms of some tokens' probabilities, beams close to each other
    s["scores"] = -20.0 * uniform(B, 1) - 3.0 * uniform(B, K)
    if c["first"]:
        s["scores"] = torch.full((B, K), -math.inf, device=DEVICE)
        s["scores"][:, 0] = 0.0
    s["finished"] = uniform(B, K) < 0.3 if c["done"] else None
    s["lengths"] = (1 + 40 * uniform(B, K)).to(torch.int64) if c["alpha"] else None
    return s


def _prepare_reorder(c, gen):
    shape = (c["B"], c["K"], c["H"], c["L"], c["D"])
    t, s = _type(c["dtype"]), {"states": []}
    for _ in range(c["layers"]):
        if t.is_floating_point:
            x = torch.randn(*shape, generator=gen, device=DEVICE, dtype=t)
        else:
            x = torch.randint(0, 256, shape, generator=gen, device=DEVICE).to(t)
        s["states"].append(x[:, :, :, :c["used"]])
    # a selection keeps a few of the beams, in the order of their scores
    u = torch.rand(c["B"], c["n"], generator=gen, device=DEVICE)
    s["parents"] = (c["K"] * u.square()).long().clamp_(max=c["K"] - 1)
    return s


def prepare(case, seed):
    """The tensors in a program's hands before the call, from the seed alone."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    s = {"embed": _prepare_embed, "select": _prepare_select, "reorder": _prepare_reorder}[case["op"]](case, gen)
    s["case"] = case
    return s


# ---------------------------------------------------------------- plain forms
def _plain_embed(s):
    c = s["case"]
    w, V = s["weight"].detach(), c["V"]
    tokens = s["tokens"].reshape(-1).long()
    there = (tokens >= 0) & (tokens < V)
    at = torch.where(there, tokens, 0)
    y = torch.where(there[:, None], w[at].float() * s["scale"], 0.0)
    out = {"y": y.reshape(c["B"], c["S"], c["E"]).to(_type(c["out"]))}
    if c["train"]:
        dy = torch.where(there[:, None], s["dy"].reshape(-1, c["E"]).float(), 0.0)
        dw = torch.zeros(V, c["E"], device=DEVICE).index_add_(0, at, dy)
        out["dweight"] = (dw * s["scale"]).to(w.dtype)
    return out


def _plain_select(s):
    c = s["case"]
    B, K, V, n = c["B"], c["K"], c["V"], c["n"]
    # in 64 bits: which of two beams goes on hangs on the difference of their sums
    x, score = s["logits"].double(), s["scores"].double()
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))) + score[:, :, None]
    grown = torch.ones(B, K, device=x.device)
    if s["finished"] is not None:
        only = torch.full((B, K, V), -math.inf, dtype=x.dtype, device=x.device)
        only[:, :, 0] = score
        x = torch.where(s["finished"][:, :, None], only, x)
        grown = grown - s["finished"].float()
    rank = x
    if s["lengths"] is not None:
        rank = x / ((s["lengths"] + grown).clamp_min(1.0).double() ** c["alpha"])[:, :, None]
    x, rank = x.reshape(B, K * V), rank.reshape(B, K * V).clone()
    at = []
    for _ in range(n):  # argmax takes the first of equal ones
        at.append(rank.argmax(-1, keepdim=True))
        rank.scatter_(1, at[-1], -math.inf)
    at = torch.cat(at, 1)
    score = x.gather(1, at)
    gone = score == -math.inf  # fewer candidates than n: no parent, no token
    return {"scores": score.float(), "parents": torch.where(gone, 0, at // V), "tokens": torch.where(gone, 0, at % V)}


def _plain_reorder(s):
    row = torch.arange(s["case"]["B"], device=s["parents"].device)[:, None]
    return [x[row, s["parents"]] for x in s["states"]]


# ------------------------------------------------------------ the framework's
def _own_embed(s):
    from spiky_amd import embed_tokens
    c = s["case"]
    if not c["train"]:
        return {"y": embed_tokens(s["tokens"], s["weight"], s["scale"], dtype=_type(c["out"]))}
    with torch.autograd.set_multithreading_enabled(False):
        y = embed_tokens(s["tokens"], s["weight"], s["scale"], dtype=_type(c["out"]))
        return {"y": y.detach(), "dweight": torch.autograd.grad(y, s["weight"], s["dy"])[0]}


def _own_select(s):
    from spiky_amd import beam_select
    c = s["case"]
    scores, parents, tokens = beam_select(s["logits"], s["scores"], c["n"], finished=s["finished"], pad=0,
                                          lengths=s["lengths"], length_penalty=c["alpha"])
    return {"scores": scores, "parents": parents, "tokens": tokens}


def _own_reorder(s):
    from spiky_amd import reorder_states
    return reorder_states(s["states"], s["parents"])


def run(state):
    """One pass: a training step's forward and gradient, a lookup, a selection or a reordering."""
    op = state["case"]["op"]
    if own:
        return {"embed": _own_embed, "select": _own_select, "reorder": _own_reorder}[op](state)
    return {"embed": _plain_embed, "select": _plain_select, "reorder": _plain_reorder}[op](state)


# ---------------------------------------------------------------- definitions
def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits; gradients by differentiation."""
    c, s = case, prepare(case, seed)
    if c["op"] == "embed":
        w = s["weight"].detach().double().requires_grad_(c["train"])
        kept = (s["tokens"] >= 0) & (s["tokens"] < c["V"])
        y = torch.zeros(c["B"], c["S"], c["E"], dtype=torch.float64, device=DEVICE)
        y = y.index_put(kept.nonzero(as_tuple=True), w.index_select(0, s["tokens"][kept].long()) * s["scale"])
        out = {"y": y.detach()}
        if c["train"]:
            out["dweight"] = torch.autograd.grad(y, w, s["dy"].double())[0]
        return out
    if c["op"] == "select":
        found = {"scores": [], "parents": [], "tokens": []}
        for b in range(c["B"]):
            rows = []
            for k in range(c["K"]):
                before = s["scores"][b, k].double()
                if s["finished"] is not None and bool(s["finished"][b, k]):
                    v, x, more = torch.zeros(1, dtype=torch.int64, device=DEVICE), before[None], 0
                else:
                    x = torch.log_softmax(s["logits"][b, k].double(), 0) + before
                    v = torch.sort(x, descending=True, stable=True)[1][:c["n"]]
                    x, more = x[v], 1
                length = max(1, int(s["lengths"][b, k]) + more) if s["lengths"] is not None else 1
                rows += [(-r, k, t, e) for r, t, e in zip((x / float(length) ** c["alpha"]).tolist(), v.tolist(), x.tolist())
                         if e > -math.inf]
            rows = sorted(rows)[:c["n"]]
            rows += [(0.0, 0, 0, -math.inf)] * (c["n"] - len(rows))
            found["scores"].append([r[3] for r in rows])
            found["parents"].append([r[1] for r in rows])
            found["tokens"].append([r[2] for r in rows])
        return {k: torch.tensor(v, dtype=torch.float64 if k == "scores" else torch.int64, device=DEVICE)
                for k, v in found.items()}
    return [torch.stack([torch.stack([x[b, p] for p in chosen]) for b, chosen in enumerate(s["parents"].tolist())])
            for x in s["states"]]


# ----------------------------------------------------------------------- work
def _distinct(total, n):
    """How many of `total` tokens n tokens of a text hold: their r-th most frequent has probability about 1 / r."""
    weight = 1.0 / math.log(total + 1.0)
    found, r = 0.0, 1.0
    while r <= total:  # ranks r to 1.1 r alike
        up = min(max(r + 1.0, 1.1 * r), total + 1.0)
        found += (up - r) * -math.expm1(-n * weight / r)
        r = up
    return found


def work(case):
    """Bytes read once and written once, and the arithmetic, of one pass."""
    c = case
    size = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "int64": 8, "uint8": 1}
    if c["op"] == "embed":
        tokens = c["B"] * c["S"]
        n = int(tokens * c["E"] * (0.8 if c["padded"] else 1.0))
        rows = int(_distinct(c["V"], tokens * (0.8 if c["padded"] else 1.0)))
        total = tokens * size[c["token"]] + rows * c["E"] * size[c["weight"]] + tokens * c["E"] * size[c["out"]]
        if c["train"]:  # the tokens again, the output's gradient, the whole table's
            total += tokens * size[c["token"]] + n * size[c["out"]] + c["V"] * c["E"] * size[c["weight"]]
        return {"bytes": total, "flops": n * (2 if c["train"] else 1)}
    if c["op"] == "select":
        # a beam that is not alive, or has finished, has nothing to read
        rows = c["B"] * (1 if c["first"] else c["K"]) * (0.7 if c["done"] else 1.0)
        n = int(rows * c["V"])
        return {"bytes": n * size[c["dtype"]] + 20 * c["B"] * c["n"] + 13 * c["B"] * c["K"], "flops": 4 * n}
    each = c["layers"] * c["H"] * c["used"] * c["D"] * size[c["dtype"]]
    # of K beams, the expected number that a selection keeps
    kept = sum(1.0 - (1.0 - (math.sqrt((k + 1) / c["K"]) - math.sqrt(k / c["K"]))) ** c["n"] for k in range(c["K"]))
    return {"bytes": int(each * c["B"] * (kept + c["n"])) + 8 * c["B"] * c["n"], "flops": 1}

"""Performance cases of the operators around the LUT blocks of a language model: dropout, the
residual join of a block with its norms, and the processing of logits before a token is chosen.

  listed()   named cases, each with what it stands for
  draw(rng)  one more case of the same ranges
  prepare / run / exact / work   see each function

`own` false: `run` computes the plain form, elementary torch operations in 32 bits.
`own` true: `run` calls spiky_amd's operators.

A case is a dict of plain values.  `op` selects the operator:

  dropout    counter_dropout, forward and backward: [rows, D], type, p
  residual   residual_norm over [B, S, D]: `act` the type of the branch and of the normed output,
             `res` of the residual stream, `par` of the norms' parameters; `post` and `pre` norm
             (none, rms, layer); `gate` (none, channel, sample, full); `biases`; p; scales;
             `train` (forward + backward) or evaluation
  logits     process_logits over [B, V]: `dtype` in and `out` type; a history of at most L tokens
             a row; dense bias (none, shared, row), K sparse biases a row, mask (none, bits, bool),
             `per_row` penalties and temperatures or one number; `strided`: the rows are the last
             positions of a [B, 2, V] tensor
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


def listed():
    res = dict(op="residual", res="float32", act="float32", par="float32", post="rms", pre="rms", gate="none",
               biases=False, p=0.0, alpha=1.0, beta=1.0, train=True)
    log = dict(op="logits", dtype="float32", out="float32", bias="none", K=0, mask="none", per_row=False, strided=False,
               token="int64")
    return [
        # the block output of a byte-level transformer, one sequence: launches count
        dict(op="dropout", name="dropout_small", rows=256, D=256, dtype="float32", p=0.1),
        # sizes that are multiples of nothing
        dict(op="dropout", name="dropout_ragged", rows=1777, D=1237, dtype="float16", p=0.25),
        # the widened activations of a large model's step
        dict(op="dropout", name="dropout_large", rows=16384, D=8192, dtype="bfloat16", p=0.1),
        # a few sequences, one new token each: latency counts
        dict(res, name="residual_decode", B=4, S=1, D=4096, res="bfloat16", act="bfloat16", par="bfloat16", train=False),
        # the byte-level transformer of this repository in training: B 32, S 256, E 256
        dict(res, name="residual_lut_train", B=32, S=256, D=256, post="layer", pre="layer", gate="channel", biases=True,
             p=0.1),
        # odd sizes, fp16 branch beside an fp32 residual, a gate for each sample
        dict(res, name="residual_ragged_train", B=7, S=143, D=1001, act="float16", gate="sample", p=0.2, alpha=0.9,
             beta=0.5),
        # a long prompt through one block of a large model
        dict(res, name="residual_prefill", B=1, S=16384, D=8192, res="bfloat16", act="bfloat16", par="bfloat16",
             train=False),
        # a training step of a large model with a gate for each sample and dropout
        dict(res, name="residual_large_train", B=8, S=2048, D=4096, act="bfloat16", gate="sample", p=0.1),
        # a byte-level model's next byte: latency counts
        dict(log, name="logits_bytes", B=4, V=256, L=256),
        # one request with a large vocabulary and a long history
        dict(log, name="logits_one", B=1, V=130000, L=8000, dtype="bfloat16", mask="bits", K=64, token="int32"),
        # odd sizes, the last positions of a longer block, everything set for each row
        dict(log, name="logits_ragged", B=33, V=50001, L=1000, dtype="float16", out="float16", bias="row", K=37,
             mask="bool", per_row=True, strided=True),
        # a full batch of a server
        dict(log, name="logits_large", B=512, V=152000, L=4096, dtype="bfloat16", bias="shared", K=64, mask="bits",
             per_row=True, token="int32"),
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
    op = rng.choice(["dropout", "residual", "residual", "logits"])
    while True:
        if op == "dropout":
            c = dict(op=op, rows=_log(rng, 1, 65536), D=_width(rng, 1, 16384),
                     dtype=rng.choice(["float32", "bfloat16", "float16"]), p=rng.choice([0.05, 0.1, 0.25, 0.5]))
            if c["rows"] * c["D"] <= 1 << (26 if c["dtype"] == "float32" else 27):
                return c
        elif op == "residual":
            act = rng.choice(["float32", "bfloat16", "float16"])
            c = dict(op=op, B=_log(rng, 1, 64), S=_log(rng, 1, 16384), D=_width(rng, 16, 16384), act=act,
                     res=rng.choice([act, "float32"]), par=rng.choice([act, "float32"]),
                     post=rng.choice(["none", "rms", "rms", "layer"]), pre=rng.choice(["none", "rms", "rms", "layer"]),
                     gate=rng.choice(["none", "channel", "sample", "full"]), biases=rng.random() < 0.3,
                     p=rng.choice([0.0, 0.1, 0.3]), alpha=rng.choice([1.0, 0.8]), beta=rng.choice([1.0, 0.5]),
                     train=rng.random() < 0.6)
            if not c["train"]:
                c["p"] = 0.0
            if c["B"] * c["S"] * c["D"] <= 1 << 25:
                return c
        else:
            dtype = rng.choice(["float32", "bfloat16", "float16"])
            c = dict(op=op, B=_log(rng, 1, 512), V=_log(rng, 200, 260000), L=_log(rng, 1, 32768), dtype=dtype,
                     out=rng.choice([dtype, "float32"]), bias=rng.choice(["none", "shared", "row"]),
                     K=rng.choice([0, 1, 37, 300]), mask=rng.choice(["none", "bits", "bool"]),
                     per_row=rng.random() < 0.5, strided=rng.random() < 0.3, token=rng.choice(["int32", "int64"]))
            if c["B"] * c["V"] <= 1 << 25 and c["B"] * c["L"] <= 1 << 22:
                return c


# --------------------------------------------------------------------- inputs
def _type(name):
    return getattr(torch, name)


def _prepare_dropout(c, gen):
    x = torch.randn(c["rows"], c["D"], generator=gen, device=DEVICE).to(_type(c["dtype"]))
    dy = torch.randn(c["rows"], c["D"], generator=gen, device=DEVICE).to(_type(c["dtype"]))
    return {"x": x.requires_grad_(), "dy": dy}


def _prepare_residual(c, gen):
    B, S, D = c["B"], c["S"], c["D"]
    act, res, par = _type(c["act"]), _type(c["res"]), _type(c["par"])

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    s = {"z": normal(B, S, D).mul_(2.0), "a": normal(B, S, D), "w1": None, "b1": None, "g": None, "w2": None, "b2": None}
    s["z"][..., : max(1, D // 100)].mul_(20.0)  # a residual stream has a few channels far above the others
    s["z"], s["a"] = s["z"].to(res), s["a"].to(act)
    for norm, w, b in ((c["post"], "w1", "b1"), (c["pre"], "w2", "b2")):
        if norm != "none":
            s[w] = normal(D).mul_(0.1).add_(1.0).to(par)
            s[b] = normal(D).mul_(0.1).to(par) if c["biases"] else None
    if c["gate"] == "channel":
        s["g"] = normal(D).mul_(0.05).add_(0.2).to(par)
    elif c["gate"] == "sample":
        s["g"] = normal(B, 1, D).to(act)
    elif c["gate"] == "full":
        s["g"] = normal(B, S, D).to(act)
    if c["train"]:
        for k in ("z", "a", "w1", "b1", "g", "w2", "b2"):
            if s[k] is not None:
                s[k].requires_grad_()
        s["dz"] = normal(B, S, D).to(res)
        s["dh"] = normal(B, S, D).to(act) if c["pre"] != "none" else None
    return s


def _prepare_logits(c, gen):
    B, V, L = c["B"], c["V"], c["L"]

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    x = torch.randn(B, 2, V, generator=gen, device=DEVICE) if c["strided"] else torch.randn(B, V, generator=gen, device=DEVICE)
    x = x.mul_(4.0).to(_type(c["dtype"]))
    s = {"logits": x[:, -1] if c["strided"] else x, "bias": None, "ids": None, "values": None, "mask": None}
    # tokens of a text: a few are frequent, most are rare
    s["tokens"] = (V * uniform(B, L).pow_(4.0)).to(_type(c["token"])).clamp_(max=V - 1)
    s["lengths"] = (uniform(B).mul_(0.5).add_(0.5) * L).to(torch.int32).clamp_(min=0, max=L)
    s["prompts"] = (s["lengths"] * uniform(B)).to(torch.int32)
    if c["bias"] != "none":
        s["bias"] = torch.randn(*((V,) if c["bias"] == "shared" else (B, V)), generator=gen, device=DEVICE)
    if c["K"]:
        s["ids"] = (V * uniform(B, c["K"])).to(_type(c["token"])).clamp_(max=V - 1)
        s["values"] = torch.randn(B, c["K"], generator=gen, device=DEVICE).mul_(5.0)
    if c["mask"] == "bool":
        s["mask"] = uniform(B, V) < 0.3
    elif c["mask"] == "bits":
        s["mask"] = torch.randint(-(1 << 31), 1 << 31, (B, (V + 31) // 32), generator=gen, device=DEVICE).to(torch.int32)
    if c["per_row"]:
        s["rho"], s["phi"], s["pi"] = uniform(B).mul_(0.5).add_(1.0), uniform(B).mul_(0.2), uniform(B).mul_(0.5)
        s["temperature"] = uniform(B).add_(0.3)
    else:
        s["rho"], s["phi"], s["pi"], s["temperature"] = 1.2, 0.1, 0.4, 0.7
    return s


def prepare(case, seed):
    """The tensors in a program's hands before the call, from the seed alone."""
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    s = {"dropout": _prepare_dropout, "residual": _prepare_residual, "logits": _prepare_logits}[case["op"]](case, gen)
    s["case"], s["seed"], s["offset"] = case, 0x9E3779B97F4A7C15 ^ seed, 3 + seed
    return s


# ---------------------------------------------------------------- plain forms
def _kept(rows, D, p, seed, offset):
    """True where an element is kept: Philox4x32-7 over (column / 4, row, offset), word column % 4."""
    low = 0xFFFFFFFF
    r = torch.arange(rows, device=DEVICE)[:, None]
    c0 = torch.arange((D + 3) // 4, device=DEVICE)[None, :] + 0 * r
    c1, c2, c3 = r + 0 * c0, torch.full_like(c0, offset & low), torch.full_like(c0, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(7):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], -1).reshape(rows, -1)[:, :D]
    return words >= math.floor(p * 4294967296.0 + 0.5)


def _dropped(x, kept, p):
    return torch.where(kept, x.float() * (1.0 / (1.0 - p)), 0.0)


def _plain_dropout(s):
    c = s["case"]
    kept = _kept(c["rows"], c["D"], c["p"], s["seed"], s["offset"])
    return {"y": _dropped(s["x"].detach(), kept, c["p"]).to(s["x"].dtype),
            "dx": _dropped(s["dy"], kept, c["p"]).to(s["x"].dtype)}


def _norm(x, kind, eps=1e-5):
    """The normalised rows and the reciprocal of what they were divided by."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return x * r, r


def _norm_backward(dn, n, r, kind):
    if kind == "layer":
        dn = dn - dn.mean(-1, keepdim=True)
    return r * (dn - n * (dn * n).mean(-1, keepdim=True))


def _plain_residual(s):
    c = s["case"]
    t = {k: v.detach().float() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    z, a, w1, b1, g, w2, b2 = (t[k] for k in ("z", "a", "w1", "b1", "g", "w2", "b2"))
    rows, D = c["B"] * c["S"], c["D"]
    n1, r1 = _norm(a, c["post"]) if c["post"] != "none" else (a, None)
    v = n1 if w1 is None else n1 * w1
    v = v if b1 is None else v + b1
    kept = _kept(rows, D, c["p"], s["seed"], s["offset"]).reshape(a.shape) if c["p"] else None
    d = v if kept is None else _dropped(v, kept, c["p"])
    y = c["alpha"] * z + c["beta"] * (d if g is None else g * d)
    out = {"z": y.to(s["z"].dtype)}
    if c["pre"] != "none":
        n2, r2 = _norm(y, c["pre"])
        h = n2 * w2
        out["h"] = (h if b2 is None else h + b2).to(s["a"].dtype)
    if not c["train"]:
        return out
    q = t["dz"]
    if c["pre"] != "none":
        q = q + _norm_backward(t["dh"] * w2, n2, r2, c["pre"])
        out["dw2"] = (t["dh"] * n2).sum((0, 1)).to(s["w2"].dtype)
        if b2 is not None:
            out["db2"] = t["dh"].sum((0, 1)).to(s["b2"].dtype)
    out["dz"] = (c["alpha"] * q).to(s["z"].dtype)
    q = c["beta"] * q
    if g is not None:
        dg = d * q
        dg = dg.sum((0, 1)) if c["gate"] == "channel" else dg.sum(1, keepdim=True) if c["gate"] == "sample" else dg
        out["dg"] = dg.to(s["g"].dtype)
        q = g * q
    if kept is not None:
        q = _dropped(q, kept, c["p"])
    if w1 is not None:
        out["dw1"] = (q * n1).sum((0, 1)).to(s["w1"].dtype)
    if b1 is not None:
        out["db1"] = q.sum((0, 1)).to(s["b1"].dtype)
    if c["post"] != "none":
        q = _norm_backward(q * w1, n1, r1, c["post"])
    out["da"] = q.to(s["a"].dtype)
    return out


def _rowwise(v):
    return v[:, None] if isinstance(v, torch.Tensor) else v


def _plain_logits(s):
    c = s["case"]
    B, V, L = c["B"], c["V"], c["L"]
    x = s["logits"].float()
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["ids"] is not None:
        x = x.scatter_add(1, s["ids"].long(), s["values"])
    at = torch.arange(L, device=x.device)[None, :]
    said = at < s["lengths"][:, None]
    answered = said & (at >= s["prompts"][:, None])
    tokens = s["tokens"].long()
    seen = torch.zeros(B, V, dtype=torch.int32, device=x.device).scatter_add_(1, tokens, said.int())
    count = torch.zeros(B, V, dtype=torch.int32, device=x.device).scatter_add_(1, tokens, answered.int())
    rho = _rowwise(s["rho"])
    x = torch.where(seen > 0, torch.where(x > 0, x / rho, x * rho), x)
    x = x - (_rowwise(s["phi"]) * count + _rowwise(s["pi"]) * (count > 0))
    x = x / _rowwise(s["temperature"])
    if c["mask"] == "bool":
        x = x.masked_fill(~s["mask"], -math.inf)
    elif c["mask"] == "bits":
        v = torch.arange(V, device=x.device)
        x = x.masked_fill((s["mask"][:, v // 32] >> (v % 32) & 1) == 0, -math.inf)
    return x.to(_type(c["out"]))


# ------------------------------------------------------------ the framework's
def _own_dropout(s):
    from spiky_amd import counter_dropout
    c = s["case"]
    with torch.autograd.set_multithreading_enabled(False):
        y = counter_dropout(s["x"], c["p"], s["seed"], s["offset"])
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def _own_residual(s):
    from spiky_amd import residual_norm
    c = s["case"]
    how = dict(post_norm=None if c["post"] == "none" else c["post"], post_weight=s["w1"], post_bias=s["b1"],
               gate=s["g"], residual_scale=c["alpha"], branch_scale=c["beta"], dropout_p=c["p"], seed=s["seed"],
               offset=s["offset"], pre_norm=None if c["pre"] == "none" else c["pre"], pre_weight=s["w2"],
               pre_bias=s["b2"])
    if not c["train"]:
        z, h = residual_norm(s["z"], s["a"], **how)
        return {"z": z} if h is None else {"z": z, "h": h}
    with torch.autograd.set_multithreading_enabled(False):
        z, h = residual_norm(s["z"], s["a"], **how)
        names = [k for k in ("z", "a", "w1", "b1", "g", "w2", "b2") if s[k] is not None]
        outs, grads = ([z], [s["dz"]]) if h is None else ([z, h], [s["dz"], s["dh"]])
        out = {"d" + k: v for k, v in zip(names, torch.autograd.grad(outs, [s[k] for k in names], grads))}
    out["z"] = z.detach()
    if h is not None:
        out["h"] = h.detach()
    return out


def _own_logits(s):
    from spiky_amd import process_logits
    return process_logits(s["logits"], tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompts"],
                          repetition_penalty=s["rho"], frequency_penalty=s["phi"], presence_penalty=s["pi"],
                          bias=s["bias"], bias_ids=s["ids"], bias_values=s["values"], temperature=s["temperature"],
                          mask=s["mask"], dtype=_type(s["case"]["out"]))


def run(state):
    """One pass: a training step's forward and backward, or an evaluation."""
    op = state["case"]["op"]
    if own:
        return {"dropout": _own_dropout, "residual": _own_residual, "logits": _own_logits}[op](state)
    return {"dropout": _plain_dropout, "residual": _plain_residual, "logits": _plain_logits}[op](state)


# ---------------------------------------------------------------- definitions
def _exact_keep(rows, D, p, seed, offset):
    """The same mask from whole numbers of 64 bits on the host, a block of rows at a time."""
    groups, mask = -(-D // 4), np.uint64(0xFFFFFFFF)
    threshold = np.uint64(math.floor(p * 2.0 ** 32 + 0.5))
    keep = np.empty((rows, groups, 4), dtype=bool)
    step = max(1, (1 << 20) // groups)
    for r0 in range(0, rows, step):
        n = min(step, rows - r0)
        a = np.broadcast_to(np.arange(groups, dtype=np.uint64), (n, groups))
        b = np.broadcast_to(np.arange(r0, r0 + n, dtype=np.uint64)[:, None], (n, groups))
        c = np.full((n, groups), offset & 0xFFFFFFFF, dtype=np.uint64)
        d = np.full((n, groups), offset >> 32 & 0xFFFFFFFF, dtype=np.uint64)
        for i in range(7):
            ka = np.uint64((seed + i * 0x9E3779B9) & 0xFFFFFFFF)
            kb = np.uint64(((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)
            pa, pc = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
            a, b, c, d = (pc >> np.uint64(32)) ^ b ^ ka, pc & mask, (pa >> np.uint64(32)) ^ d ^ kb, pa & mask
        for j, w in enumerate((a, b, c, d)):
            keep[r0:r0 + n, :, j] = w >= threshold
    return torch.from_numpy(keep.reshape(rows, groups * 4)[:, :D].copy()).to(DEVICE)


def _exact_normed(x, kind, w, b):
    centre = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
    y = (x - centre) / torch.sqrt(((x - centre) ** 2).mean(-1, keepdim=True) + 1e-5) * w
    return y if b is None else y + b


def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits; gradients by differentiation."""
    c, s = case, prepare(case, seed)
    if c["op"] == "dropout":
        keep = _exact_keep(c["rows"], c["D"], c["p"], s["seed"], s["offset"])
        y = {}
        for k, name in (("x", "y"), ("dy", "dx")):
            y[name] = torch.zeros(keep.shape, dtype=torch.float64, device=DEVICE)
            y[name][keep] = s[k].detach()[keep].double() / (1.0 - c["p"])
        return y
    if c["op"] == "residual":
        v = {k: t.detach().double().requires_grad_(c["train"]) for k, t in s.items()
             if isinstance(t, torch.Tensor) and k not in ("dz", "dh")}
        u = v["a"]
        if c["post"] != "none":
            u = _exact_normed(u, c["post"], v["w1"], v.get("b1"))
        if c["p"]:
            keep = _exact_keep(c["B"] * c["S"], c["D"], c["p"], s["seed"], s["offset"]).reshape(u.shape)
            u = keep.double() * u / (1.0 - c["p"])
        if "g" in v:
            u = v["g"] * u
        z = c["alpha"] * v["z"] + c["beta"] * u
        out = {"z": z.detach()}
        total = 0.0
        if c["pre"] != "none":
            h = _exact_normed(z, c["pre"], v["w2"], v.get("b2"))
            out["h"] = h.detach()
            if c["train"]:
                total = (h * s["dh"].double()).sum()
        if c["train"]:
            total = total + (z * s["dz"].double()).sum()
            out.update(zip(["d" + k for k in v], torch.autograd.grad(total, list(v.values()))))
        return out
    x = s["logits"].double()
    B, V = x.shape
    host_tokens, lengths, prompts = s["tokens"].cpu().numpy(), s["lengths"].cpu().numpy(), s["prompts"].cpu().numpy()
    rho, phi, pi, heat = (v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(B, v)
                          for v in (s["rho"], s["phi"], s["pi"], s["temperature"]))
    if s["bias"] is not None:
        x = x + s["bias"].double()
    if s["ids"] is not None:
        row = torch.arange(B, device=DEVICE)[:, None].expand_as(s["ids"])
        x = x.index_put((row, s["ids"].long()), s["values"].double(), accumulate=True)
    for b in range(B):
        said = host_tokens[b, :lengths[b]]
        there = torch.from_numpy(np.unique(said).astype(np.int64)).to(DEVICE)
        old = x[b, there]
        x[b, there] = torch.where(old > 0, old / rho[b], old * rho[b])
        new, times = np.unique(host_tokens[b, prompts[b]:lengths[b]], return_counts=True)
        x[b, torch.from_numpy(new.astype(np.int64)).to(DEVICE)] -= torch.from_numpy(phi[b] * times + pi[b]).to(DEVICE)
    x = x / torch.from_numpy(heat).to(DEVICE)[:, None]
    if c["mask"] == "bool":
        x[~s["mask"]] = -math.inf
    elif c["mask"] == "bits":
        bits = np.unpackbits(s["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :V]
        x[torch.from_numpy(bits == 0).to(DEVICE)] = -math.inf
    return x


# ----------------------------------------------------------------------- work
def work(case):
    """Bytes read once and written once, and the arithmetic, of one pass."""
    c = case
    size = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "int64": 8}
    if c["op"] == "dropout":
        n = c["rows"] * c["D"]
        return {"bytes": 4 * n * size[c["dtype"]], "flops": 4 * n}
    if c["op"] == "residual":
        n, D = c["B"] * c["S"] * c["D"], c["D"]
        act, res, par = size[c["act"]], size[c["res"]], size[c["par"]]
        pre, post = c["pre"] != "none", c["post"] != "none"
        gate = {"none": 0, "channel": D * par, "sample": c["B"] * D * act, "full": n * act}[c["gate"]]
        params = (pre + post) * (2 if c["biases"] else 1) * D * par + gate
        total = n * (2 * res + act + pre * act) + params
        flops = n * (4 + 4 * pre + 4 * post)
        if c["train"]:  # the inputs are read again with the outputs' gradients; the gradients are written
            total += n * (3 * res + 2 * act + pre * act) + 2 * params
            flops += n * (6 + 10 * pre + 10 * post)
        return {"bytes": total, "flops": flops}
    n = c["B"] * c["V"]
    bias = {"none": 0, "shared": 4 * c["V"], "row": 4 * n}[c["bias"]]
    mask = {"none": 0, "bits": n // 8, "bool": n}[c["mask"]]
    history = c["B"] * c["L"] * 3 // 4 * size[c["token"]] + c["B"] * c["K"] * (4 + size[c["token"]])
    return {"bytes": n * (size[c["dtype"]] + size[c["out"]]) + bias + mask + history, "flops": 5 * n}

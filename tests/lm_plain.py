"""Plain 64-bit forms of the language-model operators, on the CPU, with the magnitudes that the
tolerances of their tests are counted in."""
import numpy as np
import torch

STEP32 = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def philox7(c0, c1, c2, c3, k0, k1):
    """Seven rounds of Philox4x32 on whole numbers (Salmon et al. 2011)."""
    for i in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32) ^ c1 ^ ((k0 + i * 0x9E3779B9) & 0xFFFFFFFF), b & 0xFFFFFFFF, \
            (a >> 32) ^ c3 ^ ((k1 + i * 0xBB67AE85) & 0xFFFFFFFF), a & 0xFFFFFFFF
    return c0, c1, c2, c3


def kept(rows, cols, p, seed, offset, row0=0):
    """Truth values [rows, cols]: the elements dropout keeps."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.broadcast_to(np.arange(-(-cols // 4), dtype=np.uint64), (rows, -(-cols // 4))),
         np.broadcast_to(np.arange(row0, row0 + rows, dtype=np.uint64)[:, None], (rows, -(-cols // 4)))]
    c += [np.full(c[0].shape, offset & 0xFFFFFFFF, np.uint64), np.full(c[0].shape, offset >> 32, np.uint64)]
    for i in range(7):
        k0, k1 = (seed + i * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & low]
    words = np.stack(c, -1).reshape(rows, -1)[:, :cols]
    return torch.from_numpy(words >= np.uint64(int(np.floor(p * 2.0 ** 32 + 0.5))))


def join(t, how, d_out=None, d_normed=None):
    """The residual join of tensors `t` (r, a, w1, b1, g, w2, b2; rows [n, D], g of n rows) in 64
    bits: outputs, gradients, and for each a magnitude that its rounding errors are relative to."""
    v = {k: (None if x is None else x.detach().double().cpu()) for k, x in t.items()}
    r, a, w1, b1, g, w2, b2 = (v[k] for k in ("r", "a", "w1", "b1", "g", "w2", "b2"))
    post, pre, p = how.get("post_norm"), how.get("pre_norm"), how.get("dropout_p", 0.0)
    alpha, beta = how.get("residual_scale", 1.0), how.get("branch_scale", 1.0)
    out, size = {}, {}

    def norm(x, mag, kind, eps=1e-5):
        m = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
        mag = mag + mag.mean(-1, keepdim=True) if kind == "layer" else mag
        s = 1.0 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
        n = (x - m) * s
        # errors of x move the deviation: relative by at most mean(|n| mag s)
        return n, s, mag * s + n.abs() * (1 + (n.abs() * mag * s).mean(-1, keepdim=True))

    z, zs = r, torch.zeros_like(r)
    if a is not None:
        n1, s1, n1s = norm(a, a.abs(), post) if post else (a, None, torch.zeros_like(a))
        d, ds = n1, n1s
        if w1 is not None:
            d, ds = d * w1, ds * w1.abs()
        if b1 is not None:
            d, ds = d + b1, ds + d.abs() + b1.abs()
        keep = torch.ones_like(a)
        if p:
            keep = kept(*a.shape, p, how.get("seed", 0), how.get("offset", 0)).double() / max(1.0 - p, 1e-300)
            d, ds = torch.where(keep > 0, d * keep, 0.0), ds * keep
        gate = torch.ones_like(a) if g is None else g
        z = alpha * r + beta * gate * d
        zs = (alpha * r).abs() + (beta * gate).abs() * (d.abs() + ds)
        out["z"], size["z"] = z, zs
    if pre:
        n2, s2, n2s = norm(z, zs + z.abs(), pre)
        h, hs = n2, n2s
        if w2 is not None:
            h, hs = h * w2, hs * w2.abs()
        if b2 is not None:
            h, hs = h + b2, hs + h.abs() + b2.abs()
        out["h"], size["h"] = h, hs
    if d_out is None and d_normed is None:
        return out, size

    def norm_back(x, xs, n, ns, s, kind):
        m = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
        ms = (x.abs() + xs).mean(-1, keepdim=True) if kind == "layer" else 0.0
        c = (x * n).mean(-1, keepdim=True)
        cs = ((x.abs() + xs) * (n.abs() + ns)).mean(-1, keepdim=True)
        return s * (x - m - n * c), s * (x.abs() + xs + ms + (n.abs() + ns) * cs)

    q = torch.zeros_like(r) if d_out is None else d_out.double().cpu()
    qs = torch.zeros_like(q)
    if pre and d_normed is not None:
        dh = d_normed.double().cpu()
        t2 = dh if w2 is None else dh * w2
        extra, extras = norm_back(t2, t2.abs(), n2, n2s, s2, pre)
        q, qs = q + extra, q.abs() + extras
        if w2 is not None:
            out["w2"], size["w2"] = (dh * n2).sum(0), (dh.abs() * (n2.abs() + n2s)).sum(0)
        if b2 is not None:
            out["b2"], size["b2"] = dh.sum(0), dh.abs().sum(0)
    if a is None:
        return {**out, "r": q}, {**size, "r": qs}
    out["r"], size["r"] = alpha * q, abs(alpha) * (q.abs() + qs)
    if g is not None:
        out["g"], size["g"] = beta * d * q, abs(beta) * (d.abs() + ds) * (q.abs() + qs)
    dv = torch.where(keep > 0, beta * gate * q * keep, 0.0)
    dvs = (beta * gate).abs() * (q.abs() + qs) * keep
    if w1 is not None:
        out["w1"], size["w1"] = (dv * n1).sum(0), (dvs * (n1.abs() + n1s)).sum(0)
    if b1 is not None:
        out["b1"], size["b1"] = dv.sum(0), dvs.sum(0)
    if post:
        dn, dns = (dv, dvs) if w1 is None else (dv * w1, dvs * w1.abs())
        out["a"], size["a"] = norm_back(dn, dns, n1, n1s, s1, post)
    else:
        out["a"], size["a"] = dv, dvs
    return out, size


def logits(x, tokens=None, lengths=None, prompts=None, rho=1.0, presence=0.0, frequency=0.0, bias=None, ids=None,
           values=None, temperature=1.0, mask=None):
    """Processed logits in 64 bits, and the magnitude of their rounding errors.  mask: truth values."""
    x = x.double().cpu().numpy().copy()
    B, V = x.shape

    def each(v):
        return v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(B, float(v))

    rho, presence, frequency, temperature = (each(v) for v in (rho, presence, frequency, temperature))
    size = np.abs(x)
    if bias is not None:
        bias = np.broadcast_to(bias.double().cpu().numpy(), x.shape)
        x, size = x + bias, size + np.abs(bias)
    for b in range(B):
        if ids is not None:
            k = ids.cpu().numpy()[b] if ids.dim() == 2 else ids.cpu().numpy()
            w = values.double().cpu().numpy()
            w = w[b] if values.dim() == 2 else w
            ok = (k >= 0) & (k < V)
            np.add.at(x[b], k[ok], w[ok])
            np.add.at(size[b], k[ok], np.abs(w[ok]) * (1 + np.arange(ok.sum())))
        if tokens is not None:
            L = tokens.shape[1]
            n = L if lengths is None else min(max(int(lengths[b]), 0), L)
            m = 0 if prompts is None else min(max(int(prompts[b]), 0), n)
            said = tokens[b].cpu().numpy()[:n]
            at = np.unique(said[(said >= 0) & (said < V)])
            f = np.where(x[b, at] > 0, 1.0 / rho[b], rho[b])
            # an error of a value at 0 may choose the other factor: both are within the larger
            x[b, at], size[b, at] = x[b, at] * f, size[b, at] * max(rho[b], 1.0 / rho[b])
            new = said[m:]
            at, times = np.unique(new[(new >= 0) & (new < V)], return_counts=True)
            off = frequency[b] * times + presence[b]
            x[b, at], size[b, at] = x[b, at] - off, size[b, at] + abs(frequency[b]) * times + abs(presence[b])
        if temperature[b] > 0:
            x[b], size[b] = x[b] / temperature[b], size[b] / temperature[b]
    if mask is not None:
        x = np.where(np.broadcast_to(mask.cpu().numpy(), x.shape), x, -np.inf)
    return torch.from_numpy(x), torch.from_numpy(size)


def near(got, want, size, steps, name=""):
    """Every value within `steps` half steps of float32 of its magnitude, and half a step of its type."""
    g = got.detach().double().cpu().reshape(want.shape)
    far = (g - want).abs()
    may = steps * STEP32 * (size + want.abs()) + half_step(got.dtype) * want.abs() * (1 + steps * STEP32)
    may = may + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = ~(far <= may) & ~(g == want) & ~(torch.isnan(g) & torch.isnan(want))
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off; worst " \
        f"{float((far / may.clamp_min(1e-300))[bad].max())} times what it may be, first at {bad.nonzero()[0].tolist()}"

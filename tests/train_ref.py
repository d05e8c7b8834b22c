"""The operators of a training step from their definitions, in 64 bits on the
CPU, each value beside its magnitude: the sum of the absolute values of the
terms that make it up."""
import numpy as np
import torch

from layers_ref import philox

BLOCK = 256


# ---------------------------------------------------------------------- AdamW

def adamw_decode(codes, scale, signed):
    """Values of codes [n] under the exponent bytes scale [blocks]."""
    c = codes.long()
    size = c & 127 if signed else c
    least = torch.exp2(scale.double() - 127).repeat_interleave(BLOCK)[:c.numel()]
    x = torch.where(size < 8, size.double() / 8, torch.exp2((size >> 3).double() - 1) * (1 + (size & 7).double() / 8))
    x = torch.where(scale.repeat_interleave(BLOCK)[:c.numel()] == 255, float("nan"), x * least)
    return torch.where(c > 127, -x, x) if signed else x


def adamw_encode(x, low, signed):
    """Codes and exponent bytes of the 32-bit values x (held in 64 bits), with
    the 8-bit random numbers `low`: multiples of a step, by definition."""
    n, top = x.numel(), 15 if signed else 31
    x, low = x.double(), torch.as_tensor(np.asarray(low), dtype=torch.float64)
    codes, scales = torch.zeros(n, dtype=torch.uint8), []
    for at in range(0, n, BLOCK):
        part, r = x[at:at + BLOCK], low[at:at + BLOCK]
        size = part.abs()
        most = float(size.max())
        if not np.isfinite(most):
            scales.append(255)
            code = torch.zeros(part.numel(), dtype=torch.long)
        else:
            binade = -126 if most < 2.0 ** -126 else int(np.floor(np.log2(most)))
            binade += most > 15 / 8 * 2.0 ** binade and most >= 2.0 ** -126  # may be rounded up into the next one
            lowest = max(binade - (top - 1), -126)
            scales.append(lowest + 127)
            _, e = torch.frexp(size)  # size = mantissa in [1/2, 1) times 2^e
            e = torch.where(size < 2.0 ** lowest, lowest, e.long() - 1)
            parts = size * torch.exp2(3 - e.double())
            if bool((size < 2.0 ** lowest).any()):  # added to the smallest normal number in 32 bits
                small = ((size + 2.0 ** lowest).float().double() - 2.0 ** lowest) * 2.0 ** (3 - lowest)
                parts = torch.where(size < 2.0 ** lowest, small, parts)
            eighths = torch.floor(parts + (r + 0.5) / 256).long()
            code = (e - lowest) * 8 + eighths
            if not signed:
                code = torch.where((size > 0) & (code == 0), 1, code)
        if signed:
            code = code + 128 * (part < 0).long()
        codes[at:at + BLOCK] = code.to(torch.uint8)
    return codes, torch.tensor(scales, dtype=torch.uint8)


def adamw_random(n, seed, t, index):
    """The bytes for the first and the second moments of n elements."""
    seed, t = seed & (2 ** 64 - 1), t & (2 ** 64 - 1)
    rows = [[], []]
    for group in range((n + 7) // 8):
        words = philox((group, index, t & 0xFFFFFFFF, t >> 32), (seed & 0xFFFFFFFF, seed >> 32))
        for k in range(2):
            rows[k] += [w >> s & 255 for w in words[2 * k:2 * k + 2] for s in (0, 8, 16, 24)]
    return [r[:n] for r in rows]


def adamw(c, t, lr, betas, eps, weight_decay, factors=None, grad_scale=None, seed=0):
    """Values and magnitudes after step t, a dict for each tensor; moments in
    8 bits as the codes of the 32-bit moments."""
    b1, b2 = betas
    outs = []
    for i, p in enumerate(c["params"]):
        n = p.numel()
        split, first, rest, decay = (factors[i] if factors else None) or (n, 1.0, 1.0, 1.0)
        rate = torch.where(torch.arange(n) < split, first, rest).double() * lr
        g = c["grads"][i].float()
        if grad_scale is not None:
            g = g * torch.tensor(grad_scale)
        m, v = c["m"][i], c["v"][i]
        if c["scales"] is not None:
            m, v = (adamw_decode(x, c["scales"][i][:, k], k == 0) for k, x in enumerate((m, v)))
        w = (c["masters"][i] if c["masters"] else p).double()
        g64, m0, v0 = g.double(), m.double(), v.double()
        m1, v1 = b1 * m0 + (1 - b1) * g64, b2 * v0 + (1 - b2) * g64 * g64
        o = dict(m=m1, v=v1, m_size=(b1 * m0).abs() + ((1 - b1) * g64).abs(), v_size=v1)
        kept = w * (1 - rate * weight_decay * decay)
        root = (v1 / (1 - b2 ** t)).sqrt() + eps
        o["param"] = kept - rate * m1 / (1 - b1 ** t) / root
        o["param_size"] = kept.abs() + rate.abs() * o["m_size"] / (1 - b1 ** t) / root
        if c["scales"] is not None:
            # the moments of 32 bits, product by product
            f = np.float32
            m32 = m.float() * float(f(b1)) + g * float(f(1 - b1))
            v32 = v.float() * float(f(b2)) + (g * float(f(1 - b2))) * g
            low = adamw_random(n, seed, t, i) if n else ([], [])
            o["m_code"], sm = adamw_encode(m32, low[0], True)
            o["v_code"], sv = adamw_encode(v32, low[1], False)
            o["scales"] = torch.stack([sm, sv], 1)
        outs.append(o)
    return outs


# ----------------------------------------------------------------- group norm

def norm(x, groups, w=None, b=None, eps=1e-5, silu=False, lengths=None, grad=None):
    """Values of out and (with grad) dx, dw, db, and what each is made of:
    sizes of the terms that may cancel."""
    f64 = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    x, w, b, grad = f64(x), f64(w), f64(b), f64(grad)
    B, C = x.shape[:2]
    shape = x.shape
    x = x.reshape(B, C, -1)
    L, cg = x.shape[2], C // groups
    w = torch.ones(C, dtype=torch.float64) if w is None else w
    b = torch.zeros(C, dtype=torch.float64) if b is None else b
    v = {"out": torch.zeros(B, C, L, dtype=torch.float64)}
    m = {"out": torch.zeros(B, C, L, dtype=torch.float64)}
    if grad is not None:
        grad = grad.reshape(B, C, -1)
        for d in (v, m):
            d.update(dx=torch.zeros(B, C, L, dtype=torch.float64), dw=torch.zeros(C, dtype=torch.float64),
                     db=torch.zeros(C, dtype=torch.float64))
    for i in range(B):
        n = L if lengths is None else min(max(int(lengths[i]), 0), L)
        if n == 0:
            continue
        for g in range(groups):
            c = slice(g * cg, (g + 1) * cg)
            p = x[i, c, :n]
            mean = p.mean()
            rstd = 1 / ((p - mean).square().mean() + eps).sqrt()
            xhat = (p - mean) * rstd
            wc, bc = w[c, None], b[c, None]
            pre = xhat * wc + bc
            sig = torch.sigmoid(pre)
            act = sig if silu else torch.ones_like(pre)
            slope = sig * (1 + pre * (1 - sig)) if silu else torch.ones_like(pre)
            # x itself is exact, its mean off by a rounding of the values' size: xhat by that times rstd
            off = xhat.abs() + rstd * p.abs().mean()
            v["out"][i, c, :n] = pre * act
            m["out"][i, c, :n] = (off * wc.abs() + bc.abs()) * ((1 + pre.abs()) if silu else 1)
            if grad is None:
                continue
            d = grad[i, c, :n]
            h = d * slope
            hsize = d.abs() * (1.1 + (off * wc.abs() + bc.abs() if silu else 0))  # (the slope is at most 1.1, its own at most 1/2)
            hw, hx = (h * wc).mean(), (h * wc * xhat).mean()
            v["dx"][i, c, :n] = rstd * (h * wc - hw - xhat * hx)
            top = hsize * wc.abs()
            m["dx"][i, c, :n] = rstd * (top + top.mean() + off * (top * off).mean())
            v["dw"][c] += (h * xhat).sum(1)
            m["dw"][c] += (hsize * off).sum(1)
            v["db"][c] += h.sum(1)
            m["db"][c] += hsize.sum(1)
    for d in (v, m):
        for k in ("out", "dx"):
            if k in d:
                d[k] = d[k].view(shape)
    return v, m


# ----------------------------------------------------------- linear attention

def attention(q, k, v, g, scale=None, init=None, lengths=None, grad=None, grad_final=None, chunk=64):
    """One token at a time: values and magnitudes of out, final and (with
    grad) dq, dk, dv, dg (for each token) and dinit."""
    f64 = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    q, k, v, g, init, grad, grad_final = (f64(t) for t in (q, k, v, g, init, grad, grad_final))
    B, H, dv, L = v.shape
    G, dk = q.shape[1:3]
    scale = dk ** -0.5 if scale is None else scale
    if g.dim() == 1:
        g = g[:, None].expand(B, H, L)
    owner = torch.arange(H) // (H // G)
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    vals = {"out": z(B, H, dv, L), "final": z(B, H, dk, dv)}
    mags = {"out": z(B, H, dv, L), "final": z(B, H, dk, dv)}
    if grad is not None:
        for d in (vals, mags):
            d.update(dq=z(B, G, dk, L), dk=z(B, G, dk, L), dv=z(B, H, dv, L), dg=z(B, H, L), dinit=z(B, H, dk, dv))
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        for absolute, d in ((False, vals), (True, mags)):
            f = torch.abs if absolute else (lambda t: t)
            Q, K = f(q[b, owner]), f(k[b, owner])
            V = f(v[b])
            S = f(init[b]) if init is not None else z(H, dk, dv)
            states = [S]
            for t in range(n):
                S = torch.exp(g[b, :, t])[:, None, None] * S + K[:, :, t, None] * V[:, None, :, t]
                states.append(S)
                d["out"][b, :, :, t] = f(torch.tensor(scale, dtype=torch.float64)) * torch.einsum("hk,hkv->hv", Q[:, :, t], S)
            d["final"][b] = S
            if grad is None:
                continue
            s_ = abs(scale) if absolute else scale
            R = f(grad_final[b]) if grad_final is not None else z(H, dk, dv)
            O = f(grad[b])
            for t in reversed(range(n)):
                D = R + s_ * Q[:, :, t, None] * O[:, None, :, t]
                a = torch.exp(g[b, :, t])[:, None, None]
                dq = s_ * torch.einsum("hkv,hv->hk", states[t + 1], O[:, :, t])
                d["dq"][b, :, :, t].index_add_(0, owner, dq)
                d["dk"][b, :, :, t].index_add_(0, owner, torch.einsum("hkv,hv->hk", D, V[:, :, t]))
                d["dv"][b, :, :, t] = torch.einsum("hkv,hk->hv", D, K[:, :, t])
                d["dg"][b, :, t] += (a * states[t] * D).sum((1, 2))
                if absolute:  # pairs on one side of a token of the chunk are added and taken away again
                    c = t // chunk * chunk
                    d["dg"][b, :, c:min(c + chunk, n)] += (Q[:, :, t] * dq).sum(1)[:, None]
                R = a * D
            d["dinit"][b] = R
    return vals, mags

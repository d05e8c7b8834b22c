"""The sequence operators from their definitions, in 64 bits on the CPU, one
token at a time, each value beside its magnitude: the sum of the absolute
values of the terms that make it up.  An implementation that computes a term
with k roundings of 32 bits is off by about k 2^-24 times the magnitude,
whatever cancels in the value."""
import numpy as np
import torch

U32 = 2.0 ** -24  # half a unit in the last place of a 32-bit number, relative


def f64(t):
    return None if t is None else t.detach().cpu().double()


# ------------------------------------------------------------------- dropout

def philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) in whole numbers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def halves(group, seed, offset):
    """The eight 16-bit numbers of elements 8*group .. 8*group+7."""
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    words = philox((group & 0xFFFFFFFF, group >> 32, offset & 0xFFFFFFFF, offset >> 32),
                   (seed & 0xFFFFFFFF, seed >> 32))
    return [h for w in words for h in (w & 0xFFFF, w >> 16)]


def kept_mask(n, p, seed, offset):
    limit = round(p * 65536)
    bits = [h for g in range((n + 7) // 8) for h in halves(g, seed, offset)][:n]
    return torch.tensor([h >= limit for h in bits], dtype=torch.bool)


def keep_scale(p):
    limit = round(p * 65536)
    return 65536 / (65536 - limit) if limit < 65536 else 0.0


# -------------------------------------------------------- causal convolution

def conv(x, w, bias, silu, init=None, lengths=None, grad=None, grad_final=None):
    """Values and magnitudes of out, final and (with grad) dx, dw, db, dinit."""
    x, w, bias, init, grad, grad_final = (f64(t) for t in (x, w, bias, init, grad, grad_final))
    B, D, L = x.shape
    K = w.shape[1]
    counts = [L] * B if lengths is None else [min(max(int(n), 0), L) for n in lengths]
    line = torch.zeros(B, D, K - 1 + L, dtype=torch.float64)
    if init is not None:
        line[..., :K - 1] = init
    live = torch.zeros(B, 1, L, dtype=torch.bool)
    for b, n in enumerate(counts):
        line[b, :, K - 1:K - 1 + n] = x[b, :, :n]
        live[b, :, :n] = True
    pre, mag = torch.zeros(B, D, L, dtype=torch.float64), torch.zeros(B, D, L, dtype=torch.float64)
    for k in range(K):
        pre += w[:, k, None] * line[..., k:k + L]
        mag += (w[:, k, None] * line[..., k:k + L]).abs()
    if bias is not None:
        pre += bias[:, None]
        mag += bias.abs()[:, None]
    sig = 1 / (1 + torch.exp(-pre))
    out = pre * sig if silu else pre
    v = {"out": torch.where(live, out, 0.0),
         "final": torch.stack([line[b, :, n:n + K - 1] for b, n in enumerate(counts)]) if B else line[..., :K - 1]}
    m = {"out": mag, "final": v["final"].abs()}
    if grad is None:
        return v, m
    slope = sig * (1 + pre * (1 - sig)) if silu else torch.ones_like(pre)
    # the slope's own error goes with that of pre: |silu''| <= 1/2
    dpre, dmag = torch.where(live, grad * slope, 0.0), torch.where(live, grad.abs() * (1.1 + 0.5 * mag), 0.0)
    dline, dlmag = torch.zeros_like(line), torch.zeros_like(line)
    dw, dwm = torch.zeros_like(w), torch.zeros_like(w)
    for k in range(K):
        dline[..., k:k + L] += w[:, k, None] * dpre
        dlmag[..., k:k + L] += w[:, k, None].abs() * dmag
        dw[:, k] = (dpre * line[..., k:k + L]).sum((0, 2))
        dwm[:, k] = (dmag * line[..., k:k + L].abs()).sum((0, 2))
    if grad_final is not None:
        for b, n in enumerate(counts):
            dline[b, :, n:n + K - 1] += grad_final[b]
            dlmag[b, :, n:n + K - 1] += grad_final[b].abs()
    v.update(dx=dline[..., K - 1:], dw=dw, db=dpre.sum((0, 2)), dinit=dline[..., :K - 1])
    m.update(dx=dlmag[..., K - 1:], dw=dwm, db=dmag.sum((0, 2)), dinit=dlmag[..., :K - 1])
    return v, m


# ---------------------------------------------------------- state space scan

def scan(u, delta, A, B, C, D=None, z=None, bias=None, softplus=False, init=None, lengths=None, grad=None,
         grad_final=None):
    """Values and magnitudes of out, final and (with grad) the gradients."""
    u, delta, A, B, C, D, z, bias, init, grad, grad_final = (
        f64(t) for t in (u, delta, A, B, C, D, z, bias, init, grad, grad_final))
    nb, ch, L = u.shape
    N, G = A.shape[1], B.shape[1]
    owner = torch.arange(ch) // max(1, ch // G)
    B, C = B[:, owner], C[:, owner]  # [batch, channels, states, length]
    counts = torch.full((nb,), L) if lengths is None else lengths.cpu().long().clamp(0, L)
    live = (torch.arange(L) < counts[:, None])[:, None]  # [batch, 1, length]

    def zero(t):
        return torch.where(live, t, 0.0)

    raw = delta + (bias[:, None] if bias is not None else 0.0)
    # the kernels' softplus is the identity above 20, where it differs by less than 2^-28
    d = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    u, d, raw = zero(u), zero(d), zero(raw)
    B, C = torch.where(live[:, :, None], B, 0.0), torch.where(live[:, :, None], C, 0.0)
    skip = D[:, None] if D is not None else torch.zeros(ch, 1, dtype=torch.float64)
    if z is not None:
        z = zero(z)
        sig = 1 / (1 + torch.exp(-z))
        gate, gslope = z * sig, sig * (1 + z * (1 - sig))
    else:
        gate, gslope = torch.ones_like(u), torch.zeros_like(u)
    # the relative error of a step's d in 32-bit roundings, over 4: raw may cancel
    weight = 1 + (raw.abs() + (delta.abs() if bias is None else delta.abs() + bias.abs()[:, None])) / 4
    weight = zero(weight)
    a = torch.exp(d[:, :, None] * A[..., None])
    h = torch.zeros(nb, ch, N, L + 1, dtype=torch.float64)
    hm = torch.zeros_like(h)
    if init is not None:
        h[..., 0], hm[..., 0] = init, init.abs()
    for t in range(L):
        x = (d * u)[:, :, None, t] * B[..., t]
        h[..., t + 1] = a[..., t] * h[..., t] + x
        # decays: exp of a product off by up to 1 + |d A| weight roundings
        hm[..., t + 1] = a[..., t] * hm[..., t] + x.abs()
    y = (C * h[..., 1:]).sum(2) + skip * u
    ym = (C.abs() * hm[..., 1:]).sum(2) + (skip * u).abs()
    v = {"out": zero(y * gate), "final": h[..., L].clone()}
    m = {"out": ym * gate.abs(), "final": hm[..., L].clone()}
    v["weight"] = weight.max() if weight.numel() else torch.tensor(1.0)
    if grad is None:
        return v, m
    grad = zero(grad)
    dy = grad * gate
    r = torch.zeros(nb, ch, N, dtype=torch.float64) if grad_final is None else grad_final.clone()
    rm = r.abs()
    names = ["du", "dd", "dA", "dB", "dC"]
    v.update({n: torch.zeros_like(t) for n, t in zip(names, (u, u, A, B, C))})
    m.update({n: torch.zeros_like(t) for n, t in zip(names, (u, u, A, B, C))})
    for t in reversed(range(L)):
        dh, dhm = r + dy[:, :, t, None] * C[..., t], rm + (dy[:, :, t, None] * C[..., t]).abs()
        x = (d * u)[:, :, t, None]
        v["dC"][..., t], m["dC"][..., t] = dy[:, :, t, None] * h[..., t + 1], dy[:, :, t, None].abs() * hm[..., t + 1]
        v["dB"][..., t], m["dB"][..., t] = dh * x, dhm * x.abs()
        through, throughm = (dh * B[..., t]).sum(2), (dhm * B[..., t].abs()).sum(2)
        r, rm = a[..., t] * dh, a[..., t] * dhm
        moved, movedm = r * h[..., t], rm * hm[..., t]
        v["du"][..., t] = d[..., t] * through + skip[:, 0] * dy[..., t]
        m["du"][..., t] = d[..., t].abs() * throughm + (skip[:, 0] * dy[..., t]).abs()
        v["dd"][..., t] = u[..., t] * through + (moved * A).sum(2)
        m["dd"][..., t] = u[..., t].abs() * throughm + (movedm * A.abs()).sum(2)
        v["dA"] += (moved * d[..., t, None]).sum(0)
        m["dA"] += (movedm * d[..., t, None].abs()).sum(0)
    for n in ("dB", "dC"):
        for q in (v, m):
            q[n] = q[n].view(nb, G, ch // G, N, L).sum(2) if ch else torch.zeros(nb, G, N, L, dtype=torch.float64)
    m["dd"] = zero(m["dd"])
    if softplus:
        v["dd"] = v["dd"] / (1 + torch.exp(-raw))
    v["dd"] = zero(v["dd"])
    v["dD"], m["dD"] = (dy * u).sum((0, 2)), (dy * u).abs().sum((0, 2))
    v["dbias"], m["dbias"] = v["dd"].sum((0, 2)), m["dd"].sum((0, 2))
    if z is not None:
        v["dz"], m["dz"] = zero(grad * y * gslope), grad.abs() * ym * 1.1
    v["dinit"], m["dinit"] = r, rm
    return v, m


def excess(got, value, mag, units):
    """max of |got - value| over what one rounding to got's type (of a value
    that is itself off by `units` 32-bit roundings of its magnitude) allows;
    at most 1 passes.  The subnormal step of the type counts once."""
    dtype = got.dtype
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (got.shape, value.shape)
    if got.numel() == 0:
        return 0.0
    assert torch.isfinite(got).all() and torch.isfinite(value).all()
    info = torch.finfo(dtype)
    inner = units * U32 * mag
    own = info.eps / 2 if dtype != torch.float32 else U32
    allowed = own * (value.abs() + inner) + inner + info.tiny * info.eps + 1e-37
    return float(((got - value).abs() / allowed).max())


def rand(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=gen, dtype=torch.float64) * scale + shift).to(dtype)


def numpy_seeded(seed):
    return torch.Generator().manual_seed(int(np.uint32(seed)))

"""Cases of the sequence operators: dropout, the short causal convolution and
the state space scan, each forward, backward and (for the last two) for single
tokens.

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once at the end), or with ``own`` set through the package's
entry points.  ``exact`` computes the same from the definitions in 64 bits.

Tensors are [batch, channels, length], as a convolution layer's [N, C, H*W]
map is when its rows are taken one after the other.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # The residual branch of a training step over 16384 tokens of 4096 channels.
        {"name": "dropout_train_bf16", "op": "dropout", "dtype": "bf16", "rows": 16384, "cols": 4096, "p": 0.1,
         "residual": True, "train": True},
        # Dropout behind a 64-channel 32x32 convolution layer at a batch of 128 images.
        {"name": "dropout_map_fp32", "op": "dropout", "dtype": "fp32", "rows": 128 * 64, "cols": 32 * 32, "p": 0.25,
         "residual": False, "train": True},
        # A few rows of an odd width: the launch is what counts.
        {"name": "dropout_small_fp16", "op": "dropout", "dtype": "fp16", "rows": 7, "cols": 1021, "p": 0.5,
         "residual": True, "train": False},
        # A training step of the convolution in front of the scan.
        {"name": "conv_train_bf16", "op": "conv", "dtype": "bf16", "batch": 4, "channels": 4096, "length": 2048,
         "taps": 4, "bias": True, "silu": True, "ragged": False, "carried": False, "train": True},
        # Prompts of several lengths that go on from a kept state, in a padded batch of an odd length.
        {"name": "conv_prompt_ragged_fp16", "op": "conv", "dtype": "fp16", "batch": 8, "channels": 2047,
         "length": 1333, "taps": 4, "bias": True, "silu": True, "ragged": True, "carried": True, "train": False},
        # One token for each of 64 requests, their states among 96 places.
        {"name": "conv_step_bf16", "op": "conv_step", "dtype": "bf16", "batch": 64, "channels": 4096, "taps": 4,
         "bias": True, "silu": True, "places": 96},
        # A training step of the scan, gated, at 8192 tokens.
        {"name": "scan_train_bf16", "op": "scan", "dtype": "bf16", "batch": 4, "channels": 2048, "length": 2048,
         "states": 16, "groups": 1, "gate": True, "ragged": False, "carried": False, "train": True},
        # A training step of the scan over the map of a 64-channel 32x32 convolution layer, 128 images.
        {"name": "scan_map_fp32", "op": "scan", "dtype": "fp32", "batch": 128, "channels": 64, "length": 1024,
         "states": 16, "groups": 1, "gate": False, "ragged": False, "carried": False, "train": True},
        # One long prompt: few rows, a long axis.
        {"name": "scan_prompt_long_bf16", "op": "scan", "dtype": "bf16", "batch": 1, "channels": 2048,
         "length": 16384, "states": 16, "groups": 1, "gate": True, "ragged": False, "carried": False, "train": False},
        # Prompts of several lengths that go on from a kept state; odd sizes, two groups, 24 states.
        {"name": "scan_prompt_ragged_fp16", "op": "scan", "dtype": "fp16", "batch": 7, "channels": 1002,
         "length": 777, "states": 24, "groups": 2, "gate": True, "ragged": True, "carried": True, "train": False},
        # One token for each of 64 requests, their states among 96 places.
        {"name": "scan_step_bf16", "op": "scan_step", "dtype": "bf16", "batch": 64, "channels": 4096, "states": 16,
         "groups": 1, "gate": True, "places": 96},
        # One token of one request of a small model.
        {"name": "scan_step_small_fp32", "op": "scan_step", "dtype": "fp32", "batch": 1, "channels": 768,
         "states": 16, "groups": 1, "gate": True, "places": 1},
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)))


def draw(rng):
    op = rng.choice(["dropout", "conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step"])
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "dropout":
        rows = _spread(rng, 1, 16384)
        return {**case, "rows": rows, "cols": _spread(rng, 1, min(8192, (1 << 25) // rows)),
                "p": round(rng.uniform(0.02, 0.6), 3), "residual": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op == "conv_step":
        batch = _spread(rng, 1, 256)
        return {**case, "batch": batch, "channels": _spread(rng, 64, 4096), "taps": rng.randint(2, 8),
                "bias": rng.random() < 0.7, "silu": rng.random() < 0.7, "places": batch + rng.randint(0, 64)}
    if op == "scan_step":
        batch, groups = _spread(rng, 1, 256), rng.choice([1, 1, 2, 4])
        return {**case, "batch": batch, "channels": groups * _spread(rng, 16, 1024), "states": _spread(rng, 4, 64),
                "groups": groups, "gate": rng.random() < 0.7, "places": batch + rng.randint(0, 64)}
    train = rng.random() < 0.5
    ragged = not train and rng.random() < 0.6
    if op == "conv":
        batch = _spread(rng, 1, 16)
        channels = _spread(rng, 64, 4096)
        return {**case, "batch": batch, "channels": channels,
                "length": _spread(rng, 1, min(16384, (1 << 25) // (batch * channels))), "taps": rng.randint(2, 8),
                "bias": rng.random() < 0.7, "silu": rng.random() < 0.7, "ragged": ragged,
                "carried": rng.random() < 0.5, "train": train}
    batch, groups, states = _spread(rng, 1, 16), rng.choice([1, 1, 2, 4]), _spread(rng, 4, 64)
    channels = groups * _spread(rng, 16, 512)
    return {**case, "batch": batch, "channels": channels,
            "length": _spread(rng, 1, min(8192, (1 << 27) // (batch * channels * states))), "states": states,
            "groups": groups, "gate": rng.random() < 0.7, "ragged": ragged, "carried": rng.random() < 0.5,
            "train": train}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=kind):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)

    def uniform(low, high, *shape):
        return torch.rand(shape, generator=g, device="cuda") * (high - low) + low

    s = {"case": case}
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        s["x"] = normal(*shape)
        s["residual"] = normal(*shape) if case["residual"] else None
        s["grad"] = normal(*shape) if case["train"] else None
        s["key"] = torch.randint(-(1 << 62), 1 << 62, (2,), generator=g, device="cuda")
        wanted = ["x", "residual"]
    else:
        batch, channels = case["batch"], case["channels"]
        step = case["op"].endswith("step")
        length = () if step else (case["length"],)
        if step:  # the requests' places, in no order
            s["slots"] = torch.randperm(case["places"], generator=g, device="cuda")[:batch].to(torch.int32)
        else:
            s["lengths"] = None
            if case["ragged"]:  # padded rows of any length; the first full, one of them empty, one of one token
                s["lengths"] = torch.randint(1, case["length"] + 1, (batch,), generator=g, device="cuda").to(torch.int32)
                s["lengths"][:1] = case["length"]
                s["lengths"][1:3] = torch.arange(2, device="cuda", dtype=torch.int32)[:max(0, min(2, batch - 1))]
        rows = case["places"] if step else batch
        if case["op"].startswith("conv"):
            taps = case["taps"]
            s["x"] = normal(batch, channels, *length)
            s["weight"] = normal(channels, taps, scale=taps ** -0.5)
            s["bias"] = normal(channels, scale=0.1) if case["bias"] else None
            s["state"] = normal(rows, channels, taps - 1) if step or case["carried"] else None
            wanted = ["x", "weight", "bias", "state"]
        else:
            states, groups = case["states"], case["groups"]
            s["u"] = normal(batch, channels, *length)
            s["delta"] = normal(batch, channels, *length, scale=0.5)
            s["z"] = normal(batch, channels, *length) if case["gate"] else None
            s["B"] = normal(batch, groups, states, *length)
            s["C"] = normal(batch, groups, states, *length)
            # decays from 1 to N for each channel, and steps from 0.001 to 0.1, as such layers begin with
            s["A"] = -(torch.arange(1, states + 1, device="cuda") * uniform(0.8, 1.25, channels, states))
            s["skip"] = normal(channels, scale=0.1, shift=1.0, dtype=torch.float32)
            first = torch.exp(uniform(math.log(0.001), math.log(0.1), channels))
            s["delta_bias"] = first + torch.log(-torch.expm1(-first))
            s["state"] = normal(rows, channels, states, dtype=torch.float32) if step or case["carried"] else None
            wanted = ["u", "delta", "A", "B", "C", "skip", "z", "delta_bias", "state"]
        if not step and case["train"]:
            s["grad"] = normal(batch, channels, *length)
            s["grad_state"] = None
            if case["carried"]:
                s["grad_state"] = torch.randn(s["state"].shape, generator=g, device="cuda").to(s["state"].dtype)
    s["wanted"] = []
    if case.get("train"):
        s["wanted"] = [n for n in wanted if s[n] is not None]
        for n in s["wanted"]:
            s[n].requires_grad_(True)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    with torch.no_grad():
        if op == "dropout":
            return _plain_dropout(state)
        if op == "conv":
            return _plain_conv(state)
        if op == "conv_step":
            return _plain_conv_step(state)
        if op == "scan":
            return _plain_scan(state)
        return _plain_scan_step(state)


def _own(s):
    import paraconv2d_b200 as pc

    case = s["case"]
    op = case["op"]
    act = "silu" if case.get("silu") else None
    if op == "conv_step":
        out = pc.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation=act, slots=s["slots"])
        return {"out": out, "state": s["state"]}
    if op == "scan_step":
        out = pc.ssm_scan_step(s["u"], s["delta"], s["state"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"],
                               delta_bias=s["delta_bias"], delta_softplus=True, slots=s["slots"])
        return {"out": out, "state": s["state"]}
    if op == "dropout":
        outs = {"out": pc.dropout(s["x"], case["p"], s["key"], residual=s["residual"])}
        grads = [s["grad"]]
    else:
        keep = case["carried"] or case["ragged"]
        if op == "conv":
            out = pc.causal_conv(s["x"], s["weight"], s["bias"], activation=act, initial_state=s["state"],
                                 lengths=s["lengths"], return_final_state=keep)
        else:
            out = pc.ssm_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"],
                              delta_bias=s["delta_bias"], delta_softplus=True, initial_state=s["state"],
                              lengths=s["lengths"], return_final_state=keep)
        outs = {"out": out[0], "state": out[1]} if keep else {"out": out}
        grads = [s.get("grad"), s.get("grad_state")][:len(outs)]
    if case["train"]:
        got = torch.autograd.grad(list(outs.values()), [s[n] for n in s["wanted"]], grads)
        outs.update({"grad_" + n: v for n, v in zip(s["wanted"], got)})
    return outs


# ------------------------------------------------------------------ dropout

def _bits(n, key):
    """n 16-bit numbers: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011)
    under the key key[0], of the counters (i // 8, key[1]); number i is half
    i % 8 of the four words, the low half first."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 7) // 8, device=key.device)
    x = [block & low, block >> 32, (key[1] & low).expand_as(block), ((key[1] >> 32) & low).expand_as(block)]
    k0, k1 = key[0] & low, (key[0] >> 32) & low
    for _ in range(10):
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [((p1 >> 32) & low) ^ x[1] ^ k0, p1 & low, ((p0 >> 32) & low) ^ x[3] ^ k1, p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack(x, -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:n]


def _plain_dropout(s):
    x, p = s["x"], s["case"]["p"]
    limit = round(p * 65536)
    scale = 65536 / (65536 - limit) if limit < 65536 else 0.0
    kept = (_bits(x.numel(), s["key"]) >= limit).view(x.shape)
    out = torch.where(kept, x.float() * scale, 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    outs = {"out": out.to(x.dtype)}
    if s["case"]["train"]:
        outs["grad_x"] = torch.where(kept, s["grad"].float() * scale, 0.0).to(x.dtype)
        if s["residual"] is not None:
            outs["grad_residual"] = s["grad"].clone()
    return outs


# ---------------------------------------------------------- causal convolution

def _silu_slope(v):
    e = torch.sigmoid(v)
    return e * (1 + v * (1 - e))


def _inside(s, length):
    """True where a row has a token, [batch, 1, length]; None without lengths."""
    if s["lengths"] is None:
        return None
    return (torch.arange(length, device="cuda") < s["lengths"][:, None])[:, None]


def _plain_conv(s):
    case, x = s["case"], s["x"]
    batch, channels, length = x.shape
    taps, inside = case["taps"], _inside(s, length)
    w = s["weight"].float()
    value = x.float()
    if inside is not None:
        value = torch.where(inside, value, 0.0)
    before = value.new_zeros(batch, channels, taps - 1) if s["state"] is None else s["state"].float()
    line = torch.cat([before, value], -1)
    windows = line.unfold(-1, taps, 1)
    pre = (windows * w[:, None]).sum(-1)
    if s["bias"] is not None:
        pre = pre + s["bias"].float()[:, None]
    out = pre * torch.sigmoid(pre) if case["silu"] else pre
    if inside is not None:
        out = torch.where(inside, out, 0.0)
    outs = {"out": out.to(x.dtype)}
    keep = case["carried"] or case["ragged"]
    if keep:
        count = torch.full((batch,), length, device="cuda") if s["lengths"] is None else s["lengths"].long()
        places = (count[:, None] + torch.arange(taps - 1, device="cuda"))[:, None].expand(batch, channels, taps - 1)
        outs["state"] = line.gather(-1, places).to(x.dtype)
    if not case["train"]:
        return outs
    dpre = s["grad"].float()
    if case["silu"]:
        dpre = dpre * _silu_slope(pre)
    if inside is not None:
        dpre = torch.where(inside, dpre, 0.0)
    spread = torch.nn.functional.pad(dpre, (taps - 1, taps - 1)).unfold(-1, taps, 1)
    dline = (spread * w.flip(-1)[:, None]).sum(-1)
    if s["grad_state"] is not None:
        dline = dline.scatter_add(-1, places, s["grad_state"].float())
    outs["grad_x"] = dline[..., taps - 1:].to(x.dtype)
    outs["grad_weight"] = (windows * dpre[..., None]).sum((0, 2), dtype=torch.float64).to(x.dtype)
    if s["bias"] is not None:
        outs["grad_bias"] = dpre.sum((0, 2), dtype=torch.float64).to(x.dtype)
    if s["state"] is not None:
        outs["grad_state"] = dline[..., :taps - 1].to(x.dtype)
    return outs


def _plain_conv_step(s):
    x, state, slots = s["x"], s["state"], s["slots"].long()
    line = torch.cat([state[slots], x[..., None]], -1)
    pre = (line.float() * s["weight"].float()).sum(-1)
    if s["bias"] is not None:
        pre = pre + s["bias"].float()
    out = pre * torch.sigmoid(pre) if s["case"]["silu"] else pre
    state[slots] = line[..., 1:]
    return {"out": out.to(x.dtype), "state": state}


# ----------------------------------------------------------- state space scan

def _running(a, b):
    """h_t = a_t h_(t-1) + b_t along the last axis, from h = 0, by doubling."""
    n = 1
    while n < b.shape[-1]:
        b = torch.cat([b[..., :n], torch.addcmul(b[..., n:], a[..., n:], b[..., :-n])], -1)
        a = torch.cat([a[..., :n], a[..., n:] * a[..., :-n]], -1)
        n *= 2
    return b


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _per_channel(v, channels):
    """[batch, groups, states, ...] -> [batch, channels, states, ...] in 32 bits."""
    return v.float().repeat_interleave(channels // v.shape[1], 1)


def _plain_scan(s):
    case, kind = s["case"], s["u"].dtype
    batch, channels, length = s["u"].shape
    inside = _inside(s, length)

    def masked(v):
        return v if inside is None else torch.where(inside, v, 0.0)

    u = masked(s["u"].float())
    raw = s["delta"].float() + s["delta_bias"][:, None]
    delta = masked(_softplus(raw))
    near = masked(s["B"].float().flatten(1, 2)).view_as(s["B"])  # nothing behind the last token
    far = masked(s["C"].float().flatten(1, 2)).view_as(s["C"])
    A = s["A"][:, :, None]
    B, C = _per_channel(near, channels), _per_channel(far, channels)
    a = torch.exp(delta[:, :, None] * A)
    b = (delta * u)[:, :, None] * B
    if s["state"] is not None:
        b[..., 0] += a[..., 0] * s["state"]
    h = _running(a, b)
    y = (C * h).sum(2) + s["skip"][:, None] * u
    z = None if s["z"] is None else masked(s["z"].float())
    outs = {"out": (y if z is None else y * z * torch.sigmoid(z)).to(kind)}
    if case["carried"] or case["ragged"]:
        outs["state"] = h[..., -1].clone()
    if not case["train"]:
        return outs
    grad = masked(s["grad"].float())
    dy = grad if z is None else grad * z * torch.sigmoid(z)
    db = C * dy[:, :, None]
    if s["grad_state"] is not None:
        db[..., -1] += s["grad_state"]
    after = torch.cat([a[..., 1:], torch.zeros_like(a[..., :1])], -1)
    dh = _running(after.flip(-1), db.flip(-1)).flip(-1)
    first = torch.zeros_like(h[..., :1]) if s["state"] is None else s["state"][..., None]
    moved = dh * a * torch.cat([first, h[..., :-1]], -1)
    through = (dh * B).sum(2)
    ddelta = masked(u * through + (moved * A).sum(2))
    outs["grad_u"] = (delta * through + s["skip"][:, None] * dy).to(kind)
    draw_ = ddelta * torch.sigmoid(raw)
    outs["grad_delta"] = draw_.to(kind)
    outs["grad_A"] = (moved * delta[:, :, None]).sum((0, 3), dtype=torch.float64).float()
    groups = case["groups"]
    shape = (batch, groups, channels // groups, case["states"], length)
    outs["grad_B"] = (dh * (delta * u)[:, :, None]).view(shape).sum(2).to(kind)
    outs["grad_C"] = (h * dy[:, :, None]).view(shape).sum(2).to(kind)
    outs["grad_skip"] = (dy * u).sum((0, 2), dtype=torch.float64).float()
    if z is not None:
        outs["grad_z"] = (grad * y * _silu_slope(z)).to(kind)
    outs["grad_delta_bias"] = draw_.sum((0, 2), dtype=torch.float64).float()
    if s["state"] is not None:
        outs["grad_state"] = dh[..., 0] * a[..., 0]
    return outs


def _plain_scan_step(s):
    channels, slots, state = s["u"].shape[1], s["slots"].long(), s["state"]
    u = s["u"].float()
    delta = _softplus(s["delta"].float() + s["delta_bias"])
    B, C = _per_channel(s["B"], channels), _per_channel(s["C"], channels)
    h = torch.exp(delta[..., None] * s["A"]) * state[slots] + (delta * u)[..., None] * B
    state[slots] = h
    y = (C * h).sum(-1) + s["skip"] * u
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z * torch.sigmoid(z)
    return {"out": y.to(s["u"].dtype), "state": state}


# ----------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    if case["op"] == "dropout":
        return _exact_dropout(s)
    if case["op"] == "conv":
        return _exact_conv(s)
    if case["op"] == "conv_step":
        return _exact_conv_step(s)
    if case["op"] == "scan":
        return _exact_scan(s)
    return _exact_scan_step(s)


def _philox(counter, key):
    """Philox4x32-10 of counters in numpy's unsigned 64-bit numbers."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(q >> half) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> half) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def _exact_dropout(s):
    """The generator on the host, apart from the plain form's."""
    x, p = s["x"], s["case"]["p"]
    n = x.numel()
    seed, offset = (int(v) & 0xFFFFFFFFFFFFFFFF for v in s["key"].tolist())
    limit = round(p * 65536)
    block = np.arange((n + 7) // 8, dtype=np.uint64)
    words = _philox((block & np.uint64(0xFFFFFFFF), block >> np.uint64(32),
                     np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)),
                    (seed & 0xFFFFFFFF, seed >> 32))
    kept = np.empty((block.size, 8), dtype=bool)
    for i, word in enumerate(words):
        kept[:, 2 * i] = (word & np.uint64(0xFFFF)) >= limit
        kept[:, 2 * i + 1] = (word >> np.uint64(16)) >= limit
    kept = torch.from_numpy(kept.reshape(-1)[:n]).to(x.device).view(x.shape)
    scale = 65536 / (65536 - limit) if limit < 65536 else 0.0
    out = torch.where(kept, x.double() * scale, 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].double()
    outs = {"out": out}
    if s["case"]["train"]:
        outs["grad_x"] = torch.where(kept, s["grad"].double() * scale, 0.0)
        if s["residual"] is not None:
            outs["grad_residual"] = s["grad"].double()
    return outs


def _exact_conv(s):
    """Tap by tap; a row beyond its length by setting what is read there to 0."""
    case = s["case"]
    x, w = s["x"].double(), s["weight"].double()
    batch, channels, length = x.shape
    taps = case["taps"]
    counts = [length] * batch if s["lengths"] is None else s["lengths"].tolist()
    line = x.new_zeros(batch, channels, taps - 1 + length)
    live = x.new_zeros(batch, 1, length)
    if s["state"] is not None:
        line[..., :taps - 1] = s["state"].double()
    for i, n in enumerate(counts):
        line[i, :, taps - 1:taps - 1 + n] = x[i, :, :n]
        live[i, :, :n] = 1
    pre = x.new_zeros(batch, channels, length)
    for k in range(taps):
        pre += w[:, k, None] * line[..., k:k + length]
    if s["bias"] is not None:
        pre += s["bias"].double()[:, None]
    gate = 1 / (1 + torch.exp(-pre)) if case["silu"] else torch.ones_like(pre)
    outs = {"out": pre * gate * live}
    if case["carried"] or case["ragged"]:
        outs["state"] = torch.stack([line[i, :, n:n + taps - 1] for i, n in enumerate(counts)])
    if not case["train"]:
        return outs
    slope = gate + pre * gate * (1 - gate) if case["silu"] else gate
    dpre = s["grad"].double() * slope * live
    dline = torch.zeros_like(line)
    dw = []
    for k in range(taps):
        dline[..., k:k + length] += w[:, k, None] * dpre
        dw.append((dpre * line[..., k:k + length]).sum((0, 2)))
    if s["grad_state"] is not None:
        for i, n in enumerate(counts):
            dline[i, :, n:n + taps - 1] += s["grad_state"][i].double()
    outs["grad_x"] = dline[..., taps - 1:].clone()
    outs["grad_weight"] = torch.stack(dw, -1)
    if s["bias"] is not None:
        outs["grad_bias"] = dpre.sum((0, 2))
    if s["state"] is not None:
        outs["grad_state"] = dline[..., :taps - 1].clone()
    return outs


def _exact_conv_step(s):
    state = s["state"].double()
    w, taps = s["weight"].double(), s["case"]["taps"]
    rows = s["slots"].long()
    pre = s["x"].double() * w[:, taps - 1]
    for k in range(taps - 1):
        pre = pre + state[rows][..., k] * w[:, k]
    if s["bias"] is not None:
        pre = pre + s["bias"].double()
    for k in range(taps - 2):
        state[rows, :, k] = state[rows, :, k + 1]
    if taps > 1:
        state[rows, :, taps - 2] = s["x"].double()
    return {"out": pre / (1 + torch.exp(-pre)) if s["case"]["silu"] else pre, "state": state}


def _exact_scan(s):
    """Token by token, forwards and backwards."""
    case = s["case"]
    u, raw = s["u"].double(), s["delta"].double() + s["delta_bias"].double()[:, None]
    batch, channels, length = u.shape
    states, groups = case["states"], case["groups"]
    delta = torch.logaddexp(raw, torch.zeros_like(raw))
    counts = None if s["lengths"] is None else s["lengths"]
    A, skip = s["A"].double(), s["skip"].double()
    each = channels // groups

    def at(v, t):  # [batch, groups, 1, states] of one token, over the group's channels
        return v[..., t].double()[:, :, None]

    def wide(v):  # [batch, channels, ...] as [batch, groups, each, ...]
        return v.view(batch, groups, each, *v.shape[2:])

    h = u.new_zeros(batch, channels, states) if s["state"] is None else s["state"].double()
    hs, y = [h], torch.empty_like(u)
    for t in range(length):
        new = torch.exp(delta[..., t, None] * A) * h
        new = new + (wide((delta[..., t] * u[..., t])[..., None]) * at(s["B"], t)).view_as(new)
        h = new if counts is None else torch.where((t < counts)[:, None, None], new, h)
        if case["train"]:
            hs.append(h)
        y[..., t] = (wide(h) * at(s["C"], t)).sum(-1).view(batch, channels)
    y += skip[:, None] * u
    gate = torch.ones_like(y)
    if s["z"] is not None:
        z = s["z"].double()
        sig = 1 / (1 + torch.exp(-z))
        gate = z * sig
    live = torch.ones_like(y)
    if counts is not None:
        live = (torch.arange(length, device=u.device) < counts[:, None])[:, None].double()
    outs = {"out": y * gate * live}
    if case["carried"] or case["ragged"]:
        outs["state"] = h
    if not case["train"]:  # (a training case has no lengths)
        return outs
    grad = s["grad"].double()
    dy = grad * gate
    du, ddelta = skip[:, None] * dy, torch.zeros_like(u)
    dA = torch.zeros_like(A)
    dB, dC = (torch.zeros(batch, groups, states, length, dtype=torch.float64, device=u.device) for _ in range(2))
    r = torch.zeros_like(h) if s["grad_state"] is None else s["grad_state"].double()
    for t in reversed(range(length)):
        dh = r + (wide(dy[..., t])[..., None] * at(s["C"], t)).view_as(r)
        a = torch.exp(delta[..., t, None] * A)
        dC[..., t] = (wide(dy[..., t])[..., None] * wide(hs[t + 1])).sum(2)
        dB[..., t] = (wide(dh) * wide(delta[..., t] * u[..., t])[..., None]).sum(2)
        through = (wide(dh) * at(s["B"], t)).sum(-1).view(batch, channels)
        r = a * dh
        du[..., t] += delta[..., t] * through
        ddelta[..., t] = u[..., t] * through + (r * hs[t] * A).sum(-1)
        dA += (r * hs[t] * delta[..., t, None]).sum(0)
    draw_ = ddelta / (1 + torch.exp(-raw))
    outs.update(grad_u=du, grad_delta=draw_, grad_A=dA, grad_B=dB, grad_C=dC, grad_skip=(dy * u).sum((0, 2)))
    if s["z"] is not None:
        outs["grad_z"] = grad * y * (sig + gate * (1 - sig))
    outs["grad_delta_bias"] = draw_.sum((0, 2))
    if s["state"] is not None:
        outs["grad_state"] = r
    return outs


def _exact_scan_step(s):
    batch, channels = s["u"].shape
    groups = s["case"]["groups"]
    state, rows = s["state"].double(), s["slots"].long()
    u, z = s["u"].double(), None if s["z"] is None else s["z"].double()
    raw = s["delta"].double() + s["delta_bias"].double()
    delta = torch.logaddexp(raw, torch.zeros_like(raw))
    owner = torch.arange(channels, device=u.device) // (channels // groups)
    B, C = s["B"].double()[:, owner], s["C"].double()[:, owner]
    h = torch.exp(torch.einsum("bc,cn->bcn", delta, s["A"].double())) * state[rows]
    h = h + torch.einsum("bc,bcn->bcn", delta * u, B)
    y = torch.einsum("bcn,bcn->bc", h, C) + s["skip"].double() * u
    state[rows] = h
    return {"out": y if z is None else y * z / (1 + torch.exp(-z)), "state": state}


def work(case):
    """Bytes that have to be read and written once, and operations, of one pass."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        passes = 3 if case["residual"] else 2
        if case["train"]:  # the gradient read, the input's written (the residual's is the gradient itself)
            passes += 2
        return {"bytes": n * size * passes, "flops": n * (2 if case["train"] else 1)}
    batch, channels = case["batch"], case["channels"]
    if case["op"] == "conv_step":
        taps, n = case["taps"], batch * channels
        return {"bytes": size * (n * 2 * taps + channels * (taps + 1)), "flops": n * 2 * taps}
    if case["op"] == "scan_step":
        n, states = batch * channels, case["states"]
        arrays = 4 if case["gate"] else 3
        return {"bytes": 8 * n * states + size * (arrays * n + 2 * batch * case["groups"] * states)
                + 4 * channels * (states + 2), "flops": 7 * n * states}
    n = batch * channels * case["length"]
    if case["op"] == "conv":
        taps = case["taps"]
        if case["train"]:  # forwards x, out; backwards x, the gradient, x's gradient
            return {"bytes": size * 5 * n, "flops": n * 2 * taps * 3}
        return {"bytes": size * (2 * n + (2 * batch * channels * (taps - 1) if case["carried"] else 0)),
                "flops": n * 2 * taps}
    states = case["states"]
    arrays = 4 if case["gate"] else 3
    shared = 2 * batch * case["groups"] * states * case["length"]
    kept = 8 * batch * channels * states if case["carried"] else 0
    if case["train"]:  # backwards: all inputs and the gradient again, and a gradient for each input
        arrays = 4 + 7 if case["gate"] else 3 + 5
        return {"bytes": size * (arrays * n + 3 * shared) + 2 * kept, "flops": 27 * n * states}
    return {"bytes": size * (arrays * n + shared) + kept, "flops": 7 * n * states}

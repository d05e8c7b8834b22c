"""Cases of the operators that a training step of a network needs beside its
layers: group norm with an activation, linear attention with a decay for each
head (whole sequences and single tokens), and an AdamW step over many tensors
with states in 32 or in 8 bits.

``run`` computes a case in its plain form (elementary torch operations in 32
bits, in 64 where sums are long, rounded once at the end), or with ``own`` set
through the package's entry points.  ``exact`` computes the same from the
definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BETAS, EPS = (0.9, 0.999), 1e-8
BLOCK = 256  # elements that share an exponent where states are held in 8 bits
CHUNK = 64  # tokens that the plain form of linear attention takes at once


def listed():
    return [
        # Behind the convolution of 64 to 128 channels over 56x56 maps, a training step in the layer's own order.
        {"name": "norm_train_map_fp32", "op": "norm", "dtype": "fp32", "batch": 64, "channels": 128, "length": 56 * 56,
         "groups": 32, "last": False, "silu": True, "ragged": False, "train": True},
        # A training step over 64x64 maps of 512 channels, channels last.
        {"name": "norm_train_last_bf16", "op": "norm", "dtype": "bf16", "batch": 16, "channels": 512,
         "length": 64 * 64, "groups": 32, "last": True, "silu": True, "ragged": False, "train": True},
        # Two small maps of an odd extent at inference: the launch is what counts.
        {"name": "norm_small_last_fp16", "op": "norm", "dtype": "fp16", "batch": 2, "channels": 320, "length": 17 * 31,
         "groups": 32, "last": True, "silu": True, "ragged": False, "train": False},
        # A training step at 8192 tokens, a decay for each token and head.
        {"name": "attention_train_bf16", "op": "attention", "dtype": "bf16", "batch": 4, "heads": 32, "groups": 32,
         "length": 2048, "keys": 64, "values": 64, "tokens": True, "ragged": False, "carried": False, "train": True},
        # One long prompt: few heads, a long axis, one decay for each head.
        {"name": "attention_prompt_long_bf16", "op": "attention", "dtype": "bf16", "batch": 1, "heads": 16,
         "groups": 16, "length": 16384, "keys": 128, "values": 128, "tokens": False, "ragged": False,
         "carried": False, "train": False},
        # Prompts of several lengths that go on from a kept state; odd sizes, queries and keys shared by two heads.
        {"name": "attention_prompt_ragged_fp16", "op": "attention", "dtype": "fp16", "batch": 7, "heads": 10,
         "groups": 5, "length": 777, "keys": 48, "values": 80, "tokens": True, "ragged": True, "carried": True,
         "train": False},
        # One token for each of 64 requests, their states among 96 places.
        {"name": "attention_step_bf16", "op": "attention_step", "dtype": "bf16", "batch": 64, "heads": 32,
         "groups": 32, "keys": 128, "values": 128, "tokens": False, "places": 96},
        # One token of one request of a small model.
        {"name": "attention_step_small_fp32", "op": "attention_step", "dtype": "fp32", "batch": 1, "heads": 12,
         "groups": 12, "keys": 64, "values": 64, "tokens": True, "places": 1},
        # The weights of two layers of width 2048 in 16 bits, with their copies and states in 32.
        {"name": "adamw_train_bf16", "op": "adamw", "dtype": "bf16", "grads": "bf16", "width": 2048, "layers": 2,
         "tagged": False, "masters": True, "bits": 32, "scaled": True},
        # A stack of four convolution layers of 64 channels: few and small tensors with their own rates.
        {"name": "adamw_stack_fp32", "op": "adamw", "dtype": "fp32", "grads": "fp32", "width": 64, "layers": 4,
         "tagged": True, "masters": False, "bits": 32, "scaled": False},
        # A layer of width 2048 in 16 bits, states in 8 bits, which are then read out as a checkpoint does.
        {"name": "adamw_8bit_bf16", "op": "adamw", "dtype": "bf16", "grads": "bf16", "width": 2048, "layers": 1,
         "tagged": False, "masters": False, "bits": 8, "scaled": True},
        # Tensors of odd sizes, states in 8 bits.
        {"name": "adamw_8bit_odd_fp32", "op": "adamw", "dtype": "fp32", "grads": "fp32", "width": 333, "layers": 4,
         "tagged": False, "masters": False, "bits": 8, "scaled": True},
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5)))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm", "attention", "attention", "attention", "attention_step", "adamw", "adamw"])
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "norm":
        batch, groups = _spread(rng, 1, 64), rng.choice([1, 4, 8, 16, 32])
        channels = groups * _spread(rng, 1, 32)
        last = rng.random() < 0.5
        return {**case, "batch": batch, "channels": channels,
                "length": _spread(rng, 1, min(16384, (1 << 24) // (batch * channels))), "groups": groups,
                "last": last, "silu": rng.random() < 0.7, "ragged": rng.random() < 0.3, "train": rng.random() < 0.6}
    if op == "adamw":
        tagged, bits = rng.random() < 0.3, rng.choice([32, 8])
        layers = _spread(rng, 1, 15 if tagged else 3)
        most = math.isqrt((1 << 25) // (layers * (18 if tagged else 11)))
        return {**case, "grads": rng.choice([case["dtype"], "fp32"]), "width": _spread(rng, 1, min(1024, most)),
                "layers": layers, "tagged": tagged, "masters": case["dtype"] != "fp32" and rng.random() < 0.5,
                "bits": bits, "scaled": rng.random() < 0.5}
    groups = _spread(rng, 1, 16)
    heads = groups * rng.choice([1, 1, 2, 4])
    case.update(heads=heads, groups=groups, keys=_spread(rng, 8, 128), values=_spread(rng, 8, 128),
                tokens=rng.random() < 0.5)
    if op == "attention_step":
        batch = _spread(rng, 1, 32)
        return {**case, "batch": batch, "places": batch + rng.randint(0, 32)}
    batch, train = _spread(rng, 1, 8), rng.random() < 0.5
    return {**case, "batch": batch, "length": _spread(rng, 1, min(16384, (1 << 16) // (batch * heads))),
            "ragged": rng.random() < 0.4, "carried": rng.random() < 0.5, "train": train}


def _shapes(case):
    """The shapes of an optimizer's tensors: of layers of a width, or the flat parameters of convolutions."""
    w = case["width"]
    if case["tagged"]:  # the first one of 3 channels
        return [(2 * w * (1 + 9 * (3 if i == 0 else w)),) for i in range(case["layers"])]
    return [s for _ in range(case["layers"]) for s in ((w, w), (2 * w, w), (4 * w, w), (w, 4 * w), (w,))]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=kind):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)

    def uniform(low, high, *shape):
        return torch.rand(shape, generator=g, device="cuda") * (high - low) + low

    def lengths(batch, most):  # padded rows of any length; the first full, one of them empty, one of one token
        n = torch.randint(1, most + 1, (batch,), generator=g, device="cuda").to(torch.int32)
        n[:1] = most
        n[1:3] = torch.arange(2, device="cuda", dtype=torch.int32)[:max(0, min(2, batch - 1))]
        return n

    s = {"case": case, "wanted": []}
    if case["op"] == "norm":
        batch, channels, length = case["batch"], case["channels"], case["length"]

        def drawn(**kw):
            if not case["last"]:
                return normal(batch, channels, length, **kw)
            return normal(batch, length, channels, **kw).transpose(1, 2)  # [batch, channels, length], channels last

        # channels of their own means, as a convolution gives them
        s["x"] = drawn()
        s["x"] += normal(channels, 1)
        s["weight"] = normal(channels, scale=0.2, shift=1.0)
        s["bias"] = normal(channels, scale=0.2)
        s["lengths"] = lengths(batch, length) if case["ragged"] else None
        if case["train"]:
            s["grad"] = drawn()
            s["wanted"] = ["x", "weight", "bias"]
    elif case["op"] == "adamw":
        s["params"], s["grads"], s["m"], s["v"] = [], [], [], []
        s["masters"] = [] if case["masters"] else None
        s["scales"] = [] if case["bits"] == 8 else None
        s["factors"] = [] if case["tagged"] else None
        for shape in _shapes(case):
            n = math.prod(shape)
            weight = normal(*shape, scale=0.05, dtype=torch.float32)
            s["params"].append(weight.to(kind))
            if case["masters"]:
                s["masters"].append(weight)
            # gradients of very different sizes, as the rows of an embedding or the channels of a map have them
            size = torch.exp(uniform(math.log(1e-4), math.log(1e-2), shape[0], *([1] * (len(shape) - 1))))
            s["grads"].append((torch.randn(shape, generator=g, device="cuda") * size).to(TYPES[case["grads"]]))
            m = 0.3 * size * torch.randn(shape, generator=g, device="cuda")
            v = size * size * uniform(0.5, 1.5, *shape)
            if case["bits"] == 8:
                blocks = -(-n // BLOCK)
                low = torch.randint(0, 256, (2, n), generator=g, device="cuda", dtype=torch.int32)
                scales = torch.empty(blocks, 2, dtype=torch.uint8, device="cuda")
                m, scales[:, 0] = _encode(m.flatten(), low[0], True)
                v, scales[:, 1] = _encode(v.flatten(), low[1], False)
                s["scales"].append(scales)
            s["m"].append(m)
            s["v"].append(v)
            if case["tagged"]:  # half of a layer's parameters at one rate, half at another; a decay of its own
                s["factors"].append((n // 2, 1.0, 0.5, 0.25))
        s["step"] = torch.full((1,), 1000, dtype=torch.int64, device="cuda")
        s["scale"] = uniform(0.2, 1.0, 1) if case["scaled"] else None  # what clips the gradients' norm
        s["seed"] = seed
    else:
        batch, heads, groups = case["batch"], case["heads"], case["groups"]
        step = case["op"] == "attention_step"
        length = () if step else (case["length"],)
        s["q"] = normal(batch, groups, case["keys"], *length)
        s["k"] = normal(batch, groups, case["keys"], *length, scale=case["keys"] ** -0.5)
        s["v"] = normal(batch, heads, case["values"], *length)
        if case["tokens"]:  # from nearly none to a factor of 1/e and less at a token
            s["log_decay"] = -torch.exp(uniform(math.log(1e-3), math.log(2.0), batch, heads, *length))
        else:  # memories of 32 to 4096 tokens over the heads
            s["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(5, 12, heads, device="cuda")))
        s["lengths"] = lengths(batch, case["length"]) if case.get("ragged") else None
        s["state"] = None
        if step or case["carried"]:
            s["state"] = normal(case["places"] if step else batch, heads, case["keys"], case["values"],
                                dtype=torch.float32)
        if step:  # the requests' places, in no order
            s["slots"] = torch.randperm(case["places"], generator=g, device="cuda")[:batch].to(torch.int32)
        elif case["train"]:
            s["grad"] = normal(*s["v"].shape)
            s["grad_state"] = normal(*s["state"].shape, dtype=torch.float32) if case["carried"] else None
            s["wanted"] = ["q", "k", "v", "log_decay"] + (["state"] if case["carried"] else [])
    for n in s["wanted"]:
        s[n].requires_grad_(True)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    with torch.no_grad():
        if op == "norm":
            return _plain_norm(state)
        if op == "adamw":
            return _plain_adamw(state)
        if op == "attention":
            return _plain_attention(state)
        return _plain_attention_step(state)


def _own(s):
    import paraconv2d_b200 as pc

    case = s["case"]
    if case["op"] == "attention_step":
        out = pc.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"])
        return {"out": out, "state": s["state"]}
    if case["op"] == "adamw":
        pc.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], lr=1e-3, betas=BETAS, eps=EPS,
                      weight_decay=0.1, masters=s["masters"], scales=s["scales"], factors=s["factors"],
                      grad_scale=s["scale"], seed=s["seed"])
        m, v = s["m"], s["v"]
        if case["bits"] == 8:
            m, v = pc.adamw_state_values(m, v, s["scales"], dtype=torch.bfloat16)
        return _adamw_outputs(s, m, v)
    if case["op"] == "norm":
        outs = {"out": pc.group_norm(s["x"], case["groups"], s["weight"], s["bias"],
                                     activation="silu" if case["silu"] else None, lengths=s["lengths"])}
        grads = [s.get("grad")]
    else:
        out = pc.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["state"],
                                  lengths=s["lengths"], return_final_state=_keeps(case))
        outs = {"out": out[0], "state": out[1]} if _keeps(case) else {"out": out}
        grads = [s.get("grad"), s.get("grad_state")][:len(outs)]
    if case["train"]:
        given = [(o, g) for o, g in zip(outs.values(), grads) if g is not None]
        got = torch.autograd.grad([o for o, _ in given], [s[n] for n in s["wanted"]], [g for _, g in given])
        outs.update({"grad_" + n: v for n, v in zip(s["wanted"], got)})
    return outs


def _keeps(case):
    """Whether a call returns the state after the last token."""
    return case["carried"] or case["ragged"] or not case["train"]


def _inside(s, length):
    """True where a row has a token, [batch, 1, length]; None without lengths."""
    if s["lengths"] is None:
        return None
    return (torch.arange(length, device="cuda") < s["lengths"][:, None])[:, None]


# ----------------------------------------------------------------- group norm

def _plain_norm(s):
    case, kind = s["case"], s["x"].dtype
    batch, channels, length = s["x"].shape
    groups = case["groups"]
    inside = _inside(s, length)

    def masked(v):
        return v if inside is None else torch.where(inside, v, 0.0)

    def mean(v):  # over a group's channels and tokens, back at every channel
        sums = v.sum(2, dtype=torch.float64).view(batch, groups, -1).sum(2)
        return (sums / count).float().repeat_interleave(channels // groups, 1)[..., None]

    tokens = torch.full((batch, 1), length, device="cuda") if inside is None else s["lengths"][:, None].clamp(min=1)
    count = tokens * (channels // groups)
    x, w, b = masked(s["x"].float()), s["weight"].float()[:, None], s["bias"].float()[:, None]
    off = masked(x - mean(x))
    rstd = torch.rsqrt(mean(off * off) + 1e-5)
    xhat = off * rstd
    pre = xhat * w + b
    sig = torch.sigmoid(pre)
    outs = {"out": masked(pre * sig if case["silu"] else pre).to(kind)}
    if case["train"]:
        h = masked(s["grad"].float())
        if case["silu"]:
            h = h * sig * (1 + pre * (1 - sig))
        hw = h * w
        outs["grad_x"] = masked(rstd * (hw - mean(hw) - xhat * mean(hw * xhat))).to(kind)
        outs["grad_weight"] = (h * xhat).sum((0, 2), dtype=torch.float64).to(kind)
        outs["grad_bias"] = h.sum((0, 2), dtype=torch.float64).to(kind)
    return outs


# ----------------------------------------------------------- linear attention

def _tokens_first(v, heads):
    """[batch, groups, dim, length] -> [batch, heads, length, dim] in 32 bits."""
    return v.float().transpose(2, 3).repeat_interleave(heads // v.shape[1], 1)


def _decays(s):
    """The decays' logarithms, [batch, heads, length] in 64 bits."""
    g = s["log_decay"].double()
    return g if s["case"]["tokens"] else g[:, None].expand(s["v"].shape[0], -1, s["v"].shape[3])


def _plain_attention(s):
    case, kind = s["case"], s["v"].dtype
    batch, heads, _, length = s["v"].shape
    groups, keys, scale = case["groups"], case["keys"], case["keys"] ** -0.5
    inside = _inside(s, length)
    count = -(-length // CHUNK)

    def chunks(v):  # zeros at what is no token, and up to a whole chunk; [batch, heads, chunks, CHUNK, ...]
        if inside is not None:
            v = torch.where(inside if v.dim() == 3 else inside[..., None], v, 0.0)
        tail = torch.zeros_like(v[:, :, :1]).expand(-1, -1, count * CHUNK - length, *v.shape[3:])
        v = torch.cat([v, tail], 2)
        return v.view(batch, heads, count, CHUNK, *v.shape[3:])

    def whole(v):  # and back: [batch, heads, dim, length]
        return v.reshape(batch, heads, count * CHUNK, -1)[:, :, :length].transpose(2, 3)

    q, k, v = (chunks(_tokens_first(s[n], heads)) for n in "qkv")
    g = chunks(_decays(s))
    upto = g.cumsum(-1)  # of the decays' logarithms from a chunk's first token on
    near = torch.tril(torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda"))
    between = torch.where(near, torch.exp(upto[..., :, None] - upto[..., None, :]).float(), 0.0)
    begin, end = torch.exp(upto).float()[..., None], torch.exp(upto[..., -1:] - upto).float()[..., None]
    past = torch.exp(upto[..., -1]).float()[..., None, None]
    scores = (q * scale) @ k.transpose(-1, -2) * between
    added = (k * end).transpose(-1, -2) @ v
    state = torch.zeros_like(added[:, :, 0]) if s["state"] is None else s["state"].float()
    before = []
    for c in range(count):
        before.append(state)
        state = past[:, :, c] * state + added[:, :, c]
    before = torch.stack(before, 2)
    outs = {"out": whole(scores @ v + begin * ((q * scale) @ before)).to(kind)}
    if _keeps(case):
        outs["state"] = state.clone()
    if not case["train"]:
        return outs
    grad = chunks(_tokens_first(s["grad"], heads))
    left = ((q * scale) * begin).transpose(-1, -2) @ grad
    dstate = torch.zeros_like(state) if s["grad_state"] is None else s["grad_state"]
    behind = []
    for c in reversed(range(count)):
        behind.append(dstate)
        dstate = past[:, :, c] * dstate + left[:, :, c]
    behind = torch.stack(behind[::-1], 2)
    dscores = grad @ v.transpose(-1, -2) * between
    dq_old = begin * (grad @ before.transpose(-1, -2)) * scale
    dk_new = end * (v @ behind.transpose(-1, -2))
    dq = dscores @ k * scale + dq_old
    dk = dscores.transpose(-1, -2) @ (q * scale) + dk_new
    dv = scores.transpose(-1, -2) @ grad + end * (k @ behind)
    # a decay at token t acts between every earlier token and t or a later one: pairs within the chunk, of its
    # tokens and the state before it, of its tokens and what comes behind it, and of the two beyond it
    pairs = (scores * (grad @ v.transpose(-1, -2))).double()
    old, new = (q * dq_old).sum(-1, dtype=torch.float64), (k * dk_new).sum(-1, dtype=torch.float64)
    late = pairs.sum(-1) - pairs.sum(-2) + old
    across = (past * before * behind).sum((-1, -2), dtype=torch.float64)[..., None]
    dg = late.flip(-1).cumsum(-1).flip(-1) + new.cumsum(-1) - new + across
    dg = dg.reshape(batch, heads, -1)[..., :length].float()
    if inside is not None:
        dg = torch.where(inside, dg, 0.0)

    def summed(v):  # over the heads of a group
        v = whole(v)
        if inside is not None:
            v = torch.where(inside[:, :, None], v, 0.0)
        return v.reshape(batch, groups, heads // groups, keys, length).sum(2).to(kind)

    outs["grad_q"], outs["grad_k"] = summed(dq), summed(dk)
    dv = whole(dv)
    outs["grad_v"] = (dv if inside is None else torch.where(inside[:, :, None], dv, 0.0)).to(kind)
    outs["grad_log_decay"] = dg if case["tokens"] else dg.sum((0, 2), dtype=torch.float64).float()
    if s["state"] is not None:
        outs["grad_state"] = dstate
    return outs


def _plain_attention_step(s):
    heads, slots, state = s["v"].shape[1], s["slots"].long(), s["state"]
    q, k = (s[n].float().repeat_interleave(heads // s[n].shape[1], 1) for n in "qk")
    a = torch.exp(s["log_decay"])[..., None, None]
    new = a * state[slots] + k[..., None] * s["v"].float()[:, :, None]
    state[slots] = new
    out = (q[..., None] * new).sum(2) * s["case"]["keys"] ** -0.5
    return {"out": out.to(s["v"].dtype), "state": state}


# ----------------------------------------------------------------- AdamW step

def _bits8(n, seed, step, index):
    """Two rows of n 8-bit numbers: Philox4x32-10 (Salmon, Moraes, Dror and
    Shaw, 2011) under the key `seed`, of the counters (i // 8, index, step):
    the first two words' bytes are the first row's, in their order, the last
    two's the second's."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 7) // 8, device=step.device)
    x = [block, torch.full_like(block, index), (step & low).expand_as(block), ((step >> 32) & low).expand_as(block)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [((p1 >> 32) & low) ^ x[1] ^ k0, p1 & low, ((p0 >> 32) & low) ^ x[3] ^ k1, p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    shifts = torch.arange(0, 32, 8, device=block.device)
    rows = [((torch.stack(x[i:i + 2], -1)[..., None] >> shifts) & 255).reshape(-1)[:n] for i in (0, 2)]
    return torch.stack(rows).to(torch.int32)


def _encode(x, low, signed):
    """The values x as 8-bit floats with 3 bits of mantissa, under the
    exponent of the smallest normal number of each block of 256: the one that
    brings the block's largest, rounded up to a code, into the topmost of 15
    (beside a sign) or 31 binades.  Rounded up with the probability of what is cut off, by the
    8-bit numbers `low`."""
    n, top = x.numel(), 15 if signed else 31
    size = x.abs()
    blocks = torch.nn.functional.pad(size, (0, -n % BLOCK)).view(-1, BLOCK)
    most = blocks.amax(1).view(torch.int32)
    scale = torch.where(most >> 23 == 255, 255, ((most + 0xFFFFF >> 23) - (top - 1)).clamp(min=1))
    least = (scale << 23).view(torch.float32).repeat_interleave(BLOCK)[:n]
    wide = scale.repeat_interleave(BLOCK)[:n] << 3
    down = low * 4096 + 2048
    normal = size >= least
    shifted = torch.where(normal, size, size + least).view(torch.int32)
    code = ((shifted + down) >> 20) - wide + torch.where(normal, 8, 0)
    if not signed:  # a second moment that is not zero stays so: the step is divided by its root
        code = torch.where((size > 0) & (code == 0), 1, code)
    code = torch.where(wide == 255 << 3, 0, code)
    if signed:
        code = code | torch.where(x < 0, 128, 0)
    return code.to(torch.uint8), scale.to(torch.uint8)


def _decode(code, scale, signed):
    n = code.numel()
    code = code.to(torch.int32)
    size = code & 127 if signed else code
    least = (scale.to(torch.int32) << 23).repeat_interleave(BLOCK)[:n]
    small = size < 8
    value = (torch.where(small, size << 20, size - 8 << 20) + least).view(torch.float32)
    value = torch.where(small, value - least.view(torch.float32), value)
    value = torch.where(least == 255 << 23, float("nan"), value)
    return torch.where(code > 127, -value, value) if signed else value


def _adamw_outputs(s, m, v):
    outs = {}
    for name, tensors in (("param", s["params"]), ("master", s["masters"] or []), ("m", m), ("v", v)):
        outs.update({f"{name}{i}": t for i, t in enumerate(tensors)})
    outs["step"] = s["step"]
    return outs


def _plain_adamw(s):
    bits8 = s["case"]["bits"] == 8
    step = s["step"].add_(1)
    b1, b2 = BETAS
    t = step.double()
    size1, size2 = 1 - b1 ** t, (1 - b2 ** t).rsqrt().float()
    values_m, values_v = [], []
    for i, param in enumerate(s["params"]):
        n = param.numel()
        split, first, rest, decay = s["factors"][i] if s["factors"] else (n, 1.0, 1.0, 1.0)
        lr = torch.where(torch.arange(n, device="cuda") < split, first, rest).double() * 1e-3
        g = s["grads"][i].float().flatten()
        if s["scale"] is not None:
            g = g * s["scale"]
        m, v = s["m"][i].flatten(), s["v"][i].flatten()
        if bits8:
            m, v = _decode(m, s["scales"][i][:, 0], True), _decode(v, s["scales"][i][:, 1], False)
        # each product and sum rounded to 32 bits: what they are decides the codes of 8 bits
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * (1 - b2)) * g
        weight = (s["masters"][i] if s["masters"] else param).flatten()
        new = weight.float() * (1 - lr * 0.1 * decay).float()
        new = new - (lr / size1).float() * (m / (v.sqrt() * size2 + EPS))
        if s["masters"]:
            s["masters"][i].copy_(new.view(param.shape))
        param.copy_(new.view(param.shape))
        if bits8:
            low = _bits8(n, s["seed"], step, i)
            s["m"][i], s["scales"][i][:, 0] = _encode(m, low[0], True)
            s["v"][i], s["scales"][i][:, 1] = _encode(v, low[1], False)
            values_m.append(_decode(s["m"][i], s["scales"][i][:, 0], True).to(torch.bfloat16))
            values_v.append(_decode(s["v"][i], s["scales"][i][:, 1], False).to(torch.bfloat16))
        else:
            s["m"][i].copy_(m.view(param.shape))
            s["v"][i].copy_(v.view(param.shape))
    return _adamw_outputs(s, values_m, values_v) if bits8 else _adamw_outputs(s, s["m"], s["v"])


# ----------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"] == "attention":
        return _exact_attention(s)
    return _exact_attention_step(s)


def _exact_norm(s):
    """One row at a time: its tokens alone, as [groups, channels of a group, tokens]."""
    case = s["case"]
    batch, channels, length = s["x"].shape
    shape = (case["groups"], channels // case["groups"], -1)
    w, b = s["weight"].double().view(shape), s["bias"].double().view(shape)
    new = lambda: torch.zeros(batch, channels, length, dtype=torch.float64, device="cuda")  # noqa: E731
    outs = {"out": new()}
    if case["train"]:
        outs.update(grad_x=new(), grad_weight=torch.zeros_like(w), grad_bias=torch.zeros_like(b))
    counts = [length] * batch if s["lengths"] is None else s["lengths"].tolist()
    for i, n in enumerate(counts):
        if n == 0:
            continue
        x = s["x"][i, :, :n].double().reshape(shape)
        centre = x.mean((1, 2), keepdim=True)
        spread = ((x - centre) ** 2).mean((1, 2), keepdim=True)
        unit = (x - centre) / (spread + 1e-5) ** 0.5
        pre = torch.addcmul(b, unit, w)
        gate = 1 / (1 + torch.exp(-pre)) if case["silu"] else torch.ones_like(pre)
        outs["out"][i, :, :n] = (pre * gate).reshape(channels, n)
        if case["train"]:
            h = s["grad"][i, :, :n].double().reshape(shape)
            if case["silu"]:
                h = h * (gate + pre * gate * (1 - gate))
            outs["grad_weight"] += (h * unit).sum(2, keepdim=True)
            outs["grad_bias"] += h.sum(2, keepdim=True)
            d = h * w
            d = d - d.mean((1, 2), keepdim=True) - unit * (d * unit).mean((1, 2), keepdim=True)
            outs["grad_x"][i, :, :n] = (d / (spread + 1e-5) ** 0.5).reshape(channels, n)
    for n in ("grad_weight", "grad_bias"):
        if n in outs:
            outs[n] = outs[n].reshape(channels)
    return outs


def _exact_attention(s):
    """Every pair of tokens of one row and head at a time, without chunks."""
    case = s["case"]
    batch, heads, values, length = s["v"].shape
    keys, groups = case["keys"], case["groups"]
    f64 = dict(dtype=torch.float64, device="cuda")
    outs = {"out": torch.zeros(batch, heads, values, length, **f64)}
    if _keeps(case):
        outs["state"] = torch.zeros(batch, heads, keys, values, **f64)
    if case["train"]:
        outs["grad_q"], outs["grad_k"] = (torch.zeros(batch, groups, keys, length, **f64) for _ in range(2))
        outs["grad_v"] = torch.zeros_like(outs["out"])
        outs["grad_log_decay"] = torch.zeros(batch, heads, length, **f64)
        if case["carried"]:
            outs["grad_state"] = torch.zeros(batch, heads, keys, values, **f64)
    counts = [length] * batch if s["lengths"] is None else s["lengths"].tolist()
    for i in range(batch):
        n = counts[i]
        for h in range(heads):
            share = h * groups // heads
            q, k = s["q"][i, share, :, :n].double().T * keys ** -0.5, s["k"][i, share, :, :n].double().T
            v = s["v"][i, h, :, :n].double().T
            g = s["log_decay"][i, h, :n].double() if case["tokens"] else s["log_decay"][h].double().expand(n)
            first = torch.zeros(keys, values, **f64) if s["state"] is None else s["state"][i, h].double()
            c = torch.cumsum(g, 0)
            total = c[-1] if n else torch.zeros((), **f64)
            decay = torch.tril(c[:, None] - c[None, :]).exp_().tril_()
            weight = q @ k.T * decay
            fade, tail = torch.exp(c)[:, None], torch.exp(total - c)[:, None]
            outs["out"][i, h, :, :n] = (weight @ v + fade * (q @ first)).T
            if _keeps(case):
                outs["state"][i, h] = torch.exp(total) * first + (tail * k).T @ v
            if not case["train"]:
                continue
            d = s["grad"][i, h, :, :n].double().T
            last = torch.zeros(keys, values, **f64) if s["grad_state"] is None else s["grad_state"][i, h].double()
            dweight = d @ v.T
            old, new = fade * (d @ first.T), tail * (v @ last.T)
            outs["grad_q"][i, share, :, :n] += ((dweight * decay) @ k + old).T * keys ** -0.5
            outs["grad_k"][i, share, :, :n] += ((dweight * decay).T @ q + new).T
            outs["grad_v"][i, h, :, :n] = (weight.T @ d + tail * (k @ last)).T
            flow = weight * dweight
            behind = (flow.sum(1) - flow.sum(0) + (q * old).sum(1)).flip(0).cumsum(0).flip(0)
            ahead = (k * new).sum(1)
            outs["grad_log_decay"][i, h, :n] = (behind + ahead.cumsum(0) - ahead
                                                + torch.exp(total) * (first * last).sum())
            if case["carried"]:
                outs["grad_state"][i, h] = torch.exp(total) * last + (fade * q).T @ d
    if case["train"] and not case["tokens"]:
        outs["grad_log_decay"] = outs["grad_log_decay"].sum((0, 2))
    return outs


def _exact_attention_step(s):
    heads, groups, rows = s["v"].shape[1], s["q"].shape[1], s["slots"].long()
    owner = torch.arange(heads, device="cuda") * groups // heads
    q, k, v = s["q"].double()[:, owner], s["k"].double()[:, owner], s["v"].double()
    state = s["state"].double()
    a = torch.exp(s["log_decay"].double()).expand(v.shape[:2])
    new = torch.einsum("bh,bhkv->bhkv", a, state[rows]) + torch.einsum("bhk,bhv->bhkv", k, v)
    state[rows] = new
    return {"out": torch.einsum("bhk,bhkv->bhv", q, new) / math.sqrt(s["case"]["keys"]), "state": state}


def _philox(counter, key):
    """Philox4x32-10 of counters in numpy's unsigned 64-bit numbers."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(q >> half) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> half) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def _held(x, chance, top):
    """What 8 bits hold of x >= 0: the multiple of its step (an eighth of its
    binade; of the lowest binade's under that) below it, or above it with the
    chance's probability."""
    blocks = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    # (above 15/8 of its binade, a block's largest may be rounded up into the next one)
    most = torch.floor(torch.log2((blocks.amax(1) * (16 / 15)).clamp(min=2.0 ** -126)))
    lowest = (most - (top - 1)).clamp(min=-126).repeat_interleave(BLOCK)[:x.numel()]
    binade = torch.maximum(torch.floor(torch.log2(x.clamp(min=1e-300))), lowest)
    step = torch.exp2(binade - 3)
    return torch.floor(x / step + chance) * step


def _exact_adamw(s):
    case = s["case"]
    bits8 = case["bits"] == 8
    t = int(s["step"]) + 1
    (b1, b2), lr = BETAS, 1e-3
    params, masters, ms, vs = [], [], [], []
    for i, param in enumerate(s["params"]):
        n = param.numel()
        g = s["grads"][i].double().flatten() * (1.0 if s["scale"] is None else s["scale"].double())
        if bits8:
            # a code's value: its eighths, with the one that a normal number has, at its exponent
            def value(code, scale):
                e = (code >> 3).clamp(min=1) - 1
                parts = torch.where(code >= 8, 8 + (code & 7), code).double()
                lowest = (scale.double() - 127).repeat_interleave(BLOCK)[:n]
                return parts / 8 * torch.exp2(lowest + e)

            code = s["m"][i].long()
            m = value(code & 127, s["scales"][i][:, 0]) * (1 - 2 * (code >> 7)).double()
            v = value(s["v"][i].long(), s["scales"][i][:, 1])
        else:
            m, v = s["m"][i].double().flatten(), s["v"][i].double().flatten()
        m = torch.lerp(g, m, b1)
        v = torch.lerp(g * g, v, b2)
        w = (s["masters"][i] if s["masters"] else param).double().flatten()
        rate = torch.full_like(w, lr)
        decay = 0.1
        if s["factors"]:
            split, first, rest, f = s["factors"][i]
            rate[:split] *= first
            rate[split:] *= rest
            decay *= f
        w = w - rate * decay * w - rate * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + EPS)
        params.append(w.view(param.shape))
        masters.append(w.view(param.shape))
        if bits8:
            groups = np.arange((n + 7) // 8, dtype=np.uint64)
            words = _philox((groups, np.full_like(groups, i), np.full_like(groups, t), np.zeros_like(groups)),
                            (s["seed"] & 0xFFFFFFFF, (s["seed"] >> 32) & 0xFFFFFFFF))
            low = [np.stack([(w_ >> np.uint64(8 * j)) & np.uint64(255) for w_ in words[p:p + 2] for j in range(4)], -1)
                   for p in (0, 2)]
            chance = [(torch.from_numpy(x.reshape(-1)[:n].astype(np.float64)).cuda() + 0.5) / 256 for x in low]
            m = torch.sign(m) * _held(m.abs(), chance[0], 15)
            held = _held(v, chance[1], 31)
            v = torch.where((held == 0) & (v > 0), _held(v, 1.0, 31), held)
        shape = (n,) if bits8 else param.shape
        ms.append(m.view(shape))
        vs.append(v.view(shape))
    outs = {}
    for name, tensors in (("param", params), ("master", masters if case["masters"] else []), ("m", ms), ("v", vs)):
        outs.update({f"{name}{i}": x for i, x in enumerate(tensors)})
    outs["step"] = s["step"] + 1
    return outs


def work(case):
    """Bytes that have to be read and written once, and operations, of one pass."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["batch"] * case["channels"] * case["length"]
        if case["train"]:  # forwards x, out; backwards x, the gradient, x's gradient
            return {"bytes": 5 * size * n, "flops": 30 * n}
        return {"bytes": 2 * size * n, "flops": 10 * n}
    if case["op"] == "adamw":
        n = sum(math.prod(shape) for shape in _shapes(case))
        each = (4 if case["grads"] == "fp32" else 2) + 2 * size
        if case["masters"]:  # the copies are read and written, the parameters only written
            each += 8 - size
        # states read and written, those of 8 bits also read out in 16
        each += 16 if case["bits"] == 32 else 4 + 2 + 4
        return {"bytes": each * n, "flops": 14 * n}
    batch, heads, groups = case["batch"], case["heads"], case["groups"]
    keys, values = case["keys"], case["values"]
    states = 4 * batch * heads * keys * values
    if case["op"] == "attention_step":
        return {"bytes": 2 * states + size * batch * (2 * groups * keys + 2 * heads * values),
                "flops": 5 * batch * heads * keys * values}
    tokens = batch * case["length"]
    decays = 4 * tokens * heads if case["tokens"] else 0
    shared, each = size * tokens * groups * keys, size * tokens * heads * values
    # with a state, a token costs a product and a sum for it and the same for its output
    flops = 4 * tokens * heads * keys * values
    kept = states * (case["carried"] + _keeps(case))
    if case["train"]:  # backwards: q, k, v, the gradient, and their gradients
        return {"bytes": 2 * shared + 2 * each + decays + kept + 4 * shared + 3 * each + 2 * decays + kept,
                "flops": 3 * flops}
    return {"bytes": 2 * shared + 2 * each + decays + kept, "flops": flops}

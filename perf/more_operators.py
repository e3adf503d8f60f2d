"""What a network on panoramas is trained with besides attention, as measurable cases.

Three operators of `mappedconvolutions_amd._C`: a gated linear recurrence along a sequence, group
norm with an activation over tokens whose channels lie last, and the AdamW step over a list of
tensors with moments in 32 or 8 bits.  `run` calls them where `own` is true and computes the same
from elementary torch operations in 32 bits where it is not; `exact` computes them in 64 bits.
`listed()` names the cases, `draw()` gives more of the same ranges.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}
BLOCK = 256  # values that share a scale in 8 bits
BETA1, BETA2, EPS, RATE, DECAY, STEP, SEED = 0.9, 0.999, 1e-8, 1e-3, 0.01, 100, 7


def listed():
    return [
        # One new token of each of 16 sequences, from the state kept for them.
        dict(name="recur_one_token_bf16", kind="recur", dtype="bf16", B=16, L=1, C=1024, gated=True,
             carried=True, ragged=False, reverse=False, train=False),
        # Training over the rows of eight 256 x 512 panoramas with 128 channels.
        dict(name="recur_rows_train_bf16", kind="recur", dtype="bf16", B=2048, L=512, C=128,
             gated=True, carried=False, ragged=False, reverse=False, train=True),
        # Training over all pixels of two 128 x 256 images in scan order.
        dict(name="recur_scan_train_bf16", kind="recur", dtype="bf16", B=2, L=32768, C=1024,
             gated=True, carried=False, ragged=False, reverse=False, train=True),
        # All pixels of 125 x 250 images from the last to the first, sequences of different lengths,
        # an unusual number of channels, in single precision, without an output gate.
        dict(name="recur_odd_train_fp32", kind="recur", dtype="fp32", B=3, L=31250, C=90,
             gated=False, carried=True, ragged=True, reverse=True, train=True),
        # Prompts of up to 2562 tokens before single tokens follow.
        dict(name="recur_prompt_bf16", kind="recur", dtype="bf16", B=4, L=2562, C=2048, gated=True,
             carried=True, ragged=True, reverse=False, train=False),
        # One 16 x 32 image of an encoder's last level: what counts is latency.
        dict(name="group_small_bf16", kind="group", dtype="bf16", B=1, N=512, C=128, groups=32,
             activation="silu", train=False),
        # Training on eight 256 x 512 panoramas with 64 channels, groups of four channels.
        dict(name="group_panorama_train_bf16", kind="group", dtype="bf16", B=8, N=131072, C=64,
             groups=16, activation="silu", train=True),
        # All pixels of 125 x 250 images in single precision, groups of 15 channels, no activation.
        dict(name="group_odd_train_fp32", kind="group", dtype="fp32", B=3, N=31250, C=90, groups=6,
             activation=None, train=True),
        # Many channels on few pixels, as deep in an encoder: 32 images of 32 x 64.
        dict(name="group_deep_train_bf16", kind="group", dtype="bf16", B=32, N=2048, C=512,
             groups=32, activation="gelu", train=True),
        # A small encoder's step, with its gradients clipped: a few dozen weights and biases.
        dict(name="adamw_encoder_fp32", kind="adamw", dtype="fp32", bits=32, tensors=30,
             largest=147456, spread=2304, clipped=True),
        # A large network's step: over half a billion weights, gradients in bf16.
        dict(name="adamw_large_bf16", kind="adamw", dtype="bf16", bits=32, tensors=300,
             largest=8388608, spread=64, clipped=False),
        # The same kind of network with its moments in 8 bits.
        dict(name="adamw_large_8bit_bf16", kind="adamw", dtype="bf16", bits=8, tensors=100,
             largest=8388608, spread=64, clipped=False),
    ]


def _log(rng, low, high):
    """A whole number between low and high, uniform in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("recur", "recur", "group", "group", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if kind == "adamw":
        bits = rng.choice((32, 8))
        return dict(kind="adamw", dtype=dtype, bits=bits, tensors=_log(rng, 1, 300 if bits == 32 else 100),
                    largest=_log(rng, 1000, 4000000), spread=_log(rng, 1, 1000),
                    clipped=rng.choice((True, False)))
    train = rng.choice((True, True, False))
    if kind == "group":
        groups = rng.choice((1, 2, 4, 6, 8, 16, 32))
        per = rng.choice((1, 2, 3, 4, 5, 8, 15, 16, 24, 32))
        C = groups * per
        # (a norm of a few dozen values at least)
        N = _log(rng, -(-48 // per), min(130000, 67000000 // C))
        B = _log(rng, 1, max(1, min(256, 33000000 // (N * C))))
        return dict(kind="group", dtype=dtype, B=B, N=N, C=C, groups=groups,
                    activation=rng.choice((None, "silu", "gelu")), train=train)
    C = rng.choice((_log(rng, 1, 2048), 8 * _log(rng, 1, 256), 64 * _log(rng, 1, 32)))
    L = rng.choice((1, _log(rng, 1, 40000), _log(rng, 1, 40000)))
    B = _log(rng, 1, max(1, min(4096, 33000000 // (L * C))))
    return dict(kind="recur", dtype=dtype, B=B, L=L, C=C, gated=rng.choice((True, False)),
                carried=rng.choice((True, False)), ragged=rng.choice((True, False)),
                reverse=rng.choice((True, False)), train=train)


def _lengths(case):
    """Tokens in use of every sequence: all of them, or from a half to all."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    return [max(1, L - (i * 7919 % max(1, B)) * L // (2 * B)) for i in range(B)]


def _sizes(case):
    """Sizes of the tensors: from `largest` down to `largest / spread`, odd ones among them."""
    n, top, spread = case["tensors"], case["largest"], case["spread"]
    sizes = []
    for i in range(n):
        part = (i * 0.6180339887) % 1.0
        size = int(top * math.exp(-part * math.log(spread)) if spread > 1 else top)
        sizes.append(max(1, size if i % 3 else size | 1))
    return sizes


def _blocks(sizes):
    return [-(-n // BLOCK) for n in sizes]


def _parts(flat, sizes):
    """The part of every tensor in the buffer of all, each from a whole block on."""
    padded = flat.split([BLOCK * n for n in _blocks(sizes)])
    return [part[:n] for part, n in zip(padded, sizes)]


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "recur":
        n = sum(_lengths(case)) * case["C"]
        wide = 3 if case["gated"] else 2
        streams = wide + 1 + ((2 * wide + 1) if case["train"] else 0)
        state = 4 * case["B"] * case["C"] * ((2 if case["carried"] else 1) + (2 if case["train"] else 0))
        return {"bytes": streams * n * size + state, "flops": n * (50 if case["train"] else 20)}
    if case["kind"] == "group":
        n = case["B"] * case["N"] * case["C"]
        return {"bytes": n * size * (5 if case["train"] else 2), "flops": n * (40 if case["train"] else 15)}
    n = sum(_sizes(case))
    moments = 16 if case["bits"] == 32 else 4 + 4  # read and written; in 8 bits also as values
    return {"bytes": n * (8 + size + moments), "flops": 20 * n}


# ---- moments in 8 bits --------------------------------------------------------------------
# A block's values over a power of two (twice the largest one's), as 3 bits behind the point with 4
# bits of exponent and a sign (first moment) or 5 bits of exponent (second): below 2^-14 or 2^-30
# the steps stay as they are.  Rounded up with the probability of what is cut off, by 16 bits of a
# word that seed, step and the value's index give; a second moment above zero stays above zero.

def _mix(x):
    """32 bits from 32 bits, in 64-bit whole numbers."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _words(first, n, device):
    """The random words of values first to first + n of the list."""
    key = _mix(_mix(STEP & 0xFFFFFFFF) ^ (SEED & 0xFFFFFFFF))
    at = torch.arange(first, first + n, device=device)
    return _mix(((at & 0xFFFFFFFF) ^ (((at >> 32) * 0x9E3779B1) & 0xFFFFFFFF)) + key & 0xFFFFFFFF)


def _scales(x):
    """The power of two of each block of |x| (whole blocks, 32 bits): twice the largest value's."""
    e = x.view(-1, BLOCK).amax(1).view(torch.int32) >> 23
    return torch.where(x.view(-1, BLOCK).amax(1) > 0, torch.ldexp(torch.ones_like(e, dtype=x.dtype),
                                                                (e - 126).clamp(-125, 127)), 0.0)


def _encode(x, words, low, signed):
    """(codes, scales) of one tensor's values in 32 bits; 2^low is the least with 3 bits."""
    n = x.numel()
    wide = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK))
    scale = _scales(wide)
    y = (wide.view(-1, BLOCK) * torch.where(scale > 0, 1 / scale, 0.0)[:, None]).view(-1)[:n]
    tiny = y < 2.0 ** low
    bits = torch.where(tiny, y + 2.0 ** low, y).view(torch.int32).long()
    least = (127 + low) << 3
    code = ((bits + ((words << 4) | 8)) >> 20) - least + torch.where(tiny, 0, 8)
    if signed:
        return (code.clamp_(max=127) | ((x < 0).long() << 7)).to(torch.uint8), scale
    return torch.where(x > 0, code.clamp_(1, 255), 0).to(torch.uint8), scale


def _decode(code, scale, low, signed):
    """The values that codes stand for, in 32 bits."""
    n, c = code.numel(), code.int()
    sign = 1 - 2 * (c >> 7) if signed else 1
    c = c & 127 if signed else c
    e, fraction = c >> 3, c & 7
    y = torch.ldexp((fraction + torch.where(e > 0, 8, 0)).float(), (e.clamp_min(1) - 1) + (low - 3))
    y = y * sign
    return (torch.nn.functional.pad(y, (0, -n % BLOCK)).view(-1, BLOCK) * scale[:, None]).view(-1)[:n]


# ---- inputs -------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    st = dict(case=case)
    if case["kind"] == "recur":
        B, L, C = case["B"], case["L"], case["C"]
        # parts of one projection, as a block has them; the forget gates of the channels reach from
        # a few tokens to hundreds
        parts = 3 if case["gated"] else 2
        packed = randn(B, L, parts * C)
        packed[..., C:2 * C] += torch.linspace(0.0, 6.0, C, device=dev, dtype=dtype)
        st["v"], st["f"] = packed[..., :C], packed[..., C:2 * C]
        st["g"] = packed[..., 2 * C:] if case["gated"] else None
        st["h"] = randn(B, C, dtype=torch.float32) if case["carried"] else None
        lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        st["lengths"] = lengths if case["ragged"] else None
        if case["train"]:
            st["go"], st["gh"] = randn(B, L, C), randn(B, C, dtype=torch.float32)
        return st
    if case["kind"] == "group":
        B, N, C = case["B"], case["N"], case["C"]
        # channels of different mean and width, as a convolution leaves them
        st["x"] = randn(B, N, C).mul_(0.5 + torch.rand(C, generator=g, device=dev).to(dtype))
        st["x"] += randn(C)
        st["w"], st["b"] = 1 + 0.1 * randn(C), 0.1 * randn(C)
        if case["train"]:
            st["go"] = randn(B, N, C)
        return st
    sizes = _sizes(case)
    total = BLOCK * sum(_blocks(sizes))
    # weights and moments of layers differ by orders of magnitude, gradients too
    st["p"] = randn(total, dtype=torch.float32).mul_(0.05)
    st["params"] = _parts(st["p"], sizes)
    width = [10.0 ** -(i % 4) for i in range(len(sizes))]
    st["grads"] = [randn(n).mul_(w) for n, w in zip(sizes, width)]
    # (no value between two tensors)
    m, v = torch.zeros(2, total, device=dev)
    [part.copy_(randn(n, dtype=torch.float32).mul_(0.3 * w))
     for part, n, w in zip(_parts(m, sizes), sizes, width)]
    [part.copy_(randn(n, dtype=torch.float32).square_().mul_(0.5).add_(0.01).mul_(w * w))
     for part, n, w in zip(_parts(v, sizes), sizes, width)]
    st["max_norm"] = 0.3 * math.sqrt(sum(n * w * w for n, w in zip(sizes, width)))
    if case["bits"] == 32:
        st["m"], st["v"] = m, v
        st["ms"], st["vs"] = _parts(m, sizes), _parts(v, sizes)
        return st
    for name, x, low, signed in (("m", m, -14, True), ("v", v, -30, False)):
        st[name], st[name + "_scale"] = _encode(x, torch.full_like(x, 32767, dtype=torch.int64), low,
                                                signed)
        st[name + "s"] = _parts(st[name], sizes)
        st[name + "_scales"] = list(st[name + "_scale"].split(_blocks(sizes)))
    return st


# ---- the plain forms ----------------------------------------------------------------------

def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along axis 1, from zero: spans of twice the length in each round."""
    span, L = 1, a.shape[1]
    while span < L:
        u = torch.cat((u[:, :span], torch.addcmul(u[:, span:], a[:, span:], u[:, :-span])), 1)
        a = torch.cat((a[:, :span], a[:, span:] * a[:, :-span]), 1)
        span *= 2
    return u


def _plain_recur(st):
    case, train = st["case"], st["case"]["train"]
    B, L, C = case["B"], case["L"], case["C"]
    v, f = st["v"].float(), st["f"].float()
    dtype, dev = st["v"].dtype, v.device
    there = None
    if st["lengths"] is not None:
        there = (torch.arange(L, device=dev) < st["lengths"][:, None])[:, :, None]
    a, away = torch.sigmoid(f), torch.sigmoid(-f)  # 1 - a without its cancellation
    u = away * v
    if there is not None:  # a token that is not in use leaves the state as it is
        a_used, u = torch.where(there, a, 1.0), torch.where(there, u, 0.0)
    else:
        a_used = a
    first = st["h"] if st["h"] is not None else v.new_zeros(B, C)
    # in the order of the steps, the initial state standing in front of them
    a_t, u_t = (a_used.flip(1), u.flip(1)) if case["reverse"] else (a_used, u)
    h = _scan(torch.cat((a_t[:, :1], a_t), 1), torch.cat((first[:, None], u_t), 1))
    before, h = h[:, :-1], h[:, 1:]
    final = h[:, -1].contiguous()
    if case["reverse"]:
        before, h = before.flip(1), h.flip(1)
    if st["g"] is not None:
        z = st["g"].float()
        sz = torch.sigmoid(z)
        out = h * (z * sz)
    else:
        out = h
    if there is not None:
        out = torch.where(there, out, 0.0)
    if not train:
        return [out.to(dtype), final]
    go = st["go"].float()
    d = go * (z * sz) if st["g"] is not None else go
    if there is not None:
        d = torch.where(there, d, 0.0)
    # the same scan from the last step to the first, each step taking the factor of the one behind it
    d_t, a_t = (d, a_used) if case["reverse"] else (d.flip(1), a_used.flip(1))
    d_t = _scan(torch.cat((a_t[:, :1], a_t[:, :1], a_t[:, :-1]), 1).clone().index_fill_(
        1, torch.tensor([1], device=dev), 1.0), torch.cat((st["gh"][:, None], d_t), 1))[:, 1:]
    g_first = a_t[:, -1] * d_t[:, -1]
    d = d_t if case["reverse"] else d_t.flip(1)
    gv, gf = d * away, d * (before - v) * (a * away)
    grads = [gv, gf]
    if st["g"] is not None:
        grads.append(go * h * (sz * (1 + z * (1 - sz))))
    if there is not None:
        grads = [torch.where(there, t, 0.0) for t in grads]
    return [out.to(dtype), final] + [t.to(dtype) for t in grads] + [g_first]


def _act(u, name):
    if name == "silu":
        return u * torch.sigmoid(u)
    if name == "gelu":
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    return u


def _act_slope(u, name):
    if name == "silu":
        s = torch.sigmoid(u)
        return s * (1 + u * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    return torch.ones_like(u)


def _plain_group(st):
    case = st["case"]
    B, N, C, G = (case[n] for n in ("B", "N", "C", "groups"))
    x, dtype = st["x"].float().view(B, N, G, C // G), st["x"].dtype
    w, b = st["w"].float().view(G, C // G), st["b"].float().view(G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    away = x - mean
    r = torch.rsqrt((away * away).mean((1, 3), keepdim=True) + 1e-5)
    hat = away * r
    u = hat * w + b
    y = _act(u, case["activation"]).view(B, N, C).to(dtype)
    if not case["train"]:
        return [y]
    g = st["go"].float().view(B, N, G, C // G) * _act_slope(u, case["activation"])
    gw, gb = (g * hat).sum((0, 1)).view(C), g.sum((0, 1)).view(C)
    g = g * w
    gx = r * (g - g.mean((1, 3), keepdim=True) - hat * (g * hat).mean((1, 3), keepdim=True))
    return [y, gx.view(B, N, C).to(dtype), gw.to(dtype), gb.to(dtype)]


def _plain_step(p, g, m, v, factor):
    """The new moments, in 32 bits; p is changed."""
    g = g.float() if factor is None else g.float() * factor
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    root = v.sqrt() * (1 / math.sqrt(1 - BETA2 ** STEP)) + EPS
    p.copy_(p * (1 - RATE * DECAY) - (RATE / (1 - BETA1 ** STEP)) * (m / root))
    return m, v


def _plain_step_8(p, g, m, v, m_scale, v_scale, factor, first):
    """The moments in use are changed, codes and scales."""
    new_m, new_v = _plain_step(p, g, _decode(m, m_scale, -14, True),
                               _decode(v, v_scale, -30, False), factor)
    words = _words(first, p.numel(), p.device)
    code, scale = _encode(new_m, words & 0xFFFF, -14, True)
    m.copy_(code), m_scale.copy_(scale)
    code, scale = _encode(new_v, words >> 16, -30, False)
    v.copy_(code), v_scale.copy_(scale)


def _plain_adamw(st):
    case, norm, factor = st["case"], None, None
    if case["clipped"]:
        norm = torch.stack([g.double().square().sum() for g in st["grads"]]).sum().sqrt().float()
        factor = (st["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
    if case["bits"] == 32:
        new = [_plain_step(p, g, m, v, factor) for p, g, m, v in
               zip(st["params"], st["grads"], st["ms"], st["vs"])]
        [m.copy_(a) for m, (a, _) in zip(st["ms"], new)]
        [v.copy_(a) for v, (_, a) in zip(st["vs"], new)]
        out = [st["p"], st["m"], st["v"]]
    else:
        blocks = _blocks(_sizes(case))
        firsts = [BLOCK * sum(blocks[:i]) for i in range(len(blocks))]
        [_plain_step_8(*of) for of in
         zip(st["params"], st["grads"], st["ms"], st["vs"], st["m_scales"], st["v_scales"],
             [factor] * len(blocks), firsts)]
        out = [st["p"], _decode(st["m"], st["m_scale"], -14, True).bfloat16(),
               _decode(st["v"], st["v_scale"], -30, False).bfloat16()]
    return out if norm is None else out + [norm]


# ---- one pass -----------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if not own:
        return {"recur": _plain_recur, "group": _plain_group, "adamw": _plain_adamw}[case["kind"]](st)
    from mappedconvolutions_amd import _C
    train = case.get("train")
    if case["kind"] == "recur":
        args = dict(lengths=st["lengths"], reverse=case["reverse"])
        out, final, saved = _C.gated_recurrence_forward(st["v"], st["f"], st["g"], initial=st["h"],
                                                        for_backward=train, **args)
        if not train:
            return [out, final]
        gv, gf, gg, gi = _C.gated_recurrence_backward(st["go"], st["v"], st["f"], st["g"], saved,
                                                      grad_final=st["gh"], **args)
        return [out, final, gv, gf] + ([gg] if case["gated"] else []) + [gi]
    if case["kind"] == "group":
        args = (case["groups"], st["w"], st["b"])
        y, saved = _C.group_norm_forward(st["x"], *args, activation=case["activation"],
                                         for_backward=train)
        if not train:
            return [y]
        return [y] + _C.group_norm_backward(st["go"], st["x"], saved, *args,
                                            activation=case["activation"])
    norm = _C.grad_norm(st["grads"]) if case["clipped"] else None
    more = dict(betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, grad_norm=norm,
                max_norm=st["max_norm"] if case["clipped"] else None)
    if case["bits"] == 32:
        _C.adamw_step(st["params"], st["grads"], st["ms"], st["vs"], STEP, RATE, **more)
        out = [st["p"], st["m"], st["v"]]
    else:
        _C.adamw_step(st["params"], st["grads"], st["ms"], st["vs"], STEP, RATE,
                      first_scales=st["m_scales"], second_scales=st["v_scales"], seed=SEED, **more)
        out = [st["p"], _C.adamw_moment(st["m"], st["m_scale"], second=False, dtype=torch.bfloat16),
               _C.adamw_moment(st["v"], st["v_scale"], second=True, dtype=torch.bfloat16)]
    return out if norm is None else out + [norm]


# ---- in 64 bits, from the definition ------------------------------------------------------

def _exact_recur(case, st):
    B, L, C = case["B"], case["L"], case["C"]
    # time first, so that a step's values lie together
    v, f = (st[n].double().transpose(0, 1).contiguous() for n in ("v", "f"))
    z = st["g"].double().transpose(0, 1).contiguous() if case["gated"] else None
    dev = v.device
    used = torch.tensor(_lengths(case), device=dev)
    live = (torch.arange(L, device=dev)[:, None] < used)[:, :, None].double()
    keep = 1 / (1 + torch.exp(-f))
    take = 1 / (1 + torch.exp(f))
    keep_used = keep * live + (1 - live)
    states = torch.zeros(L, B, C, dtype=torch.float64, device=dev)  # after each step
    prior = torch.zeros_like(states)
    given = take * v * live
    state = st["h"].double() if case["carried"] else torch.zeros(B, C, dtype=torch.float64, device=dev)
    order = range(L - 1, -1, -1) if case["reverse"] else range(L)
    for t in order:
        prior[t] = state
        torch.addcmul(given[t], keep_used[t], state, out=states[t])
        state = states[t]
    final = state.clone()
    open_ = z / (1 + torch.exp(-z)) if case["gated"] else torch.ones_like(v)

    def back(t):
        return t.transpose(0, 1).contiguous()

    out = [back(states * open_ * live), final]
    if not case["train"]:
        return out
    go = st["go"].double().transpose(0, 1).contiguous() * live
    pull = go * open_
    push = st["gh"].double()
    reach = torch.zeros_like(states)
    for t in reversed(order):
        torch.add(pull[t], push, out=reach[t])
        push = keep_used[t] * reach[t]
    reach = reach * live
    out += [back(reach * take), back(reach * (prior - v) * keep * take)]
    if case["gated"]:
        s = 1 / (1 + torch.exp(-z))
        out.append(back(go * states * (s + z * s * (1 - s))))
    return out + [push]


def _exact_group(case, st):
    B, C, G = case["B"], case["C"], case["groups"]
    y, gx = [], []
    w, b = st["w"].double().requires_grad_(), st["b"].double().requires_grad_()
    gw, gb = torch.zeros_like(w), torch.zeros_like(b)
    for i in range(B):
        x = st["x"][i].double().requires_grad_()
        # channels of a group as rows
        rows = x.t().reshape(G, -1)
        n = (rows - rows.mean(1, keepdim=True)) / torch.sqrt(rows.var(1, unbiased=False, keepdim=True) + 1e-5)
        u = n.reshape(C, -1).t() * w + b
        if case["activation"] == "silu":
            u = u / (1 + torch.exp(-u))
        elif case["activation"] == "gelu":
            u = u * torch.special.ndtr(u)
        y.append(u.detach())
        if case["train"]:
            d = torch.autograd.grad(u, (x, w, b), st["go"][i].double())
            gx.append(d[0])
            gw, gb = gw + d[1], gb + d[2]
    if not case["train"]:
        return [torch.stack(y)]
    return [torch.stack(y), torch.stack(gx), gw.detach(), gb.detach()]


def _exact_small(x, random, low, signed, dev):
    """What a tensor's values are held as: steps of an eighth of each value's power of two."""
    n = x.numel()
    size = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK)).view(-1, BLOCK)
    top = size.amax(1, keepdim=True)
    unit = torch.where(top > 0, 2.0 ** (torch.floor(torch.log2(top.clamp_min(1e-300))) + 1), 1.0)
    y = (size / unit).view(-1)[:n]
    step = 2.0 ** (torch.floor(torch.log2(y.clamp_min(2.0 ** low))) - 3)
    count = torch.floor(y / step + (random.double() + 0.5) / 65536)
    if not signed:
        count = torch.where(y > 0, count.clamp_min(1), count)
    held = torch.nn.functional.pad(count * step, (0, -n % BLOCK)).view(-1, BLOCK) * unit
    return held.view(-1)[:n] * torch.sign(x)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "recur":
        return _exact_recur(case, st)
    if case["kind"] == "group":
        return _exact_group(case, st)
    sizes, dev = _sizes(case), st["p"].device
    wide, norm, factor = st["p"].double(), None, 1.0
    if case["clipped"]:
        norm = math.sqrt(sum(g.double().square().sum().item() for g in st["grads"]))
        factor = min(1.0, st["max_norm"] / (norm + 1e-6))
    whole = [wide, torch.zeros_like(wide), torch.zeros_like(wide)]
    if case["bits"] == 32:
        whole[1].copy_(st["m"]), whole[2].copy_(st["v"])
    else:
        # the values of the codes by a table
        code = torch.arange(256, dtype=torch.float64, device=dev)
        e, part = torch.floor(code / 8), code % 8
        second = torch.where(e > 0, (8 + part) * 2.0 ** (e - 34), part * 2.0 ** -33)
        e = torch.floor((code % 128) / 8)
        first = torch.where(e > 0, (8 + part) * 2.0 ** (e - 18), part * 2.0 ** -17)
        first = torch.where(code < 128, first, -first)
        for to, table, name in ((whole[1], first, "m"), (whole[2], second, "v")):
            to.copy_((table[st[name].long()].view(-1, BLOCK) * st[name + "_scale"].double()[:, None]).view(-1))
    at = 0
    for n, p, g, m, v in zip(sizes, *[_parts(t, sizes) for t in whole[:1]], st["grads"],
                             *[_parts(t, sizes) for t in whole[1:]]):
        g = g.double() * factor
        m.lerp_(g, 1 - BETA1)
        v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
        p.mul_(1 - RATE * DECAY)
        p.sub_(RATE * (m / (1 - BETA1 ** STEP)) / (torch.sqrt(v / (1 - BETA2 ** STEP)) + EPS))
        if case["bits"] == 8:
            words = _words(at, n, dev)
            m.copy_(_exact_small(m, words & 0xFFFF, -14, True, dev))
            v.copy_(_exact_small(v, words >> 16, -30, False, dev))
        at += BLOCK * (-(-n // BLOCK))
    return whole if norm is None else whole + [torch.tensor(norm, dtype=torch.float64)]

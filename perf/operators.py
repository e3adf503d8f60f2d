"""The attention side of a network on panoramas, as measurable cases.

Three operators of `mappedconvolutions_amd._C`: the norm of queries and keys per head with the
position rotation in the same pass, attention with a learned bias by relative-position buckets,
and the clipping of a network's gradients by their global norm.  `run` calls them where `own` is
true and computes the same from elementary torch operations in 32 bits where it is not; `exact`
computes them in 64 bits.  `listed()` names the cases, `draw()` gives more of the same ranges.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}


def listed():
    return [
        # One new token of each of 8 sequences: the norm of a decoding step.
        dict(name="norm_one_token_bf16", kind="norm", dtype="bf16", B=8, L=1, Hq=16, Hk=4, D=64,
             rotated=64, adjacent=False, ids=True, train=False),
        # Training over the rows of eight 256 x 512 panoramas with 128 channels, the queries and
        # keys being parts of one packed projection.
        dict(name="norm_rows_train_bf16", kind="norm", dtype="bf16", B=2048, L=512, Hq=4, Hk=4,
             D=32, rotated=32, adjacent=False, ids=False, train=True),
        # All pixels of a 125 x 250 image, shared key heads, an unusual head size of which a part
        # is rotated, in single precision.
        dict(name="norm_odd_train_fp32", kind="norm", dtype="fp32", B=3, L=31250, Hq=6, Hk=2, D=48,
             rotated=32, adjacent=True, ids=False, train=True),
        # Training over the rows of two panoramas: 512 sequences of 512 columns that close on
        # themselves.
        dict(name="attention_rows_train_bf16", kind="attention", dtype="bf16", B=512, Lq=512,
             Lk=512, Hq=8, Hk=8, D=64, causal=False, ragged=False, buckets=32, reach=0,
             train=True),
        # The largest: training over the 64 x 128 tokens of an image in scan order.
        dict(name="attention_scan_train_bf16", kind="attention", dtype="bf16", B=1, Lq=8192,
             Lk=8192, Hq=16, Hk=4, D=128, causal=False, ragged=False, buckets=64, reach=2048,
             train=True),
        # Sequences of different lengths in single precision, causal, three query heads a key
        # head, an unusual head size.
        dict(name="attention_odd_train_fp32", kind="attention", dtype="fp32", B=2, Lq=1250,
             Lk=1250, Hq=6, Hk=2, D=48, causal=True, ragged=True, buckets=32, reach=128,
             train=True),
        # Prompts of up to 2562 tokens before decoding starts: causal, no gradients.
        dict(name="attention_prompt_bf16", kind="attention", dtype="bf16", B=4, Lq=2562, Lk=2562,
             Hq=16, Hk=4, D=64, causal=True, ragged=True, buckets=32, reach=128, train=False),
        # One token against a short cache: what counts is latency.
        dict(name="decode_small_bf16", kind="attention", dtype="bf16", B=1, Lq=1, Lk=1000, Hq=8,
             Hk=8, D=64, causal=True, ragged=False, buckets=32, reach=128, train=False),
        # A serving batch: 64 sequences, each of its own length, in caches of 8192 places.
        dict(name="decode_batch_bf16", kind="attention", dtype="bf16", B=64, Lq=1, Lk=8192, Hq=32,
             Hk=8, D=128, causal=True, ragged=True, buckets=32, reach=128, train=False),
        # Two long caches in single precision, eight query heads a key head: few rows, long sums.
        dict(name="decode_long_fp32", kind="attention", dtype="fp32", B=2, Lq=1, Lk=100001, Hq=16,
             Hk=2, D=64, causal=True, ragged=False, buckets=64, reach=512, train=False),
        # The gradients of a small encoder: a few dozen weights and biases.
        dict(name="clip_encoder_fp32", kind="clip", dtype="fp32", tensors=30, largest=147456,
             spread=2304, clipped=True),
        # The gradients of a large network, many sizes, over half a billion values in all.
        dict(name="clip_large_bf16", kind="clip", dtype="bf16", tensors=300, largest=8388608,
             spread=64, clipped=True),
    ]


def _log(rng, low, high):
    """A whole number between low and high, uniform in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("norm", "train", "prompt", "decode", "clip"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    Hk = rng.choice((1, 2, 4, 8))
    Hq = Hk * rng.choice((1, 2, 3, 4, 8))
    D = rng.choice((16, 32, 40, 48, 64, 80, 96, 128))
    buckets = rng.choice((16, 32, 48, 64, 128))
    if kind == "norm":
        L = _log(rng, 1, 40000)
        rows = _log(rng, 1, 268000000 // (2 * (Hq + Hk) * D))
        return dict(kind="norm", dtype=dtype, B=max(1, rows // L), L=L, Hq=Hq, Hk=Hk, D=D,
                    rotated=rng.choice((D, D // 2)), adjacent=rng.choice((True, False)),
                    ids=rng.choice((True, False)), train=rng.choice((True, True, False)))
    if kind == "clip":
        return dict(kind="clip", dtype=dtype, tensors=_log(rng, 1, 300),
                    largest=_log(rng, 1000, 8000000), spread=_log(rng, 1, 1000),
                    clipped=rng.choice((True, True, False)))
    if kind == "decode":
        Lk = _log(rng, 1, 100000)
        room = 500000000 // (Lk * Hk * D)
        return dict(kind="attention", dtype=dtype, B=_log(rng, 1, max(1, min(64, room))),
                    Lq=rng.choice((1, 1, 1, 2, 5)), Lk=Lk, Hq=Hq, Hk=Hk, D=D, causal=True,
                    ragged=rng.choice((True, False)), buckets=buckets,
                    reach=rng.choice((64, 128, 512)), train=False)
    train = kind == "train"
    Lk = _log(rng, 16, 4000)
    Lq = Lk if rng.random() < 0.7 else _log(rng, 16, 4000)
    pairs = 500000000 if dtype == "bf16" else 100000000  # fp32 costs several times as much
    B = _log(rng, 1, max(1, min(256, pairs // (Hq * Lq * Lk))))
    causal = rng.choice((True, False))
    return dict(kind="attention", dtype=dtype, B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hk=Hk, D=D, causal=causal,
                ragged=rng.choice((True, False)), buckets=buckets,
                reach=rng.choice((0, 64, 128, 512)), train=train)


def _lengths(case):
    """Keys in use of every sequence: all of them, or from a half to all (in decoding, where the
    cache's unused places lie behind)."""
    B, Lk = case["B"], case["Lk"]
    if not case["ragged"]:
        return [Lk] * B
    return [max(1, Lk - (i * 7919 % max(1, B)) * Lk // (2 * B)) for i in range(B)]


def _pairs(case):
    """Pairs of a query and a key that take part, over all heads."""
    n = 0
    for length in _lengths(case):
        if not case["causal"]:
            n += case["Lq"] * length
            continue
        start = length - case["Lq"] if case["Lq"] <= 8 else 0
        first, last = start + 1, start + case["Lq"]  # keys that the first and last query see
        below = max(0, min(last, length) - max(first, 1) + 1)
        lo = max(first, 1)
        n += below * (2 * lo + below - 1) // 2 + length * max(0, last - max(length, first - 1))
    return n * case["Hq"]


def _clip_sizes(case):
    """Sizes of the tensors: from `largest` down to `largest / spread`, odd ones among them."""
    n, top, spread = case["tensors"], case["largest"], case["spread"]
    sizes = []
    for i in range(n):
        part = (i * 0.6180339887) % 1.0
        size = int(top * math.exp(-part * math.log(spread)) if spread > 1 else top)
        sizes.append(max(1, size if i % 3 else size | 1))
    return sizes


def _parts(flat, sizes):
    """The part of every tensor in the buffer of all."""
    padded = flat.split([-(-n // 64) * 64 for n in sizes])
    return [part[:n] for part, n in zip(padded, sizes)]


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "clip":
        n = sum(_clip_sizes(case))
        return {"bytes": 2 * n * size, "flops": 3 * n}
    if case["kind"] == "norm":
        rows = case["B"] * case["L"]
        n = rows * (case["Hq"] + case["Hk"]) * case["D"]
        table = 2 * 4 * (case["B"] * case["L"] if case["ids"] else case["L"]) * case["rotated"] // 2
        passes = (2 + 3) if case["train"] else 2
        return {"bytes": passes * n * size + table, "flops": (8 + 16) * n if case["train"] else 8 * n}
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    rows, keys = case["B"] * case["Lq"] * Hq, sum(_lengths(case)) * Hk
    nbytes = (2 * rows + 2 * keys) * D * size
    if case["train"]:
        nbytes += (2 * rows + 2 * case["B"] * case["Lk"] * Hk) * D * size
    return {"bytes": nbytes, "flops": _pairs(case) * D * (12 if case["train"] else 4)}


def _distance_buckets(count, reach, length, device):
    """Bucket of every relative position from -(reach) to reach: near ones have their own, far ones
    share by the logarithm of the distance, each sign its half.  reach 0: the positions lie on a
    circle of `length`, and the distance is the shorter way round."""
    circle = reach == 0
    span = length - 1 if circle else reach
    r = torch.arange(-span, span + 1, dtype=torch.float64)
    away = r.abs()
    if circle:
        away = torch.minimum(away, length - away)
        side = ((r % length) * 2 > length).long()
    else:
        side = (r > 0).long()
    half = count // 2
    near = half // 2
    top = max(near + 1, length // 2 if circle else reach)
    far = near + (torch.log(away.clamp_min(1) / near) / math.log(top / near) * (half - near))
    bucket = torch.where(away < near, away, far.clamp(near, half - 1)).floor().long()
    return (bucket + side * half).to(torch.int32).to(device), span


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    st = dict(case=case)
    if case["kind"] == "clip":
        # gradients of layers differ by orders of magnitude
        sizes = _clip_sizes(case)
        st["grads"] = [randn(n).mul_(10.0 ** -(i % 4)) for i, n in enumerate(sizes)]
        # the clipped values go to one buffer, every tensor's part on a boundary of 64 values
        st["flat"] = torch.zeros(sum(-(-n // 64) * 64 for n in sizes), device=dev, dtype=dtype)
        st["out"] = _parts(st["flat"], sizes)
        expected = math.sqrt(sum(n * 100.0 ** -(i % 4) for i, n in enumerate(sizes)))
        st["max_norm"] = expected * (0.3 if case["clipped"] else 4.0)
        return st
    B, Hq, Hk, D = case["B"], case["Hq"], case["Hk"], case["D"]
    if case["kind"] == "norm":
        L, F = case["L"], case["rotated"] // 2
        packed = randn(B, L, Hq + 2 * Hk, D)
        st["q"], st["k"] = packed[:, :, :Hq], packed[:, :, Hq:Hq + Hk]
        st["qw"], st["kw"] = 1 + 0.1 * randn(D), 1 + 0.1 * randn(D)
        places = 4096 if case["ids"] else L
        turn = torch.arange(places, device=dev, dtype=torch.float64)[:, None] * (
            1000.0 ** -(torch.arange(F, device=dev, dtype=torch.float64) / max(F, 1)))[None]
        st["cos"], st["sin"] = turn.cos().float(), turn.sin().float()
        st["ids"] = torch.randint(0, places, (B, L), generator=g, device=dev) if case["ids"] else None
        if case["train"]:
            st["gq"], st["gk"] = randn(B, L, Hq, D), randn(B, L, Hk, D)
        return st
    Lq, Lk = case["Lq"], case["Lk"]
    # queries and keys as after a norm per head, the values a part of a packed projection
    st["q"], st["k"] = randn(B, Lq, Hq, D), randn(B, Lk, Hk, D)
    if Lq == Lk and case["train"]:
        st["v"] = randn(B, Lk, Hq + 2 * Hk, D)[:, :, Hq + Hk:]
    else:
        st["v"] = randn(B, Lk, Hk, D)
    st["table"] = randn(Hq, case["buckets"])
    st["buckets"], st["zero"] = _distance_buckets(case["buckets"], case["reach"], max(Lq, Lk), dev)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    st["lengths"] = lengths if case["ragged"] else None
    # a few queries are the last of their sequence, many its first
    st["start"] = lengths - Lq if case["causal"] and Lq <= 8 else None
    if case["train"]:
        st["go"] = randn(B, Lq, Hq, D)
    return st


# ---- the plain forms ----------------------------------------------------------------------

def _turn(n, cos, sin, rotated, adjacent):
    """The rotation of the first `rotated` values of the last axis."""
    head, tail = n[..., :rotated], n[..., rotated:]
    F = rotated // 2
    if adjacent:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head[..., :F], head[..., F:]
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((head, tail), -1)


def _plain_norm(x, w, g, st):
    """(y, None, None), or with g the gradients (y, dx, dw)."""
    case = st["case"]
    cos, sin = st["cos"], st["sin"]
    if st["ids"] is not None:
        cos, sin = cos[st["ids"]], sin[st["ids"]]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)  # over the heads
    dtype, x, w = x.dtype, x.float(), w.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    y = _turn(x * r * w, cos, sin, case["rotated"], case["adjacent"]).to(dtype)
    if g is None:
        return y, None, None
    dn = _turn(g.float(), cos, -sin, case["rotated"], case["adjacent"])
    dw = (dn * x * r).sum((0, 1, 2))
    u = dn * w
    dx = r * (u - x * (r * r) * (u * x).mean(-1, keepdim=True))
    return y, dx.to(dtype), dw.to(dtype)


def _plain_attention(st):
    case = st["case"]
    B, Lq, Lk, Hq, Hk, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    G, scale, dtype = Hq // Hk, D ** -0.5, st["q"].dtype
    dev = st["q"].device
    q = st["q"].float().view(B, Lq, Hk, G, D).permute(0, 2, 3, 1, 4)           # B Hk G Lq D
    q = q.reshape(B, Hk, G * Lq, D)
    k = st["k"].float().permute(0, 2, 1, 3).contiguous()                       # B Hk Lk D
    v = st["v"].float().permute(0, 2, 1, 3).contiguous()
    i, j = torch.arange(Lq, device=dev), torch.arange(Lk, device=dev)
    start = st["start"].long() if st["start"] is not None else torch.zeros(1, device=dev).long()
    rel = j[None, None, :] - (start[:, None, None] + i[None, :, None])         # 1 or B, Lq, Lk
    which = (rel + st["zero"]).clamp_(0, st["buckets"].numel() - 1)
    bias = st["table"].float()[:, st["buckets"].long()[which]]                 # Hq, 1 or B, Lq, Lk
    bias = bias.transpose(0, 1).reshape(-1, Hk, G, Lq, Lk)
    s = torch.matmul(q, k.transpose(-1, -2)).view(B, Hk, G, Lq, Lk)
    s = s.mul_(scale).add_(bias)
    if case["causal"]:
        s = s.masked_fill_((rel > 0)[:, None, None], -math.inf)
    if st["lengths"] is not None:
        s = s.masked_fill_((j >= st["lengths"][:, None])[:, None, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total)).view(B, Hk, G * Lq, Lk)
    o = torch.matmul(p, v)

    def heads_last(t):
        return t.view(B, Hk, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D).to(dtype)

    if not case["train"]:
        return heads_last(o)
    go = st["go"].float().view(B, Lq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, D)
    dv = torch.matmul(p.transpose(-1, -2), go)
    ds = torch.matmul(go, v.transpose(-1, -2))
    ds = ds.sub_((go * o).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    # the bias is shared by the batch, then by all pairs of one difference j - i, then by bucket:
    # rows padded to Lq + Lk values and read again one value shorter put a difference in a column
    per_pair = ds.view(B, Hq, Lq, Lk).sum(0).flip(1)                           # row Lq - 1 - i
    wide = torch.cat((per_pair, per_pair.new_zeros(Hq, Lq, Lq)), -1).view(Hq, -1)
    width = Lq + Lk - 1
    per_rel = wide[:, :Lq * width].view(Hq, Lq, width).sum(1)                  # column j - i + Lq - 1
    at = (torch.arange(width, device=dev) - (Lq - 1) + st["zero"]).clamp_(0, st["buckets"].numel() - 1)
    one_hot = st["buckets"].long()[at][:, None] == torch.arange(case["buckets"], device=dev)[None]
    dtable = torch.matmul(per_rel, one_hot.float())
    back = [t.permute(0, 2, 1, 3).contiguous().to(dtype) for t in (dk, dv)]
    return heads_last(o), heads_last(dq), back[0], back[1], dtable.to(dtype)


def _plain_clip(st):
    grads = [t.float() for t in st["grads"]]
    norm = torch.stack([(t * t).sum() for t in grads]).sum().sqrt()
    factor = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(t * factor) for o, t in zip(st["out"], grads)]
    return [norm, st["flat"]]


# ---- one pass -----------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if not own:
        if case["kind"] == "clip":
            return _plain_clip(st)
        if case["kind"] == "attention":
            return _plain_attention(st)
        q = _plain_norm(st["q"], st["qw"], st.get("gq"), st)
        k = _plain_norm(st["k"], st["kw"], st.get("gk"), st)
        return [q[0], k[0]] + ([q[1], k[1], q[2], k[2]] if case["train"] else [])
    from mappedconvolutions_amd import _C
    if case["kind"] == "clip":
        return [_C.clip_grad_norm(st["grads"], st["max_norm"], out=st["out"]), st["flat"]]
    if case["kind"] == "norm":
        args = (st["q"], st["k"], st["qw"], st["kw"], st["cos"], st["sin"], st["ids"], 1e-6,
                case["adjacent"])
        out = _C.qk_norm_rotate_forward(*args)
        if case["train"]:
            out = out + _C.qk_norm_rotate_backward(st["gq"], st["gk"], *args)
        return out
    args = dict(bias_table=st["table"], buckets=st["buckets"], bucket_zero=st["zero"],
                causal=case["causal"], query_start=st["start"], key_lengths=st["lengths"])
    q, k, v = st["q"], st["k"], st["v"]
    out, lse = _C.relative_attention_forward(q, k, v, for_backward=case["train"], **args)
    if not case["train"]:
        return out
    return [out] + _C.relative_attention_backward(st["go"], q, k, v, out, lse, **args)


# ---- in 64 bits, from the definition ------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "clip":
        flat = torch.cat([t.double().view(-1) for t in st["grads"]])
        norm = torch.linalg.vector_norm(flat)
        factor = min(1.0, st["max_norm"] / (norm.item() + 1e-6))
        whole = st["flat"].double()
        for o, t in zip(_parts(whole, _clip_sizes(case)), st["grads"]):
            o.copy_(t.double() * factor)
        return [norm, whole]
    if case["kind"] == "norm":
        first, grads = [], []
        for x, w, g in ((st["q"], st["qw"], st.get("gq")), (st["k"], st["kw"], st.get("gk"))):
            x = x.double().requires_grad_(case["train"])
            w = w.double().requires_grad_(case["train"])
            n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
            cos, sin = st["cos"].double(), st["sin"].double()
            if st["ids"] is not None:
                cos, sin = cos[st["ids"]], sin[st["ids"]]
            # the pairs as complex numbers, turned by cos + i sin
            R = case["rotated"]
            order = torch.arange(R, device=x.device)
            if not case["adjacent"]:
                order = order.view(2, R // 2).t().reshape(-1)
            pairs = torch.view_as_complex(n[..., order].unflatten(-1, (R // 2, 2)).contiguous())
            turned = torch.view_as_real(pairs * torch.complex(cos, sin).unsqueeze(-2)).flatten(-2)
            back = torch.argsort(order)
            y = torch.cat((turned[..., back], n[..., R:]), -1)
            first.append(y.detach())
            if case["train"]:
                grads.append(torch.autograd.grad(y, (x, w), g.double()))
        if case["train"]:
            first += [grads[0][0], grads[1][0], grads[0][1], grads[1][1]]
        return first
    B, Lq, Lk, Hq, Hk, D = (case[n] for n in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    train, dev = case["train"], st["q"].device
    leaf = [st[n].double().requires_grad_(train) for n in ("q", "k", "v", "table")]
    q, k, v, table = leaf
    sums = [torch.zeros_like(t) for t in leaf]
    outs = torch.zeros(B, Lq, Hq, D, dtype=torch.float64, device=dev)
    step = max(1, 100000000 // (Lq * Lk))
    for h in range(Hq):
        for b in range(0, B, step):
            rows = slice(b, min(B, b + step))
            n = rows.stop - rows.start
            at = torch.zeros(n, device=dev).long() if st["start"] is None else st["start"][rows].long()
            at = at[:, None] + torch.arange(Lq, device=dev)
            rel = torch.arange(Lk, device=dev) - at[:, :, None]
            which = st["buckets"][(rel + st["zero"]).clamp(0, len(st["buckets"]) - 1)].long()
            gone = rel > 0 if case["causal"] else torch.zeros_like(rel, dtype=torch.bool)
            if st["lengths"] is not None:
                gone = gone | (torch.arange(Lk, device=dev) >= st["lengths"][rows][:, None])[:, None]
            part = [t.detach().requires_grad_(train) for t in
                    (q[rows, :, h], k[rows, :, h // (Hq // Hk)], v[rows, :, h // (Hq // Hk)], table[h])]
            s = part[0] @ part[1].transpose(1, 2) / math.sqrt(D)
            s = s + part[3].index_select(0, which.view(-1)).view_as(s)
            p = torch.softmax(s.masked_fill(gone, -1e300), -1).masked_fill(gone, 0.0)
            o = p @ part[2]
            outs[rows, :, h] = o.detach()
            if train:
                d = torch.autograd.grad(o, part, st["go"][rows, :, h].double())
                sums[0][rows, :, h] += d[0]
                sums[1][rows, :, h // (Hq // Hk)] += d[1]
                sums[2][rows, :, h // (Hq // Hk)] += d[2]
                sums[3][h] += d[3]
            del s, p, o, rel, which, gone
    return [outs] + [t.detach() for t in sums] if train else outs

"""The AdamW step and its moments in 8 bits, in 64 bits on the CPU from the definition."""
import torch


def words(step, seed, first, count):
    """The random words of values first to first + count of the list (numbers below 2^32)."""
    def mix(x):
        x = x ^ (x >> 16)
        x = x * 0x6A09E667 % 2 ** 32
        x = x ^ (x >> 15)
        x = x * 0xBB67AE85 % 2 ** 32
        return x ^ (x >> 16)

    key = mix(mix(step % 2 ** 32) ^ (seed % 2 ** 32))
    at = torch.arange(first, first + count)
    return mix(((at % 2 ** 32 ^ (at >> 32) * 0x9E3779B1 % 2 ** 32) + key) % 2 ** 32)


def blocks(n):
    return -(-n // 256)


def per_block(x):
    """[blocks, 256], zeros behind the end."""
    return torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)


def decode(code, scale, second):
    low, c = (-30, code.double()) if second else (-14, (code % 128).double())
    e, part = torch.floor(c / 8), c % 8
    y = torch.where(e > 0, (8 + part) * 2 ** (e + low - 4), part * 2.0 ** (low - 3))
    if not second:
        y = torch.where(code >= 128, -y, y)
    return (per_block(y) * scale.double()[:, None]).view(-1)[:code.numel()]


def held(x, chance, second):
    """(what is held of float64 values x, the step of each, how far each is from being rounded the
    other way, in steps, how far its block's largest value is from a power of two, at which the scale
    doubles, over that value); `chance`: numbers below 2^16."""
    low, n = (-30 if second else -14), x.numel()
    top = per_block(x.abs()).amax(1, keepdim=True)
    scale = torch.where(top > 0, 2 ** (torch.floor(torch.log2(top.clamp_min(1e-300))) + 1), 1.0)
    y = (per_block(x.abs()) / scale).view(-1)[:n]
    step = 2 ** (torch.floor(torch.log2(y.clamp_min(2.0 ** low))) - 3)
    sum_ = y / step + (chance.double() + 0.5) / 65536
    count = torch.floor(sum_)
    near = (sum_ - torch.round(sum_)).abs()
    if second:
        count = torch.where(y > 0, count.clamp_min(1), count)

    def wide(t):
        return (per_block(t) * scale).view(-1)[:n]

    part = top / scale  # in [1/2, 1)
    edge = torch.where(top > 0, torch.minimum(part - 0.5, 1 - part) / part.clamp_min(0.5), 1.0)
    return (wide(count * step) * torch.sign(x), wide(step), near,
            edge.expand(-1, 256).reshape(-1)[:n])


def step(p, g, m, v, number, lr, betas=(0.9, 0.999), eps=1e-8, decay=0.0, factor=1.0):
    """(p, m, v, how much of p's change there is to round) of one tensor, in 64 bits."""
    b1, b2 = betas
    g = g.double().flatten() * factor
    new_m = b1 * m + (1 - b1) * g
    new_v = b2 * v + (1 - b2) * g * g
    root = torch.sqrt(new_v / (1 - b2 ** number)) + eps
    rate = lr / (1 - b1 ** number)
    size = (b1 * m.abs() + (1 - b1) * g.abs())
    return (p.double().flatten() * (1 - lr * decay) - rate * new_m / root, new_m, new_v,
            abs(rate) * size / root, size)

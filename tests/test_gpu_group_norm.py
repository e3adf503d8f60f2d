"""Group norm with an activation against float64.

Tolerances, u = 2^-24, s the width of a group, m its mean.  Means of up to 10^5 values in 32 bits: sums of
a few hundred values in a thread and its block, joined: 64 u of the largest value; the same of the
squares, so that n = (x - m) r is off by 64 u (|x| + |m|) r + 64 u |n|.  u = n w + b and the activation:
4 u, slopes at most 1.13, exp and erf 4 u: e = 1.2 |w| dn + 8 u (|u| + 1).  Gradients: g' carries the
second derivative's share (at most 0.8 |w| dn of gy) and 16 u; the sums over N tokens 64 u of the sum of
sizes.  bf16 outputs: 2^-8 of the value besides (half a step)."""
import math

import pytest
import torch

from mappedconvolutions_amd import _C

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def phi(u):
    return torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)


ACT = {None: lambda u: u, "silu": lambda u: u * torch.sigmoid(u), "gelu": lambda u: u * torch.special.ndtr(u)}
SLOPE = {None: torch.ones_like,
         "silu": lambda u: torch.sigmoid(u) * (1 + u * torch.sigmoid(-u)),
         "gelu": lambda u: torch.special.ndtr(u) + u * phi(u)}


def make(seed, B, N, C, dtype, mean=1.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, N, C, generator=g) * spread * (0.5 + torch.rand(C, generator=g)) + \
        mean * torch.randn(C, generator=g)
    return [t.to(dtype) for t in (x, 1 + 0.2 * torch.randn(C, generator=g),
                                  0.3 * torch.randn(C, generator=g), torch.randn(B, N, C, generator=g))]


def check(x, w, b, go, groups, activation, eps=1e-5, views=lambda t: t.cuda()):
    dtype, (B, N, C) = x.dtype, x.shape
    xc, gc = views(x), go.cuda()
    wc, bc = (None if t is None else t.cuda() for t in (w, b))
    y, saved = _C.group_norm_forward(xc, groups, wc, bc, eps, activation, for_backward=True)
    assert torch.equal(_C.group_norm_forward(xc, groups, wc, bc, eps, activation)[0], y)
    gx, gw, gb = _C.group_norm_backward(gc, xc, saved, groups, wc, bc, activation)
    assert y.dtype == gx.dtype == dtype and y.is_contiguous() and gx.is_contiguous()
    half = 2.0 ** -8 if dtype == BF16 else U

    def cut(t):
        return t.double().view(B, N, groups, C // groups)

    def whole(t):
        return torch.ones(groups, C // groups, dtype=torch.float64) if t is None else \
            t.double().view(groups, -1)

    X, G, W = cut(x), cut(go), whole(w)
    bias = torch.zeros_like(W) if b is None else whole(b)
    m = X.mean((1, 3), keepdim=True)
    var = (X - m).square().mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    n = (X - m) * r
    top = X.abs().amax((1, 3), keepdim=True)
    dn = 64 * U * (X.abs() + top) * r + 64 * U * n.abs()
    u = n * W + bias
    want = ACT[activation](u)
    e = 1.2 * W.abs() * dn + 8 * U * (u.abs() + 1) + half * want.abs()

    def close(got, want, bound, what):
        off = (got.double().cpu().view(want.shape) - want).abs()
        assert (off <= bound + 1e-30).all(), (what, (off / (bound + 1e-30)).max().item())

    close(y, want, e, "y")
    assert (saved[..., 0].double().cpu() - m[:, 0, :, 0]).abs().max() <= 64 * U * top.max()
    slope = SLOPE[activation](u)
    d = G * slope
    # (the slope of an activation that is none does not change)
    dd = G.abs() * ((0.8 * W.abs() * dn + 16 * U) if activation else 0 * dn)
    count = N * (C // groups)
    rough = 64 * U * math.sqrt(max(1, N * B) / 4096 + 1)
    s1, s2 = d.sum((0, 1)), (d * n).sum((0, 1))
    b1 = (dd + rough * d.abs()).sum((0, 1))
    b2 = ((dd + rough * d.abs()) * n.abs() + d.abs() * dn).sum((0, 1))
    if w is not None:
        close(gw, s2, b2 + half * s2.abs(), "gw")
    if b is not None:
        close(gb, s1, b1 + half * s1.abs(), "gb")
    wd = d * W
    m1, m2 = (t.sum((1, 3), keepdim=True) / count for t in (wd, wd * n))
    dm1 = ((dd + rough * d.abs()) * W.abs()).sum((1, 3), keepdim=True) / count
    dm2 = (((dd + rough * d.abs()) * n.abs() + d.abs() * dn) * W.abs()).sum((1, 3), keepdim=True) / count
    want = r * (wd - m1 - n * m2)
    part = wd.abs() + m1.abs() + (n * m2).abs()
    bound = r * (dd * W.abs() + dm1 + n.abs() * dm2 + dn * m2.abs() + 8 * U * part) + 64 * U * r * part + \
        half * want.abs()
    close(gx, want, bound, "gx")
    return y, gx, gw, gb


CASES = [  # B, N, C, groups
    (1, 1, 8, 2), (2, 1, 64, 8), (1, 7, 30, 6), (3, 50, 48, 16), (2, 100, 90, 6), (1, 1000, 64, 64),
    (2, 333, 24, 1), (1, 65, 512, 32), (2, 40, 2048, 2048), (1, 130, 2056, 8), (1, 20, 4096, 1),
    (1, 9, 4104, 3), (2, 17, 1001, 7), (1, 33, 6000, 6), (1, 5, 3, 3), (4, 8, 1, 1), (1, 4099, 6, 2),
    (300, 12, 16, 4), (1, 70001, 16, 4), (1, 12, 10008, 8), (2, 9, 8200, 8), (70000, 3, 8, 2),
    (1, 8192, 8, 1), (1, 8193, 8, 1), (2, 2048, 8, 8), (200, 300, 40, 5), (130, 1025, 24, 3)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", CASES)
def test_sizes(device, size, dtype):
    B, N, C, groups = size
    for activation in ACT:
        check(*make(1, B, N, C, dtype), groups, activation)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(130, 512, 64, 16), (40, 606, 128, 32), (70, 700, 96, 12), (129, 300, 72, 6),
                                  (65, 1023, 40, 20), (50, 257, 264, 33)])
def test_samples_held_in_parts(device, size, dtype):
    B, N, C, groups = size
    check(*make(12, B, N, C, dtype), groups, "silu")
    check(*make(13, B, N, C, dtype), groups, None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_weight_or_bias(device, dtype):
    x, w, b, go = make(2, 2, 40, 32, dtype)
    for W, b_ in ((None, None), (w, None), (None, b)):
        check(x, W, b_, go, 4, "silu")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(device, dtype):
    x, w, b, go = make(3, 3, 50, 48, dtype)

    def part_of(t, front, back):
        wide = torch.full((3, 50, front + 48 + back), 7.0, dtype=dtype, device="cuda")
        wide[..., front:front + 48] = t.cuda()
        return wide[..., front:front + 48]

    for front, back in ((16, 0), (8, 8), (2, 6), (1, 0), (0, 3)):
        check(x, w, b, go, 6, "silu", views=lambda t: part_of(t, front, back))
    # an image with its channels last, tokens of every second row, samples and tokens swapped, and an
    # input whose last axis is not dense
    check(x, w, b, go, 6, None, views=lambda t: t.cuda().view(3, 5, 10, 48).permute(0, 3, 1, 2)
          .contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1).flatten(1, 2))
    check(x, w, b, go, 6, None, views=lambda t: t.cuda().repeat_interleave(2, 1)[:, ::2])
    check(x, w, b, go, 6, None, views=lambda t: t.cuda().transpose(0, 1).contiguous().transpose(0, 1))
    check(x, w, b, go, 6, None, views=lambda t: t.cuda().transpose(1, 2).contiguous().transpose(1, 2))
    check(x[:1].expand(3, 50, 48), w, b, go, 6, None, views=lambda t: t[:1].cuda().expand(3, 50, 48))


def test_a_mean_far_from_zero(device):
    # (squares of differences of values whose own squares differ in no bit)
    x, w, b, go = make(4, 2, 3000, 32, F32, mean=0.0)
    check(x + 4096.0, w, b, go, 4, None)
    # one token that differs from all others
    x[:, 5] += 1e4
    check(x, w, b, go, 4, None)


def test_what_does_not_vary(device):
    x = torch.full((2, 100, 16), 3.0)
    y, gx, gw, gb = check(x, None, None, torch.randn(2, 100, 16), 4, None)
    assert (y == 0).all()
    # a norm of one value is zero, and so is its gradient
    one, go = torch.randn(5, 1, 8), torch.randn(5, 1, 8)
    y, saved = _C.group_norm_forward(one.cuda(), 8, for_backward=True)
    gx = _C.group_norm_backward(go.cuda(), one.cuda(), saved, 8)[0]
    assert (y == 0).all() and (gx == 0).all()


def test_empty(device):
    w = torch.ones(8, device="cuda")
    for B, N in ((0, 5), (3, 0)):
        x = torch.zeros(B, N, 8, device="cuda")
        y, saved = _C.group_norm_forward(x, 2, w, w, for_backward=True)
        assert y.shape == (B, N, 8)
        gx, gw, gb = _C.group_norm_backward(y, x, saved, 2, w, w)
        assert gx.shape == (B, N, 8) and (gw == 0).all() and (gb == 0).all()


def test_what_is_no_number_stays_in_its_group(device):
    x, w, b, go = (t.cuda() for t in make(5, 2, 500, 32, F32))
    y0, _ = _C.group_norm_forward(x, 4, w, b)
    for bad in (float("nan"), float("inf")):
        x[1, 77, 9] = bad
        y, _ = _C.group_norm_forward(x, 4, w, b)
        assert torch.isnan(y[1, 77, 9]) and torch.isnan(y[1, :, 8:16]).all() or bad == float("inf")
        assert not torch.isfinite(y[1, 77, 9])
        assert torch.equal(y[0], y0[0])
        assert torch.equal(y[1, :, :8], y0[1, :, :8]) and torch.equal(y[1, :, 16:], y0[1, :, 16:])


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_values_of_the_activation(device, dtype, activation):
    # weights that take the norm far into both tails
    x, w, b, go = make(6, 1, 400, 16, dtype)
    y, gx, gw, gb = check(x, 60 * w, b, go, 4, activation)
    for t in (y, gx, gw, gb):
        assert torch.isfinite(t).all()


def test_gradients_that_are_not_wanted(device):
    x, w, b, go = (t.cuda() for t in make(7, 2, 60, 32, BF16))
    y, saved = _C.group_norm_forward(x, 8, w, b, for_backward=True)
    every = _C.group_norm_backward(go, x, saved, 8, w, b)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (True, False, True),
                  (False, False, False)):
        some = _C.group_norm_backward(go, x, saved, 8, w, b, needs=needs)
        for a, b_, wanted in zip(some, every, needs):
            assert torch.equal(a, b_) if wanted else a is None


def test_gradient_against_differences(device):
    x, w, b, go = make(8, 1, 20, 12, F32)
    xc, wc, bc = x.cuda(), w.cuda(), b.cuda()
    _, saved = _C.group_norm_forward(xc, 3, wc, bc, activation="silu", for_backward=True)
    gx, gw, gb = _C.group_norm_backward(go.cuda(), xc, saved, 3, wc, bc, activation="silu")
    direction = torch.randn(x.shape, generator=torch.Generator().manual_seed(1))

    def value(h):
        y, _ = _C.group_norm_forward((x + h * direction).cuda(), 3, wc, bc, activation="silu")
        return (y.double().cpu() * go.double()).sum().item()

    # central differences: 10^-6 / 2 h from rounding (240 outputs of 2^-22), h^2 of the third derivative
    h = 2.0 ** -6
    slope = (value(h) - value(-h)) / (2 * h)
    assert abs(slope - (gx.double().cpu() * direction.double()).sum().item()) < 2e-2


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_in_a_graph_and_on_another_stream(device, dtype):
    for size, groups in (((2, 64, 32), 4), ((2, 5000, 64), 8)):
        x, w, b, go = (t.cuda() for t in make(9, *size, dtype))

        def both():
            y, saved = _C.group_norm_forward(x, groups, w, b, activation="gelu", for_backward=True)
            return [y] + _C.group_norm_backward(go, x, saved, groups, w, b, activation="gelu")

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
        torch.cuda.synchronize()
        for a, c in zip(other, both()):
            assert torch.equal(a, c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both()
        for k in range(3):
            x.copy_(make(20 + k, *size, dtype)[0])
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(held, both()):
                assert torch.equal(a, c)
            torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_results_past_the_cache(device, dtype):
    """Two samples whose tensors are larger than those whose results stay in the cache, and each alone."""
    N = 300000 if dtype == BF16 else 150000
    x, w, b, go = (t.cuda() for t in make(11, 2, N, 64, dtype))
    y, saved = _C.group_norm_forward(x, 16, w, b, activation="silu", for_backward=True)
    gx, gw, gb = _C.group_norm_backward(go, x, saved, 16, w, b, activation="silu")
    sums = 0
    for i in range(2):
        one, kept = _C.group_norm_forward(x[i:i + 1], 16, w, b, activation="silu", for_backward=True)
        assert torch.equal(one[0], y[i]) and torch.equal(kept[0], saved[i])
        g = _C.group_norm_backward(go[i:i + 1], x[i:i + 1], kept, 16, w, b, activation="silu")
        assert torch.equal(g[0][0], gx[i])
        sums = sums + torch.stack(g[1:]).double()
    # the halves' sums are rounded once more
    half = 2.0 ** -8 if dtype == BF16 else 2 * U
    assert ((torch.stack((gw, gb)).double() - sums).abs() <= half * (4 * sums.abs() + 2 * N ** 0.5)).all()


def test_more_than_32_bits_of_values(device):
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    # 2^32 values and some, one sample far larger than the other's strides reach in 32 bits
    N, C = (1 << 26) + 5, 64
    x = torch.zeros(1, N, C, dtype=BF16, device="cuda")
    x[0, -1, -4:] = 8
    x[0, 0, -4:] = -8
    y, saved = _C.group_norm_forward(x, 16, eps=1e-5, for_backward=True)
    r = 1 / math.sqrt(128 / N + 1e-5)
    assert abs(y[0, -1, -1].item() - 8 * r) <= 2.0 ** -7 * 8 * r
    # all others: zero but for the mean's error
    assert (y.abs() > 64 * U * 8 * r).sum().item() == 8 and (y[..., :60] == 0).all()
    assert abs(saved[0, 15, 1].item() - r) < 1e-4 * r


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(2, 60, 32), (1, 1, 32), (2, 20000, 32)])
def test_biases_that_shut_or_open_a_channel(device, size, dtype, activation):
    """Far below zero an activation and its slope vanish, far above it they are u and 1: gradients are those
    of channels whose gradient is zero, or of no activation, to the bit."""
    x, w, b, go = (t.cuda() for t in make(14, *size, dtype))
    for far in (-1e30, -torch.finfo(dtype).max, 1e30, torch.finfo(dtype).max):
        bias = b.clone()
        bias[::5] = far
        shut = torch.zeros(size[2], dtype=torch.bool, device="cuda")
        shut[::5] = True
        y, saved = _C.group_norm_forward(x, 4, w, bias, activation=activation, for_backward=True)
        gx, gw, gb = _C.group_norm_backward(go, x, saved, 4, w, bias, activation=activation)
        y0, _ = _C.group_norm_forward(x, 4, w, b, activation=activation)
        assert torch.equal(y[..., ~shut], y0[..., ~shut])
        assert all(torch.isfinite(t).all() for t in (gx, gw, gb))
        if far < 0:
            assert (y[..., shut] == 0).all() and (gw[shut] == 0).all() and (gb[shut] == 0).all()
            none = torch.where(shut, 0.0, go).to(dtype)
            gx0, gw0, gb0 = _C.group_norm_backward(none, x, saved, 4, w, b, activation=activation)
            assert torch.equal(gx, gx0) and torch.equal(gw, gw0) and torch.equal(gb, gb0)
        else:
            # (n w is lost next to the bias)
            assert torch.equal(y[..., shut], bias[shut].expand_as(y[..., shut]))
            gb0 = _C.group_norm_backward(go, x, saved, 4, w, b)[2]
            assert torch.equal(gb[shut], gb0[shut])

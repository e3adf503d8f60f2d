"""Norm of queries and keys per head with the position rotation, and its gradients, against the same
computed in float64 on the CPU.

Tolerances, from the number formats.  float32: a row's mean of squares, its root and a handful of
products, some twenty roundings of 2^-24 of values up to the row's largest: 4e-6 of the result's
largest value; the weights' gradients are sums over all rows (1e-5).  bfloat16: computed in fp32
from the same inputs and rounded once, 2^-9 of each value: 4e-3."""
import pytest
import torch

from mappedconvolutions_amd import _C

pytestmark = pytest.mark.gpu

TOL = {torch.float32: (4e-6, 1e-5), torch.bfloat16: (4e-3, 4e-3)}


def reference(x, w, cos, sin, positions, eps, adjacent, g):
    """y, grad x, grad w in float64."""
    x = x.detach().double().cpu().requires_grad_()
    w = w.detach().double().cpu().requires_grad_()
    cos, sin = cos.double().cpu(), sin.double().cpu()
    B, L = x.shape[:2]
    at = torch.arange(L).expand(B, L) if positions is None else positions.cpu()
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    F = cos.shape[1]
    y = n.clone()
    first = slice(0, 2 * F, 2) if adjacent else slice(0, F)
    second = slice(1, 2 * F, 2) if adjacent else slice(F, 2 * F)
    y[..., first] = n[..., first] * c - n[..., second] * s
    y[..., second] = n[..., second] * c + n[..., first] * s
    gx, gw = torch.autograd.grad(y, (x, w), g.detach().double().cpu())
    return y.detach(), gx, gw


def close(got, want, tol, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    if want.numel():
        off, size = (got - want).abs().max().item(), want.abs().max().item()
        assert off <= tol * max(size, 1e-3), "%s: off by %g of %g" % (what, off, size)


def problem(seed, dtype, B, L, Hq, Hk, D, F, places=None):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randn(B, L, Hq + 2 * Hk, D, generator=g).to(dtype).cuda()
    weights = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2)]
    angle = torch.rand(places or max(L, 1), F, generator=g, dtype=torch.float64) * 100
    grads = [torch.randn(B, L, H, D, generator=g).to(dtype).cuda() for H in (Hq, Hk)]
    return (packed[:, :, :Hq], packed[:, :, Hq:Hq + Hk], *weights, angle.cos().float().cuda(),
            angle.sin().float().cuda(), grads)


def check(q, k, wq, wk, cos, sin, grads, positions=None, eps=1e-6, adjacent=False):
    tol, tol_sum = TOL[q.dtype]
    args = (q, k, wq, wk, cos, sin, positions, eps, adjacent)
    out = _C.qk_norm_rotate_forward(*args)
    back = _C.qk_norm_rotate_backward(*grads, *args)
    for n, (x, w) in enumerate(((q, wq), (k, wk))):
        y, gx, gw = reference(x, w, cos, sin, positions, eps, adjacent, grads[n])
        close(out[n], y, tol, "output %d" % n)
        close(back[n], gx, tol, "gradient %d" % n)
        close(back[2 + n], gw, tol_sum, "weight gradient %d" % n)
    for a, b in zip(back, _C.qk_norm_rotate_backward(*grads, *args)):
        assert torch.equal(a, b)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("size", [
    # B, L, Hq, Hk, D, F
    (1, 1, 1, 1, 1, 0),
    (8, 1, 16, 4, 64, 32),
    (2, 37, 4, 4, 32, 16),
    (3, 101, 6, 2, 48, 16),
    (2, 33, 5, 1, 128, 64),
    (2, 19, 9, 3, 96, 20),
    (1, 70, 3, 2, 256, 128),
    (2, 50, 2, 1, 7, 3),
    (1, 41, 4, 2, 40, 20),
    (2, 900, 2, 2, 24, 0),
])
def test_sizes(device, size, dtype, adjacent):
    check(*problem(1, dtype, *size), adjacent=adjacent)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions(device, dtype):
    B, L, places = 3, 45, 1000
    args = problem(2, dtype, B, L, 4, 2, 64, 32, places)
    positions = torch.randint(0, places, (B, L), generator=torch.Generator().manual_seed(3)).cuda()
    check(*args, positions=positions)
    check(*args, positions=positions.t().contiguous().t(), adjacent=True)
    # one outside the table: that token is no number, the others are as before
    good = _C.qk_norm_rotate_forward(*args[:6], positions)
    for bad in (-1, places, 1 << 40):
        positions[1, 7] = bad
        out = _C.qk_norm_rotate_forward(*args[:6], positions)
        for a, b in zip(out, good):
            assert torch.isnan(a[1, 7]).all()
            a[1, 7] = b[1, 7]
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(device, dtype):
    q, k, wq, wk, cos, sin, grads = problem(4, dtype, 2, 30, 4, 2, 32, 16)
    want = _C.qk_norm_rotate_forward(q, k, wq, wk, cos, sin)
    dense = [t.contiguous() for t in (q, k)]
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    last = [t.transpose(1, 3).contiguous().transpose(1, 3) for t in (q, k)]
    for pair in (dense, heads, last):
        for a, b in zip(_C.qk_norm_rotate_forward(*pair, wq, wk, cos, sin), want):
            assert torch.equal(a, b)
    wide = torch.randn(2, 30, 6, 37, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    check(wide[:, :, :4, 3:35], wide[:, :, 4:, 3:35], wq, wk, cos, sin, grads)
    check(wide[:, :, :4, 3:35], wide[:, :, 4:, 3:35], wq, wk, cos, sin, grads, adjacent=True)
    # gradients in another order, weights that start at any value
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in grads]
    odd = torch.cat((wq[:1], wq, wk))
    check(q, k, odd[1:33], odd[33:], cos, sin, turned)


def test_rows_of_zeros_and_large_values(device):
    q, k, wq, wk, cos, sin, grads = problem(6, torch.float32, 1, 12, 2, 2, 64, 32)
    q = q.clone()
    q[0, 3], q[0, 4] = 0, q[0, 4] * 1e15
    out = check(q, k, wq, wk, cos, sin, grads, eps=1e-5)
    assert (out[0][0, 3] == 0).all()


def test_empty(device):
    q, k, wq, wk, cos, sin, grads = problem(7, torch.float32, 2, 0, 2, 1, 16, 8)
    assert _C.qk_norm_rotate_forward(q, k, wq, wk, cos, sin)[0].shape == (2, 0, 2, 16)
    back = _C.qk_norm_rotate_backward(*grads, q, k, wq, wk, cos, sin)
    assert (back[2] == 0).all() and (back[3] == 0).all()


def test_gradient_against_differences(device):
    # float32 steps of 1e-2 along a direction of length one: differences are off by terms of third
    # order and by roundings, 1e-4 together on derivatives of size one
    q, k, wq, wk, cos, sin, grads = problem(8, torch.float32, 1, 9, 2, 1, 32, 12)
    back = _C.qk_norm_rotate_backward(*grads, q, k, wq, wk, cos, sin)
    g = torch.Generator().manual_seed(9)
    for n in range(4):
        way = torch.randn((q, k, wq, wk)[n].shape, generator=g).cuda()
        way /= way.norm()
        ends = []
        for sign in (1, -1):
            x = [q, k, wq, wk]
            x[n] = x[n] + sign * 1e-2 * way
            out = _C.qk_norm_rotate_forward(*x, cos, sin)
            ends.append(sum((a.double() * b.double()).sum() for a, b in zip(out, grads)))
        slope = ((ends[0] - ends[1]) / 2e-2).item()
        assert abs(slope - (back[n].double() * way.double()).sum().item()) < 1e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 37])
def test_partial_gradients(device, dtype, D):
    q, k, wq, wk, cos, sin, grads = problem(10, dtype, 2, 300, 6, 2, D, 16)
    full = _C.qk_norm_rotate_backward(*grads, q, k, wq, wk, cos, sin)
    for bits in range(16):
        needs = tuple(bool(bits >> n & 1) for n in range(4))
        got = _C.qk_norm_rotate_backward(*grads, q, k, wq, wk, cos, sin, needs=needs)
        for a, b, n in zip(got, full, needs):
            assert (a is None) if not n else torch.equal(a, b)
    # no tokens: the weights' gradients are zeros
    got = _C.qk_norm_rotate_backward(grads[0][:, :0], grads[1][:, :0], q[:, :0], k[:, :0], wq, wk, cos,
                                     sin, needs=(True, False, False, True))
    assert got[0].shape == (2, 0, 6, D) and got[1] is None and got[2] is None and (got[3] == 0).all()

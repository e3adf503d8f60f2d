"""Clipping by the global norm against float64.

Tolerances: squares are summed in fp32 over a few hundred values of a thread and in fp64 from there
on, the root and the factor are rounded once: 1e-6 of the norm; a product is rounded to its type,
2^-24 or 2^-9 of the value, beside the factor's 1e-6: 2e-6 and 4e-3."""
import pytest
import torch

from mappedconvolutions_amd import _C

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 4e-3}


def tensors(seed, sizes, dtypes=(torch.float32,)):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * 10. ** -(i % 3)).to(dtypes[i % len(dtypes)]).cuda()
            for i, n in enumerate(sizes)]


def check(ts, max_norm, out=None):
    wide = [t.double().cpu() for t in ts]
    norm = torch.sqrt(sum((t * t).sum() for t in wide)).item()
    factor = min(1.0, max_norm / (norm + 1e-6))
    got = _C.clip_grad_norm(ts, max_norm, out=out)
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(got.item() - norm) <= 1e-6 * norm
    for before, after, t in zip(wide, ts if out is None else out, ts):
        want = before * factor
        if want.numel():
            off = (after.double().cpu() - want).abs()
            assert (off <= TOL[t.dtype] * want.abs() + 1e-37).all()
        if out is not None:
            assert torch.equal(t.double().cpu(), before)


BOTH = (torch.float32, torch.bfloat16)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("sizes", [
    [1], [7], [2048], [2049, 0, 3], [100001], [5, 300000, 17, 70000],
    list(range(1, 300)), [64] * 128, [64] * 129, [40000] * 257, [3000001, 1],
])
def test_sizes(device, sizes, in_place):
    for max_norm in (0.5, 1e9, 0.0):
        ts = tensors(1, sizes, BOTH)
        check(ts, max_norm, None if in_place else [torch.full_like(t, 7) for t in ts])


def test_factor_one_changes_nothing(device):
    ts = tensors(2, [1000, 50001], BOTH)
    before = [t.clone() for t in ts]
    out = [torch.empty_like(t) for t in ts]
    _C.clip_grad_norm(ts, 1e9, out=out)
    _C.clip_grad_norm(ts, 1e9)
    for a, b, c in zip(ts, before, out):
        assert torch.equal(a, b) and torch.equal(c, b)


def test_parts_of_a_buffer_at_any_address(device):
    for dtype in BOTH:
        flat = tensors(3, [50000], (dtype,))[0]
        parts = [flat[1:8], flat[8:5003], flat[5003:5003], flat[5004:30001], flat[30001:49999]]
        ends = flat[:1].clone(), flat[5003:5004].clone(), flat[49999:].clone()
        to = torch.zeros(50010, dtype=dtype, device="cuda")
        out = [to[3:10], to[10:5005], to[5005:5005], to[5005:30002], to[30003:50001]]
        check(parts, 0.25, out)
        assert to[:3].abs().sum() == 0 and to[30002] == 0 and to[50001:].abs().sum() == 0
        check(parts, 0.25)
        for a, b in zip((flat[:1], flat[5003:5004], flat[49999:]), ends):
            assert torch.equal(a, b)


def test_the_same_bits_each_time(device):
    ts = tensors(4, [123457, 99, 1000000], BOTH)
    norms = {_C.clip_grad_norm(ts, 1e9).item() for _ in range(5)}
    assert len(norms) == 1


def test_infinities_and_nan(device):
    ts = tensors(5, [1000, 1000])
    ts[1][7] = float("inf")
    norm = _C.clip_grad_norm(ts, 1.0)
    assert norm.item() == float("inf")
    assert (ts[0] == 0).all() and torch.isnan(ts[1][7]) and (ts[1][:7] == 0).all()
    ts = tensors(6, [1000, 1000])
    ts[0][3] = float("nan")
    assert torch.isnan(_C.clip_grad_norm(ts, 1.0))
    assert all(torch.isnan(t).all() for t in ts)


def test_no_values_at_all(device):
    ts = [torch.empty(0, device="cuda"), torch.empty(0, device="cuda")]
    assert _C.clip_grad_norm(ts, 1.0).item() == 0
    zero = [torch.zeros(100, device="cuda")]
    assert _C.clip_grad_norm(zero, 1.0).item() == 0 and (zero[0] == 0).all()


def test_more_than_32_bits_of_values(device):
    n = (1 << 32) + 100
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[-1], t[5] = 3, 4
    assert _C.clip_grad_norm([t], 2.5).item() == 5
    assert t[-1].item() == 1.5 and t[5].item() == 2


def test_in_a_graph(device):
    ts = tensors(7, [1000, 70001], BOTH)
    out = [torch.empty_like(t) for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _C.clip_grad_norm(ts, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = _C.clip_grad_norm(ts, 1.0, out=out)
    for n in range(3):
        for t, x in zip(ts, tensors(20 + n, [1000, 70001], BOTH)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(t) for t in ts]
        assert torch.equal(_C.clip_grad_norm(ts, 1.0, out=eager), norm)
        for a, b in zip(eager, out):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("size", [1e25, 1e18, 1e-18, 1e-25, 1e-30])
def test_values_whose_squares_leave_fp32(device, size, dtype):
    # (values a thread walks in words, those before and behind them, and a part of zeros)
    ts = [(size * t.double()).to(dtype) for t in tensors(8, [3, 5001, 300000], (dtype,))]
    ts.insert(1, torch.zeros(70000, dtype=dtype, device="cuda"))
    ts = [torch.cat((t[:1], t))[1:] for t in ts]
    wide = [t.double().cpu() for t in ts]
    norm = torch.sqrt(sum((t * t).sum() for t in wide)).item()
    out = [torch.empty_like(t) for t in ts]
    got = _C.clip_grad_norm(ts, 0.25 * norm, eps=0.0, out=out)
    assert abs(got.item() - norm) <= 1e-6 * norm
    for o, t in zip(out, wide):
        off = (o.double().cpu() - 0.25 * t).abs()
        assert (off <= TOL[dtype] * 0.25 * t.abs() + 1e-37).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_one_value_whose_square_leaves_fp32(device, dtype):
    for at in (0, 12345, 99999):
        ts = tensors(9, [50, 100000], (dtype,))
        ts[1][at] = 1e22
        check(ts, 1.0)

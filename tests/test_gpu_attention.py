"""Attention with a bias by relative-position buckets, its gradients and its form for few queries,
against the same computed in float64 on the CPU.

Tolerances, from the number formats.  float32: sums of at most a few thousand products of size one
in fp32, 2e-5 of the result's largest value (several hundred roundings of 2^-24).  bfloat16: the
inputs are the same bf16 values for both; probabilities and score gradients are rounded to bf16
(2^-9 each) before a product, the result once more: each output is a sum whose terms are off by at
most 2^-8 + 2^-9 of their size, 2e-2 of the result's largest value allows for the sum of the terms'
sizes being some three times the result."""
import math

import pytest
import torch

from mappedconvolutions_amd import _C

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-5, torch.bfloat16: 2e-2}


def reference(q, k, v, table=None, buckets=None, zero=0, scale=None, causal=False, start=None,
              lengths=None, go=None):
    """out, and with go the gradients of q, k, v and table, in float64 on the CPU."""
    q, k, v = (t.detach().double().cpu().requires_grad_(go is not None) for t in (q, k, v))
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    kk, vv = (t.repeat_interleave(Hq // Hk, 2) for t in (k, v))
    pos = torch.zeros(B, dtype=torch.int64) if start is None else start.cpu().long()
    rel = torch.arange(Lk) - (pos[:, None, None] + torch.arange(Lq)[:, None])  # B Lq Lk
    keep = torch.ones_like(rel, dtype=torch.bool)
    if causal:
        keep &= rel <= 0
    if lengths is not None:
        n = lengths.cpu().long().clamp(0, Lk)
        keep &= (torch.arange(Lk) < n[:, None])[:, None]
        used = (torch.arange(Lk) < n[:, None])[:, :, None, None]
        kk, vv = torch.where(used, kk, 0.), torch.where(used, vv, 0.)
    s = torch.einsum("bihd,bjhd->bhij", q, kk) * scale
    if table is not None:
        table = table.detach().double().cpu().requires_grad_(go is not None)
        which = buckets.cpu().long()[(rel + zero).clamp(0, buckets.numel() - 1)]
        known = (which >= 0) & (which < table.shape[1])
        bias = table[:, which.clamp(0, table.shape[1] - 1)].transpose(0, 1)
        s = s + torch.where(known[:, None], bias, 0.)
    keep = keep[:, None] & (s > -math.inf)
    top = torch.where(keep, s, -math.inf).amax(-1, keepdim=True) if Lk else s.new_zeros(B, Hq, Lq, 1)
    top = torch.where(top == -math.inf, 0., top).detach()
    e = torch.where(keep, torch.exp(torch.where(keep, s - top, 0.)), 0.)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1., total)
    out = torch.einsum("bhij,bjhd->bihd", p, vv)
    if go is None:
        return out
    leaves = [q, k, v] + ([] if table is None else [table])
    grads = torch.autograd.grad(out, leaves, go.detach().double().cpu(), allow_unused=True)
    return [out.detach()] + [torch.zeros_like(t) if g is None else g for t, g in zip(leaves, grads)]


def close(got, want, tol, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what + ": not finite"
    if got.numel():
        bound = tol * max(want.abs().max().item(), 1e-3)
        off = (got - want).abs().max().item()
        assert off <= bound, "%s: off by %g of %g" % (what, off, bound)


def problem(seed, dtype, B, Lq, Lk, Hq, Hk, D, NB=16, reach=40, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (spread * torch.randn(B, L, H, D, generator=g) for L, H in ((Lq, Hq), (Lk, Hk), (Lk, Hk)))
    go = torch.randn(B, Lq, Hq, D, generator=g)
    table = torch.randn(Hq, NB, generator=g)
    buckets = torch.randint(0, NB, (2 * reach + 1,), generator=g).int()
    q, k, v, go, table = (t.to(dtype).cuda() for t in (q, k, v, go, table))
    return q, k, v, go, table, buckets.cuda(), reach


def check(q, k, v, go, table, buckets, zero, train=True, **kw):
    tol = TOL[q.dtype]
    names = dict(bias_table=table, buckets=buckets, bucket_zero=zero,
                 query_start=kw.get("start"), key_lengths=kw.get("lengths"),
                 scale=kw.get("scale"), causal=kw.get("causal", False))
    out, stats = _C.relative_attention_forward(q, k, v, for_backward=train, **names)
    want = reference(q, k, v, table, buckets, zero, go=go if train else None, **kw)
    if not train:
        assert stats is None
        close(out, want, tol, "out")
        return out
    close(out, want[0], tol, "out")
    grads = _C.relative_attention_backward(go, q, k, v, out, stats, **names)
    for name, got, w in zip(("grad_query", "grad_key", "grad_value", "grad_bias_table"), grads, want[1:]):
        close(got, w, tol, name)
    again = _C.relative_attention_backward(go, q, k, v, out, stats, **names)
    for a, b in zip(grads, again):
        assert a is None or torch.equal(a, b)
    return out


SIZES = [
    # B, Lq, Lk, Hq, Hk, D
    (1, 1, 1, 1, 1, 1),
    (2, 5, 7, 2, 1, 8),
    (1, 64, 64, 2, 2, 64),
    (2, 128, 128, 4, 2, 64),
    (1, 129, 65, 3, 1, 40),
    (2, 200, 333, 6, 2, 48),
    (1, 257, 191, 2, 2, 96),
    (1, 300, 300, 4, 1, 128),
    (3, 33, 31, 2, 1, 13),
    (1, 700, 130, 2, 2, 32),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("causal", [False, True])
def test_forward_and_gradients(device, size, dtype, causal):
    check(*problem(1, dtype, *size), causal=causal)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(2, 100, 100, 2, 2, 32), (1, 190, 70, 4, 2, 128)])
def test_without_bias(device, size, dtype):
    q, k, v, go, _, _, _ = problem(2, dtype, *size)
    check(q, k, v, go, None, None, 0, scale=0.3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths_and_starts(device, dtype):
    # no key, one, some, all, more than there are; positions before, amid and behind the keys
    B, Lq, Lk = 6, 70, 150
    lengths = torch.tensor([0, 1, 77, 150, 400, -3], dtype=torch.int32).cuda()
    start = torch.tensor([0, -30, 20, 80, 149, 5], dtype=torch.int32).cuda()
    args = problem(3, dtype, B, Lq, Lk, 4, 2, 32)
    for causal in (False, True):
        check(*args, causal=causal, lengths=lengths, start=start)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unused_keys_may_hold_anything(device, dtype):
    q, k, v, go, table, buckets, zero = problem(4, dtype, 3, 90, 200, 2, 1, 64)
    lengths = torch.tensor([0, 130, 64], dtype=torch.int32).cuda()
    for b, n in enumerate(lengths.tolist()):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
        k[b, n + 1::2] = -float("inf")
    check(q, k, v, go, table, buckets, zero, lengths=lengths)
    # a single query takes the form that splits the keys
    check(q[:, :1], k, v, go[:, :1], table, buckets, zero, lengths=lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lq", [1, 150])
def test_buckets_taken_out_and_lowest_values(device, dtype, Lq):
    q, k, v, go, table, buckets, zero = problem(5, dtype, 2, Lq, 150, 2, 1, 32, NB=8)
    table[0, 3] = -float("inf")          # some pairs
    table[1, :] = -float("inf")          # a head of which nothing is left
    out = check(q, k, v, go, table, buckets, zero)
    assert (out[:, :, 1] == 0).all()
    table[0, 3] = torch.finfo(dtype).min  # swallows the scores it is added to
    check(q, k, v, go, table, buckets, zero)
    # rows with nothing but the lowest value: all their keys alike
    low = torch.full_like(table, torch.finfo(dtype).min)
    out, stats = _C.relative_attention_forward(q, k, v, low, buckets, zero, for_backward=True)
    close(out, v.double().cpu().mean(1, keepdim=True).expand(2, 150, 1, 32)[:, :Lq].repeat(1, 1, 2, 1),
          TOL[dtype], "mean of the values")
    grads = _C.relative_attention_backward(go, q, k, v, out, stats, low, buckets, zero)
    gv = (go.double().cpu().sum(1).sum(1) / 150)[:, None, None].expand(2, 150, 1, 32)
    close(grads[2], gv, TOL[dtype], "gradient of the values")


def test_unknown_buckets_have_no_bias(device):
    q, k, v, go, table, buckets, zero = problem(6, torch.float32, 1, 140, 140, 2, 2, 32, NB=8)
    buckets[::3] = -1
    buckets[1::7] = 8
    check(q, k, v, go, table, buckets, zero)
    check(q[:, :2], k, v, go[:, :2], table, buckets, zero)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(device, dtype):
    g = torch.Generator().manual_seed(7)
    B, L, D = 2, 130, 32
    packed = torch.randn(B, L, 8, D, generator=g).to(dtype).cuda()
    q, k, v = packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:]
    go = torch.randn(B, L, 4, D, generator=g).to(dtype).cuda()
    _, _, _, _, table, buckets, zero = problem(7, dtype, 1, 1, 1, 4, 2, D)
    check(q, k, v, go, table, buckets, zero, causal=True)
    # heads before tokens
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    check(*heads, go.transpose(1, 2).contiguous().transpose(1, 2), table, buckets, zero)
    # rows that start at any value
    wide = torch.randn(B, L, 8, D + 5, generator=g).to(dtype).cuda()[..., 3:3 + D]
    for n in (L, 1):
        check(wide[:, :n, :4], wide[:, :, 4:6], wide[:, :, 6:], go[:, :n], table, buckets, zero)
    # one row for all, and a head size that is dense in another axis
    check(q, k.expand(2, L, 2, D)[:1].expand(B, L, 2, D), v, go, table, buckets, zero)
    turned = [t.transpose(1, 3).contiguous().transpose(1, 3) for t in (q, k, v)]
    check(*turned, go, table, buckets, zero)


DECODE = [
    # B, Lq, Lk, Hq, Hk, D
    (1, 1, 1, 1, 1, 64),
    (1, 1, 1000, 8, 8, 64),
    (3, 1, 4097, 8, 2, 128),
    (2, 5, 777, 12, 4, 40),
    (1, 2, 3001, 64, 1, 32),
    (2, 1, 130, 40, 1, 96),
    (1, 40, 2000, 2, 1, 48),
    (2, 3, 5, 3, 1, 7),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", DECODE)
def test_few_queries_against_a_cache(device, size, dtype):
    B, Lq, Lk = size[:3]
    args = problem(8, dtype, *size)
    check(*args, train=False)
    lengths = torch.tensor([max(0, Lk - 61 * b) for b in range(B)], dtype=torch.int32).cuda()
    check(*args, train=False, causal=True, lengths=lengths, start=lengths - Lq)
    check(*args, causal=True, lengths=lengths, start=lengths - Lq)


def test_a_cache_beyond_32_bits(device):
    # one key head of 2^31 values and more between the batches: offsets need 64 bits
    B, Lk, D = 3, 1 << 22, 128
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    cache = torch.zeros(B, 2, Lk, 1, D, dtype=torch.bfloat16, device="cuda")
    k, v = cache[:, 0], cache[:, 1]
    g = torch.Generator().manual_seed(9)
    n = 300
    for b in range(B):
        k[b, -n:] = torch.randn(n, 1, D, generator=g).cuda().bfloat16() * 3
        v[b, -n:] = torch.randn(n, 1, D, generator=g).cuda().bfloat16()
    q = torch.randn(B, 1, 2, D, generator=g).cuda().bfloat16()
    # all but the last 300 keys are taken out by their bucket
    buckets = torch.ones(n, dtype=torch.int32, device="cuda")
    buckets[0] = 0
    table = torch.zeros(2, 2, dtype=torch.bfloat16, device="cuda")
    table[:, 0] = -float("inf")
    start = torch.full((B,), Lk - 1, dtype=torch.int32, device="cuda")
    out, _ = _C.relative_attention_forward(q, k, v, table, buckets, n - 1, causal=True, query_start=start)
    want = reference(q, k[:, -n + 1:], v[:, -n + 1:])
    close(out, want, TOL[torch.bfloat16], "out")


def test_gradient_against_differences(device):
    # float32 steps of 1e-2: the difference is off by 2nd order terms (1e-4 of the curvature, size
    # one here) and by roundings, 1e-5 / 1e-2; bound 5e-3 on derivatives of size one
    q, k, v, go, table, buckets, zero = problem(10, torch.float32, 1, 40, 50, 2, 1, 16, NB=6)

    def loss(*x):
        out, _ = _C.relative_attention_forward(*x[:3], x[3], buckets, zero, causal=True,
                                               query_start=torch.full((1,), 10, dtype=torch.int32).cuda())
        return (out.double() * go.double()).sum()

    start = torch.full((1,), 10, dtype=torch.int32).cuda()
    out, stats = _C.relative_attention_forward(q, k, v, table, buckets, zero, causal=True,
                                               query_start=start, for_backward=True)
    grads = _C.relative_attention_backward(go, q, k, v, out, stats, table, buckets, zero,
                                           causal=True, query_start=start)
    g = torch.Generator().manual_seed(11)
    for n in range(4):
        x = [q, k, v, table]
        way = torch.randn(x[n].shape, generator=g).cuda()
        way /= way.norm()
        ends = []
        for sign in (1, -1):
            y = list(x)
            y[n] = x[n] + sign * 1e-2 * way
            ends.append(loss(*y))
        slope = ((ends[0] - ends[1]) / 2e-2).item()
        assert abs(slope - (grads[n].double() * way.double()).sum().item()) < 5e-3


def test_partial_gradients(device):
    q, k, v, go, table, buckets, zero = problem(12, torch.bfloat16, 2, 100, 100, 4, 2, 64)
    out, stats = _C.relative_attention_forward(q, k, v, table, buckets, zero, for_backward=True)
    full = _C.relative_attention_backward(go, q, k, v, out, stats, table, buckets, zero)
    for needs in ((True, False, False, False), (False, True, False, False),
                  (False, False, True, False), (False, False, False, True), (False,) * 4):
        got = _C.relative_attention_backward(go, q, k, v, out, stats, table, buckets, zero, needs=needs)
        for a, b, n in zip(got, full, needs):
            assert (a is None) if not n else torch.equal(a, b)


def test_empty_sizes(device):
    q, k, v, go, table, buckets, zero = problem(13, torch.float32, 2, 10, 12, 2, 1, 16)
    out, stats = _C.relative_attention_forward(q, k[:, :0], v[:, :0], table, buckets, zero, for_backward=True)
    assert (out == 0).all()
    grads = _C.relative_attention_backward(go, q, k[:, :0], v[:, :0], out, stats, table, buckets, zero)
    assert (grads[0] == 0).all() and (grads[3] == 0).all() and grads[1].shape == (2, 0, 1, 16)
    out, stats = _C.relative_attention_forward(q[:, :0], k, v, table, buckets, zero, for_backward=True)
    assert out.shape == (2, 0, 2, 16)
    grads = _C.relative_attention_backward(go[:, :0], q[:, :0], k, v, out, stats, table, buckets, zero)
    assert all((t == 0).all() for t in grads[1:])
    out, _ = _C.relative_attention_forward(q[:0], k[:0], v[:0], table, buckets, zero)
    assert out.shape == (0, 10, 2, 16)


def test_another_stream(device):
    q, k, v, go, table, buckets, zero = problem(14, torch.bfloat16, 2, 300, 300, 4, 2, 64)
    want, _ = _C.relative_attention_forward(q, k, v, table, buckets, zero)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, stats = _C.relative_attention_forward(q, k, v, table, buckets, zero, for_backward=True)
        grads = _C.relative_attention_backward(go, q, k, v, got, stats, table, buckets, zero)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    for t in grads:
        t.record_stream(torch.cuda.current_stream())
        assert torch.isfinite(t.float()).all()


def test_in_a_graph(device):
    q, k, v, go, table, buckets, zero = problem(15, torch.bfloat16, 2, 150, 700, 4, 2, 64)

    def step():
        out, stats = _C.relative_attention_forward(q, k, v, table, buckets, zero, for_backward=True)
        one, _ = _C.relative_attention_forward(q[:, :1], k, v, table, buckets, zero)
        return [out, one] + _C.relative_attention_backward(go, q, k, v, out, stats, table, buckets, zero)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(n)).to(q))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(1, 1100, 1000, 2, 1, 64), (1, 520, 1700, 3, 3, 40), (2, 900, 600, 2, 1, 128)])
def test_small_grids_are_split_and_joined(device, size, dtype):
    # fewer workgroups than compute units: parts of the keys, of the queries, some of them empty
    args = problem(16, dtype, *size, NB=24, reach=200)
    B, Lq, Lk = size[:3]
    check(*args)
    check(*args, causal=True)
    lengths = torch.tensor([Lk // 3, 1][:B], dtype=torch.int32).cuda()
    start = torch.tensor([Lk // 2 - Lq, -5][:B], dtype=torch.int32).cuda()
    check(*args, causal=True, lengths=lengths, start=start)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 64, 96, 128])
def test_largest_table(device, dtype, D):
    check(*problem(17, dtype, 1, 200, 260, 2, 1, D, NB=512, reach=300), causal=True)
    check(*problem(18, dtype, 2, 1, 700, 40, 1, D, NB=512, reach=300), train=False)


def test_one_bucket_and_many_runs(device):
    # a new bucket every difference; and all differences in one, which shifts a row's scores alike
    # (its gradient is a sum that comes to nothing, so it is not asked for)
    q, k, v, go, table, buckets, zero = problem(19, torch.float32, 2, 250, 270, 2, 2, 32, NB=500, reach=240)
    each = torch.arange(buckets.numel(), dtype=torch.int32).cuda()
    check(q, k, v, go, table, each, zero)
    want = reference(q, k, v, go=go)
    for one, at in ((torch.full_like(buckets, 7), zero), (each[:1].clone(), 0)):
        out, saved = _C.relative_attention_forward(q, k, v, table, one, at, for_backward=True)
        grads = _C.relative_attention_backward(go, q, k, v, out, saved, table, one, at,
                                               needs=(True, True, True, False))
        for got, w in zip([out] + grads[:3], want):
            close(got, w, TOL[torch.float32], "one bucket")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(3, 300, 300, 6, 3, 32), (35, 140, 150, 4, 2, 32), (5, 260, 260, 5, 1, 64),
                                  (1, 200, 4200, 2, 1, 128)])
def test_orders_of_work(device, size, dtype):
    # key heads that the XCDs share unevenly, one and several in a row, more than an L2 holds
    B, Lk = size[0], size[2]
    args = problem(21, dtype, *size)
    lengths = torch.tensor([Lk - 37 * b % Lk for b in range(B)], dtype=torch.int32).cuda()
    start = torch.full((B,), Lk - size[1], dtype=torch.int32).cuda()
    check(*args, lengths=lengths)
    check(*args, causal=True, lengths=lengths, start=start)


# ---- rows whose largest score is far from zero ----------------------------------------------
# Zero queries (or whole numbers) make every score exact in both types, however large the bias, so the
# tolerances above hold: what is left are the roundings of exponents of size one, of sums and products.

FAR = [
    # B, Lq, Lk, Hq, Hk, D: as many workgroups as compute units, and few, split along both axes
    (64, 130, 130, 4, 2, 64),
    (1, 260, 700, 2, 1, 64),
    (1, 260, 700, 2, 1, 48),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", FAR)
@pytest.mark.parametrize("bias", [-1e3, -1e4, -1e6, -1e8, -6e8, 3e4])
def test_rows_under_one_large_bias(device, size, bias, dtype):
    q, k, v, go, table, buckets, zero = problem(30, dtype, *size)
    table = torch.full_like(table, bias)
    check(torch.zeros_like(q), k, v, go, table, buckets, zero)
    check(torch.zeros_like(q), k, v, go, table, buckets, zero, causal=True)


@pytest.mark.parametrize("size", FAR[:2])
@pytest.mark.parametrize("bias", [-1e3, -1e4, -1e6])
def test_differences_of_large_biases(device, size, bias):
    # (whole numbers: exact over the scale of 2^-3) the largest of a row lies in any of its tiles
    q, k, v, go, table, buckets, zero = problem(31, torch.float32, *size, NB=64)
    table = bias + torch.arange(64, device="cuda", dtype=torch.float32).div(8).floor().expand(size[3], 64)
    check(torch.zeros_like(q), k, v, go, table, buckets, zero)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", FAR[:2])
def test_large_scores(device, size, dtype):
    # one value of 2^13 in every query makes scores of 1024 and a little; quarters: exact products
    q, k, v, go, table, buckets, zero = problem(32, dtype, *size)
    q, k = ((4 * t).round().clamp(-12, 12) / 4 for t in (q, k))
    q[..., 0], k[..., 0] = 8192, 1
    check(q, k, v, go, torch.zeros_like(table), buckets, zero)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("near", [0.0, -1e6, -6e8])
def test_rows_of_different_size_in_a_wave(device, near, dtype):
    # ten keys in use: the first rows see them under one bias, the last under the lowest value, those
    # between under both
    q, k, v, go, _, _, _ = problem(33, dtype, 2, 150, 600, 2, 1, 64)
    buckets = torch.zeros(41, dtype=torch.int32, device="cuda")
    buckets[:5] = 1  # differences of -16 and less
    table = torch.tensor([near, torch.finfo(dtype).min]).to(dtype).cuda().expand(2, 2)
    lengths = torch.tensor([10, 333], dtype=torch.int32).cuda()
    # (a row sees one bucket or two of which one takes all: the table's gradient is a sum that comes to
    # nothing, so it is not asked for)
    q = torch.zeros_like(q)
    want = reference(q, k, v, table, buckets, 20, lengths=lengths, go=go)
    args = dict(bias_table=table, buckets=buckets, bucket_zero=20, key_lengths=lengths)
    out, saved = _C.relative_attention_forward(q, k, v, for_backward=True, **args)
    grads = _C.relative_attention_backward(go, q, k, v, out, saved, needs=(True, True, True, False), **args)
    for got, w in zip([out] + grads[:3], want):
        close(got, w, TOL[dtype], "two sizes")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", FAR)
@pytest.mark.parametrize("bias", [0.0, -1e4, -1e6, -1e8, -6e8, -1e12])
def test_probabilities_of_the_gradients_sum_to_one(device, size, bias, dtype):
    # whatever a large bias leaves of the scores: sum_j grad_value_j = sum_i grad_output_i
    q, k, v, go, table, buckets, zero = problem(34, dtype, *size)
    Hq, Hk = size[3:5]
    want = go.double().sum(1).unflatten(1, (Hk, Hq // Hk)).sum(2)
    bound = TOL[dtype] * go.double().abs().sum(1).max().item()
    for n in (size[1], 1):
        if n == 1:  # the form for few queries
            go = go[:, :1].contiguous()
            want = go.double().sum(1).unflatten(1, (Hk, Hq // Hk)).sum(2)
            bound = TOL[dtype] * go.double().abs().max().item()
        args = (torch.full_like(table, bias), buckets, zero)
        out, saved = _C.relative_attention_forward(q[:, :n], k, v, *args, for_backward=True)
        gv = _C.relative_attention_backward(go, q[:, :n], k, v, out, saved, *args)[2]
        assert ((gv.double().sum(1) - want).abs() <= bound).all()


def test_more_workgroups_than_a_launch_takes(device):
    # 2^24 workgroups of 256 threads are one thread more than a launch can have
    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("needs 32 GB")
    a_million_sequences()
    torch.cuda.empty_cache()  # (blocks of gigabytes, that small tensors of later tests would hold)


def a_million_sequences():
    B, H, D = (1 << 20) + 3, 16, 8
    g = torch.Generator(device="cuda").manual_seed(50)
    q, k, v, go = (torch.randn(B, 2, H, D, generator=g, device="cuda").bfloat16() for _ in range(4))
    table = torch.randn(H, 3, generator=g, device="cuda").bfloat16()
    buckets = torch.arange(3, dtype=torch.int32, device="cuda")
    args = dict(bias_table=table, buckets=buckets, bucket_zero=1)
    out, saved = _C.relative_attention_forward(q, k, v, for_backward=True, **args)
    gq, gk, gv, _ = _C.relative_attention_backward(go, q, k, v, out, saved, needs=(True, True, True, False),
                                                   **args)
    for at in (0, 1 << 18, 1 << 19, (1 << 20) - 2, B - 4):
        part = slice(at, at + 4)
        want = reference(q[part], k[part], v[part], table, buckets, 1, go=go[part])
        for got, w, name in zip((out, gq, gk, gv), want, ("out", "grad_query", "grad_key", "grad_value")):
            close(got[part], w, TOL[torch.bfloat16], name)


ANY_ROWS = [
    # B, Lq, Lk, Hq, Hk, D: heads that are not whole 16-byte words, of every padded size
    (1, 140, 150, 2, 1, 50),
    (2, 131, 70, 2, 2, 61),
    (1, 150, 200, 4, 2, 90),
    (1, 129, 140, 2, 1, 100),
    (1, 200, 90, 3, 1, 127),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", ANY_ROWS)
def test_heads_of_any_size(device, size, dtype):
    args = problem(40, dtype, *size)
    B, Lq, Lk = size[:3]
    lengths = torch.tensor([Lk - 31 * b - 5 for b in range(B)], dtype=torch.int32).cuda()
    check(*args)
    check(*args, causal=True, lengths=lengths)
    # few queries over many keys, in one part and split
    few = problem(41, dtype, 2, 2, 1500, *size[3:])
    lengths = torch.tensor([1500, 900], dtype=torch.int32).cuda()
    check(*few, train=False, causal=True, lengths=lengths, start=lengths - 2)
    q, k, v, go, table, buckets, zero = few
    check(q, k[:, :90], v[:, :90], go, table, buckets, zero)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_rows_at_any_address(device, D, dtype):
    # whole heads of a packed projection that starts one value behind a 16-byte boundary, and the
    # second case split along both axes
    _, _, _, _, table, buckets, zero = problem(42, dtype, 1, 1, 1, 4, 2, D)
    for B, L in ((2, 140), (1, 530)):
        g = torch.Generator().manual_seed(43)
        flat = torch.randn(B * L * 8 * D + 1, generator=g).to(dtype).cuda()
        packed = flat[1:].view(B, L, 8, D)
        q, k, v = packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:]
        go = torch.randn(B, L, 4, D, generator=g).to(dtype).cuda()
        check(q, k, v, go, table, buckets, zero, causal=True)
        check(q[:, :1], k, v, go[:, :1], table, buckets, zero)


def test_another_stream_gives_the_same_bits(device):
    # calls of different data on two streams at once, split along both axes, against each alone
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    calls = [problem(44 + n, torch.bfloat16, 1, 900, 800, 4, 2, 64) for n in range(2)]

    def step(q, k, v, go, table, buckets, zero):
        out, saved = _C.relative_attention_forward(q, k, v, table, buckets, zero, for_backward=True)
        return [out] + _C.relative_attention_backward(go, q, k, v, out, saved, table, buckets, zero)

    want = [step(*c) for c in calls]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for s, c, g in zip(sides, calls, got):
            with torch.cuda.stream(s):
                g.append(step(*c))
    for s in sides:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for run in runs:
            for a, b in zip(run, w):
                assert torch.equal(a, b)

"""The gated recurrence against float64.

Tolerances, u = 2^-24.  sigmoid(x) and 1 - sigmoid(x): the exponent's product is off by |x| u, exp2,
the sum, the reciprocal and a product by one or two roundings each: (6 + |x|) u.  A state is a sum of
values times products of factors; in whatever order they are joined, a factor adds its error to all that
went through it, so with M_t = a_t M_{t-1} + (1 - a_t) |v_t| the state is off by
E_t = a_t E_{t-1} + (8 + |f_t|) u M_t, and 16 u M_t for the joins.  The same holds for D backward.  What is
formed from them adds a dozen roundings.  bf16 outputs: 2^-8 of the value besides (half a step)."""
import pytest
import torch

from mappedconvolutions_amd import _C

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def make(seed, B, L, C, dtype):
    """value, forget, gate, grad_output [B, L, C], initial, grad_final [B, C]; forget gates of a few
    tokens up to hundreds."""
    g = torch.Generator().manual_seed(seed)
    v, f, z, go = (torch.randn(B, L, C, generator=g) for _ in range(4))
    f = 1.5 * f + 6 * torch.rand(C, generator=g)
    return [t.to(dtype) for t in (v, f, z, go)] + [torch.randn(B, C, generator=g) for _ in range(2)]


def oracle(v, f, z, go, first, last, lengths, reverse):
    """([out, final, gv, gf, gg, gi], their bounds without the outputs' rounding), in 64 bits."""
    B, L, C = v.shape
    used = [L] * B if lengths is None else [min(max(n, 0), L) for n in lengths]
    index = torch.zeros(B, L, dtype=torch.long)
    live = torch.zeros(B, L, 1, dtype=torch.bool)
    for b, n in enumerate(used):
        order = torch.arange(n)
        index[b, :n] = order.flip(0) if reverse else order
        index[b, n:] = torch.arange(n, L)
        live[b, :n] = True
    at = index[:, :, None].expand(B, L, C)

    def steps(t):  # in the order of the steps, first axis first
        return None if t is None else torch.gather(torch.where(live, t.double(), 0.0), 1, at)

    def tokens(t):
        return torch.zeros(B, L, C, dtype=torch.float64).scatter_(1, at, torch.where(live, t, 0.0))

    V, F, Z, G = (steps(t) for t in (v, f, z, go))
    a, away = torch.sigmoid(F), torch.sigmoid(-F)
    a = torch.where(live, a, 1.0)
    away = torch.where(live, away, 0.0)
    eps = torch.where(live, (8 + F.abs()) * U, 0.0)
    h = torch.zeros(B, C, dtype=torch.float64) if first is None else first.double()
    M, E = h.abs(), torch.zeros_like(h)
    hs, before, Ms, Mb, Es, Eb = ([] for _ in range(6))
    for t in range(L):
        before.append(h), Mb.append(M), Eb.append(E + 16 * U * M)
        h = a[:, t] * h + away[:, t] * V[:, t]
        M = a[:, t] * M + away[:, t] * V[:, t].abs()
        E = a[:, t] * E + eps[:, t] * M
        hs.append(h), Ms.append(M), Es.append(E + 16 * U * M)
    final, final_e = h, E + 16 * U * M

    def stack(ts):
        return torch.stack(ts, 1) if ts else torch.zeros(B, 0, C, dtype=torch.float64)

    hs, before, Ms, Mb, Es, Eb = map(stack, (hs, before, Ms, Mb, Es, Eb))
    if Z is None:
        silu, slope, zu = torch.ones_like(V), None, 0.0
    else:
        s = torch.sigmoid(Z)
        silu, slope, zu = Z * s, s * (1 + Z * (1 - s)), (10 + 2 * Z.abs()) * U
    out, out_e = hs * silu, Es * silu.abs() + zu * Ms * silu.abs()
    d = G * silu
    p = torch.zeros(B, C, dtype=torch.float64) if last is None else last.double()
    pM, pE = p.abs(), torch.zeros_like(p)
    D, DM, DE = ([None] * L for _ in range(3))
    for t in reversed(range(L)):
        D[t], DM[t] = d[:, t] + p, d[:, t].abs() + pM
        DE[t] = (zu[:, t] if Z is not None else 0.0) * d[:, t].abs() + pE + 16 * U * DM[t]
        p, pM, pE = a[:, t] * D[t], a[:, t] * DM[t], a[:, t] * (DE[t] - 16 * U * DM[t]) + eps[:, t] * DM[t]
    D, DM, DE = map(stack, (D, DM, DE))
    gv, gv_e = away * D, away * (DE + eps * DM)
    size = before.abs() + V.abs() + Mb
    gf = D * (before - V) * a * away
    gf_e = a * away * (DE * size + DM * Eb + (2 * eps + 8 * U) * DM * size)
    results = [tokens(out), final, tokens(gv), tokens(gf)]
    bounds = [tokens(out_e), final_e, tokens(gv_e), tokens(gf_e)]
    if Z is not None:
        results.append(tokens(G * hs * slope))
        bounds.append(tokens(G.abs() * (1.1 * Es + (16 * U + 2 * zu) * Ms)))
    return results + [p], bounds + [pE + 16 * U * pM]


def call(v, f, z, go, first, last, lengths, reverse):
    out, final, saved = _C.gated_recurrence_forward(v, f, z, first, lengths, reverse, for_backward=True)
    plain = _C.gated_recurrence_forward(v, f, z, first, lengths, reverse)
    assert torch.equal(plain[0], out) and torch.equal(plain[1], final) and plain[2] is None
    gv, gf, gg, gi = _C.gated_recurrence_backward(go, v, f, z, saved, last, lengths, reverse)
    assert (gg is None) == (z is None)
    return [out, final, gv, gf] + ([] if z is None else [gg]) + [gi]


def check(v, f, z, go, first, last, lengths=None, reverse=False, views=lambda *ts: ts):
    def to(t):
        return None if t is None else t.cuda()

    held = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = call(*views(to(v), to(f), to(z)), to(go), to(first), to(last), held, reverse)
    want, bounds = oracle(v, f, z, go, first, last, lengths, reverse)
    for k, (a, b, e) in enumerate(zip(got, want, bounds)):
        half = 2.0 ** -8 if a.dtype == BF16 else U
        off, bound = (a.double().cpu() - b).abs(), e + half * b.abs() + 1e-30
        assert a.is_contiguous() and a.shape == b.shape
        assert (off <= bound).all(), (k, (off / bound).max().item())
    return got


SIZES = [(1, 1, 1), (2, 2, 3), (3, 7, 64), (2, 8, 60), (2, 9, 66), (1, 127, 16), (2, 128, 4), (1, 129, 130),
         (2, 255, 20), (1, 256, 64), (3, 257, 5), (1, 513, 192), (2, 1025, 12), (1, 4097, 68),
         (600, 40, 64), (1, 1300, 2), (1, 9000, 160), (3, 5000, 33), (1, 70, 20000), (9000, 12, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(device, size, dtype):
    v, f, z, go, first, last = make(1, *size, dtype)
    for reverse in (False, True):
        check(v, f, z, go, first, last, reverse=reverse)
        check(v, f, None, go, None, None, reverse=reverse)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [15, 16, 17, 31, 32, 33])
def test_tiles_of_few_steps(device, L, dtype):
    for C in (5, 36, 66, 72):
        for reverse in (False, True):
            v, f, z, go, first, last = make(12, 3, L, C, dtype)
            check(v, f, z, go, first, last, reverse=reverse)
            check(v, f, z, go, first, last, [L, 0, L - 9], reverse)
            check(v, f, None, go, None, None, [3, L - 1, 1], reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lengths(device, dtype, reverse):
    for L, lengths in ((6, [0, 1, 6, 5]), (300, [300, 0, 257, 128]), (2100, [2100, 1, 1023, 1024]),
                       (50, [-7, 99, 50, 2])):
        v, f, z, go, first, last = make(2, 4, L, 20, dtype)
        # what is not in use may be anything
        for b, n in enumerate(lengths):
            for t in (v, f, z, go):
                t[b, max(0, n):] = float("nan")
        got = check(v, f, z, go, first, last, lengths, reverse)
        check(v, f, None, go, None, None, lengths, reverse)
        for b, n in enumerate(lengths):
            if n <= 0:  # no step: the state and its gradient pass
                assert torch.equal(got[1][b].cpu(), first[b]) and torch.equal(got[-1][b].cpu(), last[b])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(device, dtype):
    for L in (5, 270):
        v, f, z, go, first, last = make(3, 3, L, 24, dtype)

        def packed(front, between):
            def parts(*ts):
                wide = torch.full((3, L, front + 3 * (24 + between)), 9.0, dtype=dtype, device="cuda")
                at = [front + k * (24 + between) for k in range(3)]
                for a, t in zip(at, ts):
                    if t is not None:
                        wide[..., a:a + 24] = t
                return [None if t is None else wide[..., a:a + 24] for a, t in zip(at, ts)]
            return parts

        for front, between in ((0, 0), (4, 8), (2, 0), (1, 1), (0, 3)):
            check(v, f, z, go, first, last, views=packed(front, between))
        check(v, f, z, go, first, last, views=lambda *ts: [
            t.transpose(0, 1).contiguous().transpose(0, 1) for t in ts])  # steps outermost
        check(v, f, z, go, first, last, views=lambda *ts: [
            t.transpose(1, 2).contiguous().transpose(1, 2) for t in ts])  # no dense last axis
        check(v, f[:, :1].expand(3, L, 24), z, go, first, last,
              views=lambda a, b, c: (a, b[:, :1].expand(3, L, 24), c))  # one gate for all steps


def test_a_state_that_is_kept(device):
    for L in (1, 5, 300, 3000):  # a thread's walk, tiles, segments
        v, f, z, go, first, last = (t.cuda() for t in make(4, 2, L, 40, BF16))
        out, final, _ = _C.gated_recurrence_forward(v, f, z, first)
        kept = first.clone()
        again, same, _ = _C.gated_recurrence_forward(v, f, z, kept, final=kept)
        assert same is kept and torch.equal(kept, final) and torch.equal(again, out)
        # given gradients of neither state
        held = torch.empty(2, 40, device="cuda")
        _C.gated_recurrence_forward(v, f, z, None, final=held)
        assert torch.equal(held, _C.gated_recurrence_forward(v, f, z)[1])


def test_token_by_token(device):
    v, f, z, _, first, _ = (t.cuda() for t in make(5, 3, 150, 36, F32))
    whole, final, _ = _C.gated_recurrence_forward(v, f, z, first)
    state, outs = first.clone(), []
    for t in range(150):
        outs.append(_C.gated_recurrence_forward(*(x[:, t:t + 1] for x in (v, f, z)), state, final=state)[0])
    M = 1 + v.abs().max().item()
    # both are off by a hundred factors' errors at most: 150 (8 + 12) u of the largest value
    assert (torch.cat(outs, 1) - whole).abs().max().item() <= 2 * 150 * 20 * U * M
    assert (state - final).abs().max().item() <= 2 * 150 * 20 * U * M


def test_gates_that_are_open_or_shut(device):
    B, L, C = 2, 700, 8
    v, f, z, go, first, last = make(6, B, L, C, F32)
    for value, size in ((float("inf"), "open"), (200.0, "open"), (-200.0, "shut"), (-1e30, "shut")):
        f[:] = value
        got = call(*(t.cuda() for t in (v, f, z, go, first, last)), None, False)
        assert all(torch.isfinite(t).all() for t in got)
        if size == "open":  # the state is carried as it is
            assert torch.equal(got[1].cpu(), first)
            assert (got[2] == 0).all() and (got[3] == 0).all()
        else:  # every step's state is its value
            assert torch.allclose(got[1].cpu(), v[:, -1], rtol=1e-6)
            assert got[-1].abs().max() < 1e-30
    f[:] = 0.0
    f[1, 300, 3] = float("nan")
    out, final, _ = _C.gated_recurrence_forward(v.cuda(), f.cuda(), z.cuda(), first.cuda())
    bad = torch.isnan(out).cpu()
    assert bad[1, 300:, 3].all() and bad.sum() == L - 300 and torch.isnan(final).sum() == 1


@pytest.mark.parametrize("gated", [False, True])
def test_gradients_that_are_not_wanted(device, gated):
    v, f, z, go, first, last = (t.cuda() for t in make(7, 2, 1100, 24, BF16))
    z = z if gated else None
    _, _, saved = _C.gated_recurrence_forward(v, f, z, first, for_backward=True)
    every = _C.gated_recurrence_backward(go, v, f, z, saved, last)
    for needs in ((True, False, False, False), (False, True, False, False), (False, False, True, False),
                  (False, False, False, True), (True, False, True, True), (False, False, False, False)):
        some = _C.gated_recurrence_backward(go, v, f, z, saved, last, needs=needs)
        for a, b, wanted in zip(some, every, needs):
            assert a is None if not wanted or b is None else torch.equal(a, b)


def test_gradient_against_differences(device):
    v, f, z, go, first, last = make(8, 1, 40, 6, F32)
    _, _, saved = _C.gated_recurrence_forward(v.cuda(), f.cuda(), z.cuda(), first.cuda(), for_backward=True)
    grads = _C.gated_recurrence_backward(go.cuda(), v.cuda(), f.cuda(), z.cuda(), saved, last.cuda())
    g = torch.Generator().manual_seed(1)
    for k, t in enumerate((v, f, z, first)):
        way = torch.randn(t.shape, generator=g)

        def value(h):
            moved = [x + h * way if n == k else x for n, x in enumerate((v, f, z, first))]
            out, final, _ = _C.gated_recurrence_forward(*(x.cuda() for x in moved))
            return ((out.double().cpu() * go).sum() + (final.double().cpu() * last).sum()).item()

        h = 2.0 ** -7
        slope = (value(h) - value(-h)) / (2 * h)
        want = (grads[k].double().cpu() * way).sum().item()
        # 246 outputs of up to 2^-22 over 2 h, and h^2 of a third derivative of some tens
        assert abs(slope - want) < 2e-2 + 1e-3 * abs(want)


def test_the_same_bits_on_two_streams_and_in_a_graph(device):
    for size in ((4, 3, 64), (3, 2200, 64)):
        args = [t.cuda() for t in make(9, *size, BF16)]
        lengths = torch.tensor([size[1], 1, 2, 3][:size[0]], dtype=torch.int32, device="cuda")
        want = call(*args, lengths, True)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call(*args, lengths, True))
        torch.cuda.synchronize()
        for one in got:
            for a, b in zip(one, want):
                assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()

        def run():
            out, final, saved = _C.gated_recurrence_forward(*args[:3], args[4], lengths, for_backward=True)
            return [out, final] + _C.gated_recurrence_backward(args[3], *args[:3], saved, args[5], lengths)

        with torch.cuda.graph(graph):
            held = run()
        for k in range(3):
            for t, x in zip(args, make(30 + k, *size, BF16)):
                t.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(held, run()):
                assert torch.equal(a, b)
            torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_results_past_the_cache(device, dtype):
    """A batch whose tensors are larger than those whose results stay in the cache, and its halves, which
    are not: each sequence is computed alike."""
    B = 6000 if dtype == BF16 else 3000
    v, f, z, go, first, last = (t.cuda() for t in make(10, B, 100, 64, dtype))
    whole = call(v, f, z, go, first, last, None, False)
    for half in (slice(0, B // 2), slice(B // 2, B)):
        for a, b in zip(call(*(t[half] for t in (v, f, z, go, first, last)), None, False), whole):
            assert torch.equal(a, b[half])


def test_many_short_sequences(device):
    B = 1 << 21  # of 48 channels: 3 tiles each
    v, f, z, go, first, last = make(13, 64, 2, 48, BF16)
    few = call(*(t.cuda() for t in (v, f, z, go, first, last)), None, False)
    many = [t.cuda().repeat(B // 64, *[1] * (t.dim() - 1)) for t in (v, f, z, go, first, last)]
    for a, b in zip(call(*many, None, False), few):
        assert torch.equal(a.view(B // 64, *b.shape), b.expand(B // 64, *b.shape))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [1, 2, 3, 4, 6, 8, 10, 13, 24, 32])
def test_few_channels(device, C, dtype):
    for L, lengths in ((64, [64, 1, 33]), (65, [65, 64, 3]), (100, [100, 37, 0]), (257, [257, 1, 256]), (700, [3, 699, 700]), (5000, [5000, 4097, 1025])):
        v, f, z, go, first, last = make(14, 3, L, C, dtype)
        for reverse in (False, True):
            check(v, f, z, go, first, last, lengths, reverse)
            check(v, f, None, go, None, None, None, reverse)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_channels_far_apart(device, dtype):
    # as far as the kernels' addresses reach: the last step of a tile lies close to 2^32 bytes from its first
    L = 600 if dtype == BF16 else 300
    v, f, z, go, first, last = make(15, 2, L, 5, dtype)
    wide = torch.zeros(L, 1 << 22, dtype=dtype, device="cuda")

    def apart(*ts):
        out = []
        for k, t in enumerate(ts):
            view = wide[:, 10 * k:10 * k + 10].unflatten(1, (2, 5)).transpose(0, 1)
            view.copy_(t)
            out.append(view)
        return out

    for reverse in (False, True):
        check(v, f, z, go, first, last, [L, L - 7], reverse, views=apart)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_steps_backward(device, dtype):
    for L in range(1, 10):
        for C in (1, 6, 20, 68):
            v, f, z, go, first, last = make(16, 5, L, C, dtype)
            for reverse in (False, True):
                check(v, f, z, go, first, last, [L, 0, L - 1, 1, L + 3], reverse)
                check(v, f, None, go, first, None, None, reverse)
    for L in (1, 8):
        args = [t.cuda() for t in make(17, 3, L, 24, dtype)]
        _, _, saved = _C.gated_recurrence_forward(*args[:3], args[4], for_backward=True)
        every = _C.gated_recurrence_backward(args[3], *args[:3], saved, args[5])
        for k in range(4):
            some = _C.gated_recurrence_backward(args[3], *args[:3], saved, args[5], needs=[n == k for n in range(4)])
            assert all(t is None for n, t in enumerate(some) if n != k) and torch.equal(some[k], every[k])


def test_steps_far_apart(device):
    # further than the kernels' addresses reach from a tile's first: copied
    v, f, z, go, first, last = make(11, 2, 70, 16, BF16)

    def apart(*ts):
        wide = torch.zeros(70, (1 << 22) + 64, dtype=BF16, device="cuda")
        out = []
        for k, t in enumerate(ts):
            view = wide[:, 32 * k:32 * k + 32].unflatten(1, (2, 16)).transpose(0, 1)
            view.copy_(t)
            out.append(view)
        return out

    check(v, f, z, go, first, last, views=apart)


def test_empty(device):
    first, last = torch.ones(3, 8, device="cuda"), torch.full((3, 8), 2.0, device="cuda")
    x = torch.zeros(3, 0, 8, device="cuda")
    out, final, saved = _C.gated_recurrence_forward(x, x, x, first, for_backward=True)
    assert out.shape == (3, 0, 8) and torch.equal(final, first)
    assert (_C.gated_recurrence_forward(x, x, x)[1] == 0).all()
    grads = _C.gated_recurrence_backward(out, x, x, x, saved, last)
    assert grads[0].shape == (3, 0, 8) and torch.equal(grads[3], last)
    assert (_C.gated_recurrence_backward(out, x, x, x, saved)[3] == 0).all()
    x = torch.zeros(0, 5, 8, device="cuda")
    out, final, saved = _C.gated_recurrence_forward(x, x, x, for_backward=True)
    assert out.shape == (0, 5, 8) and final.shape == (0, 8)
    assert _C.gated_recurrence_backward(out, x, x, x, saved)[3].shape == (0, 8)


def test_more_than_32_bits_of_values(device):
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    L, C = (1 << 25) + 300, 128  # 2^32 values and some
    v = torch.zeros(1, L, C, dtype=BF16, device="cuda")
    f = torch.zeros(1, 1, C, dtype=BF16, device="cuda").expand(1, L, C)  # a = 1 / 2
    v[0, -3], v[0, 5] = 8, 4
    out, final, saved = _C.gated_recurrence_forward(v, f, for_backward=True)
    assert (out[0, -3:, :] == torch.tensor([4., 2., 1.], device="cuda")[:, None]).all()
    assert (out[0, 5:8, :] == torch.tensor([2., 1., .5], device="cuda")[:, None]).all()
    assert (final == 1).all()
    del out
    gv = _C.gated_recurrence_backward(v, v, f, None, saved, needs=(True, False, False, False))[0]
    assert (gv[0, -4:, 0] == torch.tensor([2., 4., 0., 0.], device="cuda")).all()
    assert (gv[0, 4:6, 127] == torch.tensor([1., 2.], device="cuda")).all()


def check_at_the_ends(v, f, z, go, first, last, reverse):
    """As check(), where gates lie far outside: forget gates below -80 count as that (a is 1.9e-35), and of the
    output gate's silu and slope, which are below 10^-36 from -90 on, nothing need be left.  Both clamps'
    whole effect is added to the bounds for the clamped gates: what is computed is then near c, and rounding
    takes half a step of that."""
    got = call(*(None if t is None else t.cuda() for t in (v, f, z, go, first, last)), None, reverse)
    near, bounds = oracle(v, f.clamp(min=-80), None if z is None else z.clamp(min=-90), go, first, last, None, reverse)
    far = (f < -80).any() or (z is not None and (z < -90).any())
    want = oracle(v, f, z, go, first, last, None, reverse)[0] if far else near
    for k, (a, b, c, e) in enumerate(zip(got, want, near, bounds)):
        half = 2.0 ** -8 if a.dtype == BF16 else U
        off, bound = (a.double().cpu() - b).abs(), e + (b - c).abs() + half * c.abs() + 1e-30
        assert (off <= bound).all(), (k, (off / bound).max().item())


# a tile; segments of four lanes, of 16, of 64 in the first launch, of words that are not whole
SHUT_SIZES = [(2, 300, 64), (3, 2100, 8), (1, 1300, 64), (2, 700, 320), (2, 1100, 33)]


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SHUT_SIZES)
def test_shut_gates_and_large_values(device, size, dtype, reverse):
    B, L, C = size
    for gated, shut, large in ((True, -21.0, 1e3), (False, -25.0, 1e4), (True, -1e30, 1e30),
                               (False, -float("inf"), 300.0)):
        v, f, z, go, first, last = make(18, B, L, C, dtype)
        v *= large
        first *= large
        # runs of shut gates of many lengths, one of hundreds of steps
        at = torch.arange(L)[:, None] + 7 * torch.arange(C)
        f[:, (at % 64) % 11 < 5] = shut
        f[:, L // 2:L // 2 + 150] = shut
        check_at_the_ends(v, f, z if gated else None, go, first, last, reverse)
    f[:] = -30.0  # all of them
    check_at_the_ends(v, f, z, go, first, last, reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SHUT_SIZES)
def test_a_shut_gate_resets_a_large_state(device, size, dtype, reverse):
    B, L, C = size
    for gated, shut in ((False, -60.0), (True, -100.0)):
        v, f, z, go, first, last = make(19, B, L, C, dtype)
        f[:, L // 2] = shut  # e^-60 = 9e-27 of the state is left
        if gated:  # and at the ends, where the states come in
            f[:, 0], f[:, -1] = shut, shut
        check_at_the_ends(v, f, z if gated else None, go, 1e12 * first, 1e12 * last, reverse)


def test_a_batch_does_not_change_its_sequences(device):
    """The same sequences in a batch that is cut into segments and in one that is not, where gates are shut and
    values large: both are within the same bound of the exact state."""
    v, f, z, go, first, last = make(21, 1, 1300, 64, BF16)
    f[:, ::2], f[:, 40:90] = -30.0, -30.0
    v *= 500
    few, many = ([t.cuda().repeat(B, *[1] * (t.dim() - 1)) for t in (v, f, z, go, first, last)] for B in (1, 300))
    bounds = oracle(v, f, z, go, first, last, None, False)
    for k, (a, b, want, e) in enumerate(zip(call(*few, None, False), call(*many, None, False), *bounds)):
        half = 2.0 ** -8 if a.dtype == BF16 else U
        off = (a.double() - b[:1].double()).abs().cpu()
        assert (off <= 2 * (e + half * want.abs()) + 1e-30).all(), k
        assert torch.equal(b, b[:1].expand_as(b))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(3, 1, 24), (3, 6, 24), (3, 14, 24)] + SHUT_SIZES)
def test_output_gates_far_from_zero(device, size, dtype, reverse):
    v, f, z, go, first, last = make(20, *size, dtype)
    for i, far in enumerate((-88.0, -100.0, -1e30, torch.finfo(dtype).min, 100.0, 1e4)):
        z[..., i::8] = far
    check_at_the_ends(v, f, z, go, first, last, reverse)
    # what is no number stays none, and stays where it is
    z[0, 0, 0] = float("nan")
    out, final, _ = _C.gated_recurrence_forward(v.cuda(), f.cuda(), z.cuda(), first.cuda(), None, reverse)
    assert torch.isnan(out[0, 0, 0]) and torch.isnan(out).sum() == 1 and torch.isfinite(final).all()

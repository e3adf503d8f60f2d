"""The AdamW step against float64.

Tolerances, u = 2^-24.  m: two constants, two products and a sum, each rounded: 3 u of |b1 m| + |c1 g|
and u of the result, 4 u in all; v: one product more, 5 u.  The change of p: m's 4 u, sqrt(v)'s half of 5 u
and its own rounding, two constants, two products, a sum, a division: 12 u of its size before
anything cancels, and in 8 bits, where root and reciprocal are off by a unit in the last place (2 u) each
and the quotient is a product more, 15 u; p's product and the difference: 3 u of p.  bf16 parameters: 2^-8 of the result
besides.  Clipping: the factor is off by 1e-6 (the norm) and a rounding: 1.2e-6 of g, 2.4e-6 of v.
In 8 bits what is held is equal to the definition's, but where the exact sum of value and chance lies
nearer to a border than 32 bits tell (4 u of the parts over the step, and 2^-19 for up to 16 steps), and in
blocks whose largest value is as near to a power of two (5 u of its parts, which are at most 2^4 of it
unless they cancel: 2^-16 is far outside): the scale, and with it the smallest steps, may be twice as
large there, so that what is held is off by two of these steps and the oracle's by one."""
import pytest
import torch

import adamw_oracle as oracle
from mappedconvolutions_amd import _C

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


class Problem:
    def __init__(self, seed, sizes, bits=32, p_types=(F32,), g_types=(F32,), at=0):
        g = torch.Generator().manual_seed(seed)

        def make(values, dtype):
            """On the GPU, `at` values behind an aligned address."""
            flat = torch.zeros(values.numel() + 16, dtype=dtype, device="cuda")
            flat[at:at + values.numel()] = values.to(dtype).cuda()
            return flat[at:at + values.numel()]

        self.bits, self.sizes = bits, sizes
        self.p, self.g, self.m, self.v, self.ms, self.vs = [], [], [], [], [], []
        for i, n in enumerate(sizes):
            wide = 10.0 ** -(i % 4)
            spread = 10 ** (-3 * torch.rand(n, generator=g))
            self.p.append(make(torch.randn(n, generator=g), p_types[i % len(p_types)]))
            self.g.append(make(torch.randn(n, generator=g) * wide * spread, g_types[i % len(g_types)]))
            m = 0.3 * wide * torch.randn(n, generator=g) * spread
            v = (0.01 + torch.rand(n, generator=g)) * wide ** 2 * spread ** 2
            if bits == 32:
                self.m.append(make(m, F32))
                self.v.append(make(v, F32))
            else:
                self.m.append(make(torch.randint(0, 256, (n,), generator=g), torch.uint8))
                self.v.append(make(torch.randint(1, 256, (n,), generator=g), torch.uint8))
                power = [2.0 ** torch.randint(-20, 4, (oracle.blocks(n),), generator=g).float()
                         for _ in "mv"]
                self.ms.append(power[0].cuda())
                self.vs.append(power[1].cuda())

    def scales(self, **kw):
        return dict(first_scales=self.ms, second_scales=self.vs, **kw) if self.bits == 8 else {}

    def moments(self):
        """In 64 bits on the CPU, of every tensor."""
        if self.bits == 32:
            return [(m.double().cpu(), v.double().cpu()) for m, v in zip(self.m, self.v)]
        return [(oracle.decode(m.cpu(), a.cpu(), False), oracle.decode(v.cpu(), b.cpu(), True))
                for m, v, a, b in zip(self.m, self.v, self.ms, self.vs)]

    def check(self, number=7, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, decay=0.1, max_norm=None,
              seed=5, run=None):
        """One step compared with the oracle; run(): takes it in place of the plain call."""
        before = [(p.double().cpu(), g.clone(), m, v) for p, g, (m, v) in
                  zip(self.p, self.g, self.moments())]
        norm = factor = None
        if max_norm is not None:
            norm = torch.sqrt(sum(g.double().square().sum() for g in self.g)).float()
            factor = min(1.0, max_norm / (norm.item() + 1e-6))
        if run is not None:
            run()
        else:
            _C.adamw_step(self.p, self.g, self.m, self.v, number, lr, betas, eps, decay,
                          grad_norm=norm, max_norm=max_norm, **self.scales(seed=seed))
        first = 0
        for t, (p0, g0, m0, v0) in enumerate(before):
            n = p0.numel()
            assert torch.equal(self.g[t], g0)
            p1, m1, v1, change, size = oracle.step(p0, g0.cpu(), m0, v0, number, lr, betas, eps, decay,
                                                   1.0 if factor is None else factor)
            more = 0.0 if factor is None else 1.2e-6
            half = 2.0 ** -8 if self.p[t].dtype == BF16 else 0.0
            bound = 3 * U * p0.abs() + ((12 if self.bits == 32 else 15) * U + 2 * more) * change + half * p1.abs() + 1e-37
            off = (self.p[t].double().cpu() - p1).abs()
            assert (off <= bound).all(), (t, n, (off / bound).max())
            m_now, v_now = self.moments()[t]
            if self.bits == 32:
                assert ((m_now - m1).abs() <= (4 * U + more) * size + 1e-37).all()
                assert ((v_now - v1).abs() <= (5 * U + 2 * more) * v1 + 1e-37).all()
            else:
                chance = oracle.words(number, seed, first, n)
                for now, exact, part, second in ((m_now, m1, chance & 65535, False),
                                                 (v_now, v1, chance >> 16, True)):
                    want, step, near, edge = oracle.held(exact, part, second)
                    room = ((5 * U + 2 * more) * (v1 if second else size) / step) + 2.0 ** -19
                    sure = (near > room) & (edge > 2.0 ** -16)
                    assert torch.equal(now[sure], want[sure])
                    assert ((now - want).abs() <= torch.where(edge > 2.0 ** -16, 1.001, 3.001) * step).all()
                first += 256 * oracle.blocks(n)


SIZES = [[1], [255, 256, 257], [0, 5, 0, 1024], [1023, 1025, 4096], [100003], list(range(1, 130)),
         [64] * 52, [300] * 53, [16385, 40000, 7, 16384]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES)
def test_sizes(device, sizes, bits):
    Problem(1, sizes, bits, (F32, BF16, F32), (F32, BF16)).check()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("at", [1, 2, 4])
def test_any_address(device, at, bits):
    problem = Problem(2, [513, 4097, 30], bits, (F32, BF16), (BF16, F32, F32), at)
    edges = [t._base for t in problem.p + problem.m + problem.v]
    before = [(b[:at].clone(), b[-(16 - at):].clone()) for b in edges]
    problem.check()
    for b, (front, back) in zip(edges, before):
        assert torch.equal(b[:at], front) and torch.equal(b[-(16 - at):], back)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kw", [
    dict(number=1), dict(number=100000), dict(betas=(0.0, 0.0)), dict(betas=(0.95, 0.9999)), dict(eps=0.5),
    dict(decay=0.0), dict(lr=0.0), dict(lr=-1e-3), dict(max_norm=0.5), dict(max_norm=1e9),
    dict(max_norm=0.0), dict(seed=2 ** 32 - 1), dict(number=2 ** 32 + 5)])
def test_numbers(device, kw, bits):
    Problem(3, [3000, 77, 1029], bits, (F32,), (BF16, F32)).check(**kw)


@pytest.mark.parametrize("bits", [32, 8])
def test_from_zero(device, bits):
    problem = Problem(4, [1000, 300], bits)
    for t in problem.m + problem.v + problem.ms + problem.vs:
        t.zero_()
    problem.g[1].zero_()  # a tensor whose gradient is zero keeps its moments zero
    problem.check(number=1)
    m, v = problem.moments()[1]
    assert (m == 0).all() and (v == 0).all()


def test_a_captured_step_counts_and_changes_its_rate(device):
    for bits in (32, 8):
        problem, twin = (Problem(5, [2000, 333], bits, (F32, BF16)) for _ in range(2))
        number = torch.tensor(6, device="cuda")
        rate, norm = torch.tensor(1e-2, device="cuda"), torch.zeros((), device="cuda")

        def call(of, step, lr, norm):
            _C.adamw_step(of.p, of.g, of.m, of.v, step, lr, weight_decay=0.1, grad_norm=norm,
                          max_norm=0.7, **of.scales(seed=3))

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            number += 1
            norm.copy_(_C.grad_norm(problem.g))
            call(problem, number, rate, norm)
        for k in range(4):
            rate.fill_(1e-2 / (k + 1))
            for a, b in zip(problem.g, twin.g):
                a.copy_(torch.randn(a.shape, device="cuda"))
                b.copy_(a)
            graph.replay()
            torch.cuda.synchronize()
            call(twin, 7 + k, rate.item(), _C.grad_norm(twin.g))
            assert number.item() == 7 + k
            for a, b in zip(problem.p + problem.m + problem.v + problem.ms + problem.vs,
                            twin.p + twin.m + twin.v + twin.ms + twin.vs):
                assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_same_bits_however_the_list_is_cut(device, bits):
    # (in 8 bits the words go by the place in the list, so only whole lists are alike)
    problem, twin = (Problem(6, [5000, 70, 100000], bits) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for k in range(3):
        _C.adamw_step(problem.p, problem.g, problem.m, problem.v, k + 1, 1e-3, **problem.scales())
        with torch.cuda.stream(side):
            _C.adamw_step(twin.p, twin.g, twin.m, twin.v, k + 1, 1e-3, **twin.scales())
    torch.cuda.synchronize()
    for a, b in zip(problem.p + problem.m + problem.v, twin.p + twin.m + twin.v):
        assert torch.equal(a, b)


def test_what_is_no_number(device):
    for bits in (32, 8):
        for bad in (float("nan"), float("inf")):
            problem, twin = (Problem(7, [1000, 600], bits) for _ in range(2))
            problem.g[0][300] = bad
            for of in (problem, twin):
                _C.adamw_step(of.p, of.g, of.m, of.v, 3, 1e-3, **of.scales())
            assert torch.equal(problem.p[1], twin.p[1])
            keep = torch.arange(1000, device="cuda") != 300
            assert torch.equal(problem.p[0][keep], twin.p[0][keep])
            assert torch.isnan(problem.p[0][300])
            m, v = problem.moments()[0]
            if bits == 8:  # the block's moments are lost, the others are not
                assert torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all()
                keep = ~torch.isnan(m)
                assert keep.sum() == 744
                assert torch.equal(m[keep], twin.moments()[0][0][keep])
            else:
                assert not torch.isfinite(m[300]) and torch.isfinite(m).sum() == 999
        # a norm that is no number makes all parameters none
        problem = Problem(8, [1000], bits)
        _C.adamw_step(problem.p, problem.g, problem.m, problem.v, 3, 1e-3, max_norm=1.0,
                      grad_norm=torch.tensor(float("nan"), device="cuda"), **problem.scales())
        assert torch.isnan(problem.p[0]).all()


def test_large_and_small_values(device):
    # gradients whose squares stay in 32 bits, from the largest down to where they vanish
    for size in (1e18, 1e-12, 1e-18, 1e-25):
        for bits in (32, 8):
            problem = Problem(9, [2000], bits)
            problem.g[0] *= size
            if bits == 32:
                problem.m[0].mul_(size), problem.v[0].mul_(min(size, 1e18)).mul_(size)
            else:
                problem.ms[0].zero_(), problem.vs[0].zero_()
            _C.adamw_step(problem.p, problem.g, problem.m, problem.v, 1, 1e-3, **problem.scales())
            assert torch.isfinite(problem.p[0]).all()
            m, v = problem.moments()[0]
            assert torch.isfinite(m).all() and torch.isfinite(v).all() and (v >= 0).all()


def test_moments_in_8_bits_follow_on_average(device):
    """2^16 values, gradients of unit variance: after 3000 steps the mean second moment is 1 - b2^3000
    of it.  Its own spread is 0.02 of a value, rounding adds a fifth; over 65536 values both are below
    0.001 of the mean, so 1 % is far outside.  Then gradients stop: it falls by b2 a step."""
    n = 65536
    p, m, v = (torch.zeros(n, dtype=t, device="cuda") for t in (F32, torch.uint8, torch.uint8))
    ms, vs = torch.zeros(n // 256, device="cuda"), torch.zeros(n // 256, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)

    def run(steps, start, size):
        for k in range(steps):
            grad = size * torch.randn(n, generator=g, device="cuda")
            _C.adamw_step([p], [grad], [m], [v], start + k + 1, 1e-3, first_scales=[ms],
                          second_scales=[vs], seed=1)
        return (_C.adamw_moment(m, ms, False).double(), _C.adamw_moment(v, vs, True).double())

    first, second = run(3000, 0, 1.0)
    assert abs(second.mean().item() / (1 - 0.999 ** 3000) - 1) < 0.01
    assert first.abs().mean() < 0.3 and abs(first.mean().item()) < 0.01
    _, later = run(1000, 3000, 0.0)
    assert abs(later.mean().item() / (second.mean().item() * 0.999 ** 1000) - 1) < 0.02


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_the_cache_holds(device, bits):
    # (enough values that they pass the cache by)
    Problem(11, [300, 10000001 if bits == 32 else 27000001], bits, (F32,), (F32, BF16)).check()


@pytest.mark.parametrize("second", [False, True])
def test_every_code(device, second):
    codes = torch.arange(256, dtype=torch.uint8).repeat(3)[:700]
    scales = torch.tensor([1.0, 2.0 ** -100, 2.0 ** 60])
    want = oracle.decode(codes, scales, second)
    for dtype in (F32, BF16):
        for at in (0, 1):
            flat = torch.zeros(710, dtype=torch.uint8, device="cuda")
            flat[at:at + 700] = codes.cuda()
            got = _C.adamw_moment(flat[at:at + 700], scales.cuda(), second, dtype)
            assert got.dtype == dtype and torch.equal(got.double().cpu(), want)
    if second:
        assert want[:256].diff().min() > 0


def test_grad_norm(device):
    problem = Problem(10, [1000, 0, 70001] + [50] * 200, 32, (F32,), (F32, BF16))
    before = [g.clone() for g in problem.g]
    norm = _C.grad_norm(problem.g)
    want = torch.sqrt(sum(g.double().square().sum() for g in before)).item()
    assert norm.dtype == F32 and abs(norm.item() - want) <= 1e-6 * want
    assert all(torch.equal(a, b) for a, b in zip(problem.g, before))
    assert torch.equal(_C.clip_grad_norm([g.clone() for g in before], 1.0), norm)


def test_many_values(device):
    n = (1 << 31) + 300  # offsets in bytes pass 32 bits, and blocks of the last values
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    p, g = (torch.zeros(n, dtype=BF16, device="cuda") for _ in range(2))
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    ms, vs = (torch.zeros(oracle.blocks(n), device="cuda") for _ in range(2))
    g[-1], g[3] = 4, -4
    _C.adamw_step([p], [g], [m], [v], 1, 0.5, first_scales=[ms], second_scales=[vs])
    assert p[-1].item() == -0.5 and p[3].item() == 0.5 and p.count_nonzero().item() == 2
    tail = _C.adamw_moment(m[-300:].contiguous()[-44:].clone(), ms[-1:], False)
    assert abs(tail[-1].item() - 0.4) <= 0.4 / 8 and tail[:-1].abs().sum() == 0


def equal(one, other, names="p m v ms vs", last=None):
    for name in names.split():
        for a, b in zip(getattr(one, name)[-last:] if last else getattr(one, name),
                        getattr(other, name)[-last:] if last else getattr(other, name)):
            assert torch.equal(a, b), name


def test_parts_of_a_list_give_the_bits_of_the_whole(device):
    """In 32 bits a tensor's result does not depend on what stands in the list beside it: in which launch it is,
    and how long its chunks are (2048 values in a list of 9 million, 1024 alone)."""
    sizes = [5000, 70, 100003, 1, 16385, 40000] + [300 + i for i in range(60)] + [9000001, 257, 2049]
    types = (F32, BF16, F32), (BF16, F32)
    whole, alone, parts = (Problem(12, sizes, 32, *types) for _ in range(3))
    numbers = (3, 1e-2, (0.9, 0.999), 1e-8, 0.1)
    clip = dict(grad_norm=_C.grad_norm(whole.g), max_norm=0.5)
    _C.adamw_step(whole.p, whole.g, whole.m, whole.v, *numbers, **clip)
    for t in range(len(sizes)):
        _C.adamw_step(alone.p[t:t + 1], alone.g[t:t + 1], alone.m[t:t + 1], alone.v[t:t + 1], *numbers, **clip)
    for part in (slice(0, 7), slice(7, 66), slice(66, None)):
        _C.adamw_step(parts.p[part], parts.g[part], parts.m[part], parts.v[part], *numbers, **clip)
    equal(whole, alone)
    equal(whole, parts)


@pytest.mark.parametrize("bits", [32, 8])
def test_an_address_does_not_change_the_bits(device, bits):
    sizes = [300, 5000, 1, 256, 16385] + [77] * 60
    problems = [Problem(13, sizes, bits, (F32, BF16, F32), (BF16, F32), at) for at in (0, 1, 2, 4)]
    for one in problems:
        _C.adamw_step(one.p, one.g, one.m, one.v, 5, 1e-3, weight_decay=0.1, **one.scales(seed=9))
    for one in problems[1:]:
        equal(problems[0], one)


def test_places_in_8_bits_count_on_over_launches(device):
    """A value's place is counted in blocks of 256 from the list's first: behind 60 tensors of 90 blocks in all,
    in a second launch, tensors are rounded as behind one of 90 blocks, and otherwise than behind none."""
    tail = [700, 256, 4097, 3]
    many, one, none = ([300] * 30 + [40] * 30, [90 * 256 - 1], [])
    problems = []
    for lead in (many, one, none):
        problem = Problem(14, lead + tail, 8)
        last = Problem(15, tail, 8)  # the same tensors at the end of every list
        for name in ("p", "g", "m", "v", "ms", "vs"):
            getattr(problem, name)[len(lead):] = getattr(last, name)
        _C.adamw_step(problem.p, problem.g, problem.m, problem.v, 5, 1e-3, **problem.scales(seed=9))
        problems.append(problem)
    assert sum(map(oracle.blocks, many)) == sum(map(oracle.blocks, one)) == 90
    equal(problems[0], problems[1], last=len(tail))
    equal(problems[0], problems[2], "p ms vs", last=len(tail))  # (what is not rounded at random)
    assert not torch.equal(problems[0].m[-2], problems[2].m[-2])


def test_scales_of_8_bits(device):
    """Twice the power of two below a block's largest value, where that is not so near to a power of two (see
    above) that 32 bits tell otherwise; zero where all are."""
    problem = Problem(16, [1000, 256, 257, 5, 40000], 8)
    problem.m[1].zero_(), problem.v[1].zero_(), problem.g[1].zero_()
    before = [(p.double().cpu(), g.cpu(), m, v) for p, g, (m, v) in zip(problem.p, problem.g, problem.moments())]
    _C.adamw_step(problem.p, problem.g, problem.m, problem.v, 5, 1e-3, **problem.scales())
    for (p, g, m, v), ms, vs in zip(before, problem.ms, problem.vs):
        _, m, v, _, _ = oracle.step(p, g, m, v, 5, 1e-3)
        for exact, got in ((m, ms), (v, vs)):
            top = oracle.per_block(exact.abs()).amax(1)
            want = torch.where(top > 0, 2 ** (torch.floor(torch.log2(top.clamp_min(1e-300))) + 1), 0.0)
            part = top / want.clamp_min(1e-300)
            sure = (top == 0) | (torch.minimum(part - 0.5, 1 - part) > 2.0 ** -16)
            assert sure.float().mean() > 0.9 and torch.equal(got.double().cpu()[sure], want[sure])

"""Host side of the attention operators: what the library and its Python boundary refuse, the
layers' parameters, buckets and angles.  Nothing here needs a GPU."""
import math

import pytest
import torch

from mappedconvolutions_amd import _C, _lib, nn, util


def desc(**kw):
    size = dict(B=1, Lq=4, Lk=4, Hq=2, Hk=1, D=16, q_stride=(128, 32, 16), k_stride=(64, 16, 16),
                v_stride=(64, 16, 16), bucket_count=9, bucket_zero=4, table_size=8, scale=0.25,
                causal=0)
    size.update(kw)
    d = _lib.AttentionDesc()
    for name, value in size.items():
        setattr(d, name, (_lib._i64 * 3)(*value) if isinstance(value, tuple) else value)
    return d


def forward(d, dtype=0, q=1, k=1, v=1, table=1, buckets=1, out=1, ws=None, nbytes=0):
    return _lib.load().mcx_attention_forward(q, k, v, table, buckets, None, None, out, None, None,
                                             ws, nbytes, d, dtype, None)


@pytest.mark.parametrize("code, kw", [
    (-1, dict(dtype=1)), (-1, dict(dtype=9)),
    (-2, dict(B=-1)), (-2, dict(Lk=-5)), (-2, dict(D=0)), (-2, dict(D=129)), (-2, dict(Hk=0)),
    (-2, dict(Hq=3, Hk=2)), (-2, dict(scale=0.0)), (-2, dict(scale=-1.0)),
    (-2, dict(scale=float("nan"))), (-2, dict(scale=1e9)), (-2, dict(table_size=513)),
    (-2, dict(table_size=0)), (-2, dict(bucket_count=0)), (-2, dict(bucket_zero=9)),
    (-2, dict(bucket_zero=-1)), (-2, dict(Lq=1 << 40)),
    (-3, dict(q=None)), (-3, dict(k=None)), (-3, dict(v=None)), (-3, dict(out=None)),
    (-3, dict(table=None)), (-3, dict(buckets=None)),
])
def test_forward_refuses(code, kw):
    outer = {n: kw.pop(n) for n in list(kw) if n in ("dtype", "q", "k", "v", "table", "buckets", "out")}
    assert forward(desc(**kw), **outer) == code
    assert forward(None) == -3


def test_workspace_is_asked_for_and_checked():
    lib = _lib.load()
    long = desc(Lq=1, Lk=100000, k_stride=(1600000, 16, 16), v_stride=(1600000, 16, 16))
    need = lib.mcx_attention_forward_workspace(long, 0)
    assert need > 0
    assert forward(long) == -4 and forward(long, ws=1, nbytes=need - 1) == -4
    assert lib.mcx_attention_forward_workspace(desc(D=500), 0) == 0
    need = lib.mcx_attention_backward_workspace(desc(), 0)
    assert need >= 3 * 2 * 4 * 4

    def backward(d, gout=1, out=1, stats=1, gtable=1, ws=1, nbytes=need, table=1):
        return lib.mcx_attention_backward(gout, 1, 1, 1, out, None, stats, table,
                                          1 if table else None, None, None, 1, 1, 1, gtable, ws,
                                          nbytes, d, 0, None)

    assert backward(desc(), nbytes=need - 1) == -4 and backward(desc(), ws=None) == -4
    assert backward(desc(), gout=None) == -3 and backward(desc(), stats=None) == -3
    assert backward(desc(), out=None) == -3 and backward(desc(table_size=0), table=None) == -3
    # nothing to do
    assert forward(desc(B=0)) == 0 and forward(desc(Lq=0)) == 0


def test_norm_refuses():
    lib = _lib.load()
    three = (_lib._i64 * 3)(64, 32, 16)

    def call(q=1, w=1, cos=1, out=1, B=1, L=2, Hq=2, Hk=1, D=16, F=8, places=2, eps=1e-6, dtype=0,
             stride=three):
        return lib.mcx_qk_norm_rotate_forward(q, 1, w, 1, cos, 1, None, out, 1, stride, three, B, L,
                                              Hq, Hk, D, F, places, eps, 0, dtype, None)

    for kw in (dict(D=0), dict(D=257), dict(F=9), dict(F=-1), dict(Hq=0), dict(B=-1), dict(eps=-1.),
               dict(eps=float("nan")), dict(places=-1), dict(L=1 << 40)):
        assert call(**kw) == -2, kw
    assert call(dtype=1) == -1
    for kw in (dict(q=None), dict(w=None), dict(cos=None), dict(out=None), dict(stride=None)):
        assert call(**kw) == -3, kw
    assert call(B=0) == 0 and call(L=0) == 0
    need = lib.mcx_qk_norm_rotate_backward_workspace(1, 2, 2, 1, 16, 0)
    assert need > 0
    assert lib.mcx_qk_norm_rotate_backward(1, 1, 1, 1, 1, 1, 1, 1, None, 1, 1, 1, 1, 1, need - 1,
                                           three, three, 1, 2, 2, 1, 16, 8, 2, 1e-6, 0, 0, None) == -4


def test_clip_refuses():
    import ctypes
    lib = _lib.load()
    one, size, kind = (ctypes.c_void_p * 1)(1), (_lib._i64 * 1)(5), (_lib._i32 * 1)(0)
    at = [ctypes.addressof(x) for x in (one, one, size, kind)]
    need = lib.mcx_clip_grad_norm_workspace(at[2], 1)
    assert need > 0
    assert lib.mcx_clip_grad_norm(*at, 1, -1.0, 1e-6, 1, 1, need, None) == -2
    assert lib.mcx_clip_grad_norm(*at, 1, 1.0, float("nan"), 1, 1, need, None) == -2
    assert lib.mcx_clip_grad_norm(*at, 1, 1.0, 1e-6, None, 1, need, None) == -3
    assert lib.mcx_clip_grad_norm(None, *at[1:], 1, 1.0, 1e-6, 1, 1, need, None) == -3
    assert lib.mcx_clip_grad_norm(*at, 1, 1.0, 1e-6, 1, 1, need - 1, None) == -4
    kind[0] = 1
    assert lib.mcx_clip_grad_norm(*at, 1, 1.0, 1e-6, 1, 1, need, None) == -1
    kind[0], size[0] = 0, -3
    assert lib.mcx_clip_grad_norm(*at, 1, 1.0, 1e-6, 1, 1, need, None) == -2


def test_python_refuses():
    q, k = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16)
    w, cos = torch.ones(16), torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        _C.qk_norm_rotate_forward(q, k, w, w, cos, cos)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        _C.relative_attention_forward(q, k, k)
    with pytest.raises(RuntimeError, match="4 dimensions"):
        _C.relative_attention_forward(q[0], k, k)
    with pytest.raises(RuntimeError, match="dimension 3"):
        _C.relative_attention_forward(q, k[..., :8], k)
    with pytest.raises(RuntimeError, match="dimension 1"):
        _C.relative_attention_forward(q, k, k[:, :4])
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        _C.relative_attention_forward(q.double(), k.double(), k.double())
    with pytest.raises(RuntimeError, match="key is"):
        _C.relative_attention_forward(q, k.bfloat16(), k)
    with pytest.raises(RuntimeError, match="dimension 1"):
        _C.qk_norm_rotate_forward(q, k[:, :4], w, w, cos, cos)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        _C.qk_norm_rotate_forward(q.half(), k.half(), w, w, cos, cos)
    with pytest.raises(RuntimeError, match="one GPU"):
        _C.clip_grad_norm([q], 1.0)
    with pytest.raises(RuntimeError, match="at least one"):
        _C.clip_grad_norm([], 1.0)
    with pytest.raises(RuntimeError, match="negative"):
        _C.clip_grad_norm([q], -1.0)
    with pytest.raises(RuntimeError, match="as many"):
        _C.clip_grad_norm([q], 1.0, out=[q, q])


def test_layers():
    norm = nn.QKNormRotation(16)
    assert set(norm.state_dict()) == {"query_weight", "key_weight"}
    buckets, zero = util.distance_buckets(16, reach=20)
    layer = nn.RelativeAttention(4, buckets, zero)
    assert set(layer.state_dict()) == {"table", "buckets"} and layer.table.shape == (4, 16)
    assert nn.RelativeAttention(4, buckets, zero, num_buckets=32).table.shape == (4, 32)
    assert nn.RelativeAttention(4).table is None
    with pytest.raises(AssertionError):
        nn.RelativeAttention(4, buckets.long(), zero)


def test_buckets_on_a_line():
    buckets, zero = util.distance_buckets(32, reach=128)
    assert buckets.dtype == torch.int32 and buckets.numel() == 257 and zero == 128
    assert buckets[zero] == 0 and buckets.min() == 0 and buckets.max() == 31
    for d in range(-128, 129):
        away, side = abs(d), 16 * (d > 0)
        want = away if away < 8 else min(15, 8 + int(math.log(away / 8) / math.log(16) * 8 + 1e-12))
        assert buckets[zero + d] == want + side, d


def test_buckets_on_a_circle():
    n = 50
    buckets, zero = util.distance_buckets(16, circle=n)
    assert zero == n - 1 and buckets.numel() == 2 * n - 1
    for a in range(n):
        for b in range(n):
            ahead = (b - a) % n
            # the same turn has the same bucket wherever the seam lies
            assert buckets[zero + b - a] == buckets[zero + ahead]
            side = 0 < ahead and 2 * ahead < n
            assert (int(buckets[zero + b - a]) >= 8) == side
    with pytest.raises(AssertionError):
        util.distance_buckets(16)
    with pytest.raises(AssertionError):
        util.distance_buckets(18, reach=5)


def test_rotation_table():
    cos, sin = util.rotation_table(10, 8)
    assert cos.shape == (10, 4) and cos.dtype == torch.float32
    assert torch.allclose(cos[3, 1].double(), torch.tensor(3 * 10000 ** -0.25, dtype=torch.float64).cos(), atol=1e-7)
    cos, sin = util.rotation_table(12, 6, circle=True)
    # turning on from the last place comes to the first
    step = torch.complex(cos[1], sin[1])
    assert torch.allclose(torch.complex(cos[11], sin[11]) * step, torch.complex(cos[0], sin[0]), atol=1e-6)


def test_clip_refuses_what_is_written_twice():
    a, b, none = torch.ones(5), torch.ones(5), torch.empty(0)
    for kw in (dict(tensors=[a, b, a]), dict(tensors=[a, b], out=[b, b.clone()]),
               dict(tensors=[a, b], out=[none.new_ones(5)] * 2), dict(tensors=[a, b, none], out=[b, a, none])):
        with pytest.raises(RuntimeError, match="twice|another one"):
            _C.clip_grad_norm(max_norm=1.0, **kw)
    # read twice, each its own, none with values: on to the next check
    for kw in (dict(tensors=[a, a], out=[b, b.clone()]), dict(tensors=[a, b], out=[a, b]),
               dict(tensors=[a, b], out=[a, b.clone()]), dict(tensors=[none, a, none.clone()])):
        with pytest.raises(RuntimeError, match="one GPU"):
            _C.clip_grad_norm(max_norm=1.0, **kw)


def test_parameters_that_share_a_gradient_are_clipped_once(monkeypatch):
    shared, other = torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(2))
    tied = torch.nn.Parameter(torch.ones(3))
    shared.grad, other.grad = torch.ones(3), torch.ones(2)
    tied.grad = shared.grad
    lists = []
    monkeypatch.setattr(_C, "clip_grad_norm", lambda ts, *rest, **kw: lists.append(ts))
    util.clip_grad_norm_([shared, other, shared, tied], 1.0)
    assert len(lists[0]) == 2 and lists[0][0] is shared.grad and lists[0][1] is other.grad


def test_norm_of_no_gradients_is_where_the_parameters_are():
    parameters = [torch.nn.Parameter(torch.ones(3, device="meta"))]
    norm = util.clip_grad_norm_(parameters, 1.0)
    assert norm.device == parameters[0].device and norm.dtype == torch.float32 and norm.dim() == 0
    assert util.clip_grad_norm_([], 1.0).item() == 0


@pytest.fixture
def without_kernels(monkeypatch):
    """Stand-ins of the operators that compute nothing: what the layers do around them."""
    asked = []

    def norm_back(gq, gk, q, k, wq, wk, *rest, needs=(True,) * 4, **kw):
        asked.append(tuple(needs))
        return [torch.ones_like(t) if n else None for t, n in zip((q, k, wq, wk), needs)]

    def attention_back(go, q, k, v, out, saved, table, *rest, needs, **kw):
        return [torch.ones_like(t) if t is not None and n else None for t, n in zip((q, k, v, table), needs)]

    monkeypatch.setattr(_C, "qk_norm_rotate_forward", lambda q, k, *rest, **kw: [q.clone(), k.clone()])
    monkeypatch.setattr(_C, "qk_norm_rotate_backward", norm_back)
    monkeypatch.setattr(_C, "relative_attention_forward",
                        lambda q, *rest, **kw: [q.clone(), [torch.zeros(1), None]])
    monkeypatch.setattr(_C, "relative_attention_backward", attention_back)
    return asked


def test_second_derivatives_are_refused(without_kernels):
    # a penalty on the gradient beside the loss itself: its part must not be left out silently
    q = torch.randn(1, 5, 2, 16).requires_grad_()
    cos = torch.ones(5, 8)
    for layer in (lambda x: nn.RelativeAttention(2)(x, x, x), lambda x: nn.QKNormRotation(16)(x, x, cos, cos)[0]):
        loss = layer(q).sum()
        gradient, = torch.autograd.grad(loss, q, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivatives"):
            (loss + gradient.square().sum()).backward()
        # a graph of the backward pass that nothing is asked of is no fault
        torch.autograd.grad(layer(q).square().sum(), q, create_graph=True)
        layer(q).sum().backward()


def test_example_keeps_its_angles_when_cast(without_kernels, monkeypatch):
    from mappedconvolutions_amd.examples import row_attention
    angles = []

    def norm(q, k, wq, wk, cos, sin, *rest, **kw):
        angles.append((cos, sin))
        return [q.clone(), k.clone()]

    monkeypatch.setattr(_C, "qk_norm_rotate_forward", norm)
    net = row_attention.RowNetwork(8, channels=16).to(torch.bfloat16)
    monkeypatch.setattr(net.convolution, "forward", lambda images, sample_map: images.expand(-1, 16, -1, -1))
    net(torch.randn(1, 1, 2, 8).bfloat16(), None)
    for got, want in zip(angles[0], util.rotation_table(8, 4, circle=True)):
        assert got.dtype == torch.float32 and torch.equal(got, want)


def test_norm_asks_for_the_gradients_that_are_wanted(without_kernels):
    norm, cos = nn.QKNormRotation(16), torch.ones(5, 8)
    q, k = torch.randn(1, 5, 2, 16).requires_grad_(), torch.randn(1, 5, 2, 16)
    norm.key_weight.requires_grad_(False)
    sum(t.sum() for t in norm(q, k, cos, cos)).backward()
    assert without_kernels == [(True, False, True, False)]


def test_norm_gradients_that_are_not_wanted():
    lib, three = _lib.load(), (_lib._i64 * 3)(64, 32, 16)

    def call(gq=1, wanted=(1, 1, 1, 1), ws=None, B=1):
        return lib.mcx_qk_norm_rotate_backward(gq, 1, 1, 1, 1, 1, 1, 1, None, *wanted, ws, 0, three, three,
                                               B, 2, 2, 1, 16, 8, 2, 1e-6, 0, 0, None)

    assert call(gq=None) == -3 and call() == -4
    # nothing to do
    assert call(wanted=(None,) * 4) == 0 and call(wanted=(1, 1, None, None), gq=None, B=0) == 0

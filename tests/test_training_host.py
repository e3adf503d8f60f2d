"""Host side of the recurrence, the group norm and the AdamW step: what the library and its Python
boundary refuse, layers' parameters, the optimizer's arguments.  Nothing here needs a GPU."""
import ctypes

import pytest
import torch

from mappedconvolutions_amd import _C, _lib, nn, util


def recurrence_desc(**kw):
    size = dict(B=2, L=9, C=16, v_stride=(144, 16), f_stride=(144, 16), g_stride=(144, 16), reverse=0)
    size.update(kw)
    d = _lib.RecurrenceDesc()
    for name, value in size.items():
        setattr(d, name, (_lib._i64 * 2)(*value) if isinstance(value, tuple) else value)
    return d


def recurrence(d, dtype=0, v=1, f=1, out=1, final=1, ws=None, nbytes=0):
    return _lib.load().mcx_gated_recurrence_forward(v, f, 1, None, None, out, final, None, ws, nbytes, d,
                                                    dtype, None)


@pytest.mark.parametrize("code, kw", [
    (-1, dict(dtype=1)), (-1, dict(dtype=7)), (-2, dict(B=-1)), (-2, dict(L=-1)), (-2, dict(C=0)),
    (-2, dict(C=(1 << 22) + 1)), (-2, dict(L=1 << 40)), (-2, dict(B=1 << 22, C=32)),
    (-2, dict(v_stride=(0, (1 << 22) + 1))), (-2, dict(f_stride=(0, -16))),
    (-3, dict(v=None)), (-3, dict(f=None)), (-3, dict(out=None)), (-3, dict(final=None)),
])
def test_recurrence_refuses(code, kw):
    outer = {n: kw.pop(n) for n in list(kw) if n in ("dtype", "v", "f", "out", "final")}
    assert recurrence(recurrence_desc(**kw), **outer) == code
    assert recurrence(None) == -3


def test_recurrence_workspace_and_spans():
    lib = _lib.load()
    long = recurrence_desc(B=1, L=100000)
    for dtype in (0, 2):
        need = lib.mcx_gated_recurrence_workspace(long, dtype)
        assert need > 0
        assert recurrence(long, dtype) == -4 and recurrence(long, dtype, ws=1, nbytes=need - 1) == -4
        assert lib.mcx_gated_recurrence_backward(1, None, 1, 1, 1, 1, None, 1, 1, 1, 1, 1, need - 1, long,
                                                 dtype, None) == -4
    assert lib.mcx_gated_recurrence_workspace(recurrence_desc(B=4096, L=512), 2) == 0
    assert lib.mcx_gated_recurrence_workspace(recurrence_desc(C=0), 0) == 0
    d = recurrence_desc()
    for kw in (dict(gout=None), dict(states=None), dict(v=None)):
        a = dict(gout=1, states=1, v=1)
        a.update(kw)
        assert lib.mcx_gated_recurrence_backward(a["gout"], None, a["v"], 1, 1, a["states"], None, 1, 1, 1, 1,
                                                 None, 0, d, 0, None) == -3
    # nothing to do
    assert recurrence(recurrence_desc(B=0)) == 0 and recurrence(recurrence_desc(L=0)) == 0
    assert lib.mcx_gated_recurrence_spans(0) == 0 and lib.mcx_gated_recurrence_spans(1) == 1
    assert lib.mcx_gated_recurrence_spans(-3) == 0


def test_group_norm_refuses():
    lib = _lib.load()
    two = (_lib._i64 * 2)(80, 16)

    def call(x=1, y=1, ws=1, nbytes=None, stride=two, B=2, N=5, C=16, G=4, eps=1e-5, act=0, dtype=0):
        need = lib.mcx_group_norm_workspace(B, N, C, G, 0, dtype)
        return lib.mcx_group_norm_forward(x, None, None, y, None, ws, need if nbytes is None else nbytes,
                                          stride, B, N, C, G, eps, act, dtype, None)

    for kw in (dict(B=-1), dict(N=-1), dict(C=0), dict(G=0), dict(G=3), dict(C=(1 << 20) + 16), dict(eps=-1.0),
               dict(eps=float("nan")), dict(act=3), dict(act=-1), dict(B=1 << 22), dict(N=1 << 33)):
        assert call(**kw) == -2, kw
    assert call(dtype=1) == -1
    for kw in (dict(x=None), dict(y=None), dict(stride=None)):
        assert call(**kw) == -3, kw
    need = lib.mcx_group_norm_workspace(2, 5, 16, 4, 0, 0)
    assert need > 0 and call(ws=None) == -4 and call(nbytes=need - 1) == -4
    assert call(B=0) == 0 and call(N=0) == 0
    assert lib.mcx_group_norm_workspace(2, 5, 16, 3, 0, 0) == 0

    def backward(gy=1, x=1, stats=1, gx=1, ws=1, nbytes=lib.mcx_group_norm_workspace(2, 5, 16, 4, 1, 0), act=0):
        return lib.mcx_group_norm_backward(gy, x, stats, None, None, gx, None, None, ws, nbytes, two, 2, 5, 16,
                                           4, act, 0, None)

    assert backward(gy=None) == -3 and backward(x=None) == -3 and backward(stats=None) == -3
    assert backward(ws=None) == -4 and backward(nbytes=10) == -4 and backward(act=9) == -2
    assert backward(gx=None) == 0  # nothing wanted


def test_adamw_refuses():
    lib = _lib.load()
    pointer, size, kind = (ctypes.c_void_p * 1)(8), (_lib._i64 * 1)(5), (_lib._i32 * 1)(0)
    p, n, k = (ctypes.addressof(x) for x in (pointer, size, kind))

    def call(lists=(p, p, p, p, p, p), count=1, sizes=n, types=k, **kw):
        o = dict(rate=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, max_norm=1.0, step=1, bits=32)
        o.update(kw)
        options = _lib.AdamWOptions()
        for name, value in o.items():
            setattr(options, name, value)
        return lib.mcx_adamw_step(*lists, sizes, types, types, count, options, None)

    for kw in (dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=float("nan")), dict(eps=-1.0),
               dict(weight_decay=-1.0), dict(bits=16), dict(step=0), dict(rate=float("inf")),
               dict(rate=float("nan")), dict(count=-1), dict(grad_norm=1, max_norm=-1.0)):
        assert call(**kw) == -2, kw
    assert lib.mcx_adamw_step(p, p, p, p, p, p, n, k, k, 1, None, None) == -3
    for i in range(4):
        assert call(lists=tuple(None if i == j else p for j in range(6))) == -3
    assert call(lists=(p, p, p, p, None, p), bits=8) == -3
    assert call(sizes=None) == -3 and call(types=None) == -3
    kind[0] = 1
    assert call() == -1
    kind[0], size[0] = 0, -2
    assert call() == -2
    size[0], pointer[0] = 5, None
    assert call() == -3
    size[0] = 0
    assert call() == 0 and call(count=0) == 0
    assert lib.mcx_adamw_moment(None, 1, 1, 5, 0, 0, None) == -3
    assert lib.mcx_adamw_moment(1, 1, 1, 5, 0, 1, None) == -1
    assert lib.mcx_adamw_moment(1, 1, 1, -5, 0, 0, None) == -2
    assert lib.mcx_adamw_moment(None, None, None, 0, 0, 0, None) == 0


def test_python_refuses():
    x = torch.zeros(2, 5, 16)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        _C.gated_recurrence_forward(x, x)
    with pytest.raises(RuntimeError, match="3 dimensions"):
        _C.gated_recurrence_forward(x[0], x[0])
    with pytest.raises(RuntimeError, match="shape"):
        _C.gated_recurrence_forward(x, x[:, :4])
    with pytest.raises(RuntimeError, match="gate is"):
        _C.gated_recurrence_forward(x, x, x.bfloat16())
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        _C.gated_recurrence_forward(x.double(), x.double())
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        _C.group_norm_forward(x, 4)
    with pytest.raises(RuntimeError, match="3 dimensions"):
        _C.group_norm_forward(x[0], 4)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        _C.group_norm_forward(x.half(), 4)
    with pytest.raises(RuntimeError, match="weight is"):
        _C.group_norm_forward(x, 4, torch.ones(16, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="one GPU"):
        _C.grad_norm([x])
    with pytest.raises(RuntimeError, match="at least one"):
        _C.grad_norm([])
    with pytest.raises(RuntimeError, match="one GPU"):
        _C.adamw_step([x], [x], [x], [x], 1, 1e-3)
    _C.adamw_step([], [], [], [], 1, 1e-3)  # nothing to do
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0),
               dict(first_scales=[x]), dict(max_norm=1.0), dict(grad_norm=x, max_norm=-1.0)):
        with pytest.raises(RuntimeError):
            _C.adamw_step([x], [x], [x], [x], 1, 1e-3, **kw)
    for step, lr in ((0, 1e-3), (-1, 1e-3), (1, float("nan")), (1, float("inf"))):
        with pytest.raises(RuntimeError):
            _C.adamw_step([x], [x], [x], [x], step, lr)
    with pytest.raises(RuntimeError, match="as many"):
        _C.adamw_step([x], [x, x], [x], [x], 1, 1e-3)


def test_layers():
    norm = nn.GroupNormActivation(4, 12, activation="silu")
    assert tuple(norm.weight.shape) == (12,) and (norm.weight == 1).all() and (norm.bias == 0).all()
    assert set(norm.state_dict()) == {"weight", "bias"}
    assert not list(nn.GroupNormActivation(4, 12, affine=False).parameters())
    with pytest.raises(AssertionError):
        nn.GroupNormActivation(5, 12)
    with pytest.raises(AssertionError):
        nn.GroupNormActivation(4, 12, activation="tanh")
    with pytest.raises(AssertionError):
        norm(torch.zeros(2, 5, 8))
    assert not list(nn.GatedRecurrence().parameters())
    with pytest.raises(AssertionError):
        nn.GatedRecurrence(reverse=True).step(torch.zeros(1, 4), *torch.zeros(2, 1, 1, 4))


def test_optimizer_arguments():
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError):
        util.AdamW([p], bits=16)
    with pytest.raises(ValueError):
        util.AdamW([])
    optimizer = util.AdamW([p], lr=0.5, bits=8)
    assert optimizer.step() is None  # no gradients yet
    assert optimizer.step(lambda: 7) == 7
    assert not optimizer.state and optimizer.param_groups[0]["bits"] == 8


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_is_not_counted(capturable, monkeypatch):
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    opt = util.AdamW([p], capturable=capturable)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="one GPU"):
            opt.step()
        assert int(opt.state[p]["step"]) == 0
    # a first step that would be captured leaves nothing behind
    opt = util.AdamW([p], capturable=capturable)
    for name in ("is_initialized", "is_current_stream_capturing"):
        monkeypatch.setattr(torch.cuda, name, lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    monkeypatch.undo()
    assert opt.state_dict()["state"] == {}
    assert util.AdamW([p]).load_state_dict(opt.state_dict()) is None


@pytest.mark.parametrize("capturable", [False, True])
def test_nothing_is_launched_before_all_is_checked(capturable, monkeypatch):
    params = [torch.nn.Parameter(torch.zeros(n)) for n in (3, 4, 5)]
    for p in params:
        p.grad = torch.ones_like(p)
    opt = util.AdamW([dict(params=params[:2]), dict(params=params[2:], lr=0.5)], capturable=capturable)
    seen = []

    def checked(ps, grads, first, second, step, lr, *rest, **kw):
        if lr == 0.5 and refuse:
            raise RuntimeError("refused")
        seen.append("checked")
        return lambda: seen.append("launched")

    monkeypatch.setattr(_C, "_adamw_call", checked)
    refuse = True
    with pytest.raises(RuntimeError, match="refused"):
        opt.step()
    assert seen == ["checked"] and [int(opt.state[p]["step"]) for p in params] == [0, 0, 0]
    refuse = False
    opt.step()
    assert seen[1:] == ["checked", "checked", "launched", "launched"]
    assert [int(opt.state[p]["step"]) for p in params] == [1, 1, 1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_moments_keep_their_types_under_another_default(dtype):
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        p = torch.nn.Parameter(torch.zeros(300, dtype=torch.float32))
        p.grad = torch.ones_like(p)
        opt = util.AdamW([p], bits=8)
        with pytest.raises(RuntimeError, match="one GPU"):
            opt.step()
    finally:
        torch.set_default_dtype(before)
    assert {n: t.dtype for n, t in opt.state[p].items() if isinstance(t, torch.Tensor)} == dict(
        first=torch.uint8, second=torch.uint8, first_scale=torch.float32, second_scale=torch.float32)


def test_a_group_of_other_bits_is_refused():
    a, b = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    with pytest.raises(ValueError, match="32 or 8"):
        util.AdamW([dict(params=[a]), dict(params=[b], bits=16)])
    opt = util.AdamW([a], bits=8)
    with pytest.raises(ValueError, match="32 or 8"):
        opt.add_param_group(dict(params=[b], bits=4))
    opt.add_param_group(dict(params=[b], bits=32))
    assert [g["bits"] for g in opt.param_groups] == [8, 32]

"""The attention layers, clipping over parameters, and the example that runs them together."""
import pytest
import torch

from mappedconvolutions_amd import _C, nn, util
from mappedconvolutions_amd.examples import row_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layers_pass_gradients_to_float32_parameters(device, dtype):
    torch.manual_seed(0)
    buckets, zero = util.distance_buckets(16, circle=40)
    norm = nn.QKNormRotation(32).to(device)
    layer = nn.RelativeAttention(4, buckets, zero).to(device)
    cos, sin = util.rotation_table(40, 32, circle=True, device=device)
    packed = torch.randn(3, 40, 8, 32, device=device).to(dtype).requires_grad_()
    q, k, v = packed.split([4, 2, 2], 2)
    out = layer(*norm(q, k, cos, sin), v)
    g = torch.randn_like(out)
    out.backward(g)
    # the same by the operators
    w = [p.to(dtype) for p in (norm.query_weight, norm.key_weight)]
    nq, nk = _C.qk_norm_rotate_forward(q, k, *w, cos, sin)
    args = dict(bias_table=layer.table.to(dtype), buckets=buckets.to(device), bucket_zero=zero)
    want, saved = _C.relative_attention_forward(nq, nk, v, for_backward=True, **args)
    assert torch.equal(out, want)
    gq, gk, gv, gt = _C.relative_attention_backward(g, nq, nk, v, want, saved, **args)
    gq, gk, gqw, gkw = _C.qk_norm_rotate_backward(gq, gk, q, k, *w, cos, sin)
    assert torch.equal(packed.grad, torch.cat((gq, gk, gv), 2))
    assert layer.table.grad.dtype == torch.float32
    assert torch.equal(layer.table.grad, gt.float())
    assert torch.equal(norm.query_weight.grad, gqw.float())
    assert torch.equal(norm.key_weight.grad, gkw.float())


def test_no_gradients_wanted(device):
    layer = nn.RelativeAttention(2).to(device)
    q = torch.randn(1, 9, 2, 16, device=device)
    assert not layer(q, q, q).requires_grad
    v = q.clone().requires_grad_()
    layer(q, q, v).sum().backward()
    assert torch.isfinite(v.grad).all()


def test_refusals_on_the_gpu(device):
    q, k = torch.zeros(2, 5, 4, 16, device=device), torch.zeros(2, 5, 2, 16, device=device)
    table, buckets = torch.zeros(4, 8, device=device), torch.zeros(5, dtype=torch.int32, device=device)
    bad = [
        dict(bias_table=table), dict(buckets=buckets),
        dict(bias_table=table[:2], buckets=buckets), dict(bias_table=table, buckets=buckets.long()),
        dict(bias_table=table, buckets=buckets, bucket_zero=5),
        dict(bias_table=torch.zeros(4, 513, device=device), buckets=buckets),
        dict(bias_table=table.bfloat16(), buckets=buckets),
        dict(bias_table=table, buckets=buckets.cpu()),
        dict(key_lengths=torch.zeros(2, dtype=torch.int64, device=device)),
        dict(query_start=torch.zeros(3, dtype=torch.int32, device=device)),
        dict(scale=0.0), dict(scale=float("inf")),
    ]
    for kw in bad:
        with pytest.raises(RuntimeError):
            _C.relative_attention_forward(q, k, k, **kw)
    with pytest.raises(RuntimeError):
        _C.relative_attention_forward(torch.zeros(2, 5, 3, 16, device=device), k, k)
    wide = torch.zeros(1, 2, 1, 136, device=device)
    with pytest.raises(RuntimeError, match="128"):
        _C.relative_attention_forward(wide, wide, wide)
    out, saved = _C.relative_attention_forward(q, k, k, for_backward=True)
    for worse in (None, [None, None], [saved[0][:, :2], None], [saved[0].double(), None]):
        with pytest.raises(RuntimeError):
            _C.relative_attention_backward(out, q, k, k, out, worse)
    w, cos = torch.ones(16, device=device), torch.zeros(5, 8, device=device)
    for args in ((q, k, w[:8], w, cos, cos), (q, k, w, w, cos.double(), cos),
                 (q, k, w, w, cos, cos[:3]), (q, k, w, w, cos[:3], cos[:3]),
                 (q, k, w, w, cos, cos, torch.zeros(2, 5, dtype=torch.int32, device=device)),
                 (q, k, w, w, cos, cos, None, -1.0), (q, k, w.bfloat16(), w, cos, cos)):
        with pytest.raises(RuntimeError):
            _C.qk_norm_rotate_forward(*args)
    with pytest.raises(RuntimeError, match="contiguous"):
        _C.clip_grad_norm([q.transpose(1, 2)], 1.0)
    with pytest.raises(RuntimeError, match="dtype"):
        _C.clip_grad_norm([q.double()], 1.0)
    with pytest.raises(RuntimeError, match="sizes"):
        _C.clip_grad_norm([q], 1.0, out=[k])
    with pytest.raises(RuntimeError, match="one GPU"):
        _C.clip_grad_norm([q, q.cpu()], 1.0)


def test_clipping_parameters(device):
    torch.manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(s, device=device)) for s in ((3, 5), (7,), (4, 6, 2, 2))]
    for p in params[:2]:
        p.grad = torch.randn_like(p)
    params[2].grad = torch.randn_like(params[2]).contiguous(memory_format=torch.channels_last)
    params.append(torch.nn.Parameter(torch.zeros(3, device=device)))  # without a gradient
    before = [p.grad.clone() for p in params[:3]]
    norm = util.clip_grad_norm_(params, 0.5)
    want = torch.sqrt(sum(g.double().square().sum() for g in before))
    assert abs(norm.item() - want.item()) < 1e-6 * want.item()
    for p, g in zip(params, before):
        assert torch.allclose(p.grad, g * (0.5 / want.item()), rtol=1e-5, atol=0)
    assert util.clip_grad_norm_(params[3], 1.0).item() == 0


def test_example_learns(device):
    losses = row_attention.train(steps=40)
    # the pixels are independent with variance one: guessing costs 1
    assert losses[-1] < 0.6 * losses[0] and losses[-1] < 0.8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_example_serves(device, dtype):
    whole, one_by_one = row_attention.serve(dtype=dtype)
    # the same numbers but for the order of sums; in bf16 two roundings of each value (2^-8 of values
    # up to 4, after a product over 128 channels that may turn one rounding into another)
    bound = 1e-4 if dtype == torch.float32 else 6e-2
    assert (whole - one_by_one).abs().max().item() <= bound


def test_nothing_is_saved_without_a_graph(device, monkeypatch):
    asked, forward = [], _C.relative_attention_forward

    def watched(*args, for_backward=False, **kw):
        asked.append(for_backward)
        return forward(*args, for_backward=for_backward, **kw)

    monkeypatch.setattr(_C, "relative_attention_forward", watched)
    buckets, zero = util.distance_buckets(8, reach=20)
    layer = nn.RelativeAttention(2, buckets, zero).to(device)
    q = torch.randn(1, 9, 2, 16, device=device)
    with torch.no_grad():
        served = layer(q, q, q)
    assert torch.equal(layer(q, q, q), served)
    assert asked == [False, True]


def test_example_trains_in_bfloat16(device):
    torch.manual_seed(3)
    net = row_attention.RowNetwork(64).to(device, torch.bfloat16)
    sample_map = util.latitude_map(16, 64).to(device)
    optimizer = torch.optim.Adam(net.parameters(), lr=3e-3)
    losses = []
    for _ in range(40):
        images = torch.randn(4, 1, 16, 64, device=device, dtype=torch.bfloat16)
        optimizer.zero_grad()
        loss = (net(images, sample_map).float() - images[:, 0].float().roll(16, -1)).square().mean()
        loss.backward()
        assert util.clip_grad_norm_(net.parameters(), 1.0).isfinite()
        optimizer.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    assert losses[-1] < 0.8 * losses[0]

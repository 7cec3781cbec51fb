"""The attention modules' need_weights=False form (ops.attention, ops.add_layer_norm) against their weight-returning form and
against the block's arithmetic in 64 bits; the operators run together as an encoder block with a position bias."""
import math

import pytest
import torch
import torch.nn.functional as F

import sequence_reference as ref

pytestmark = pytest.mark.gpu


def close(a, b, tol, what=""):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape and (a - b).abs().max() <= tol * max(b.abs().max().item(), 1e-3), (what, (a - b).abs().max().item())


@pytest.mark.parametrize("shape", [(2, 70, 48), (2, 3, 70, 48)])
def test_scaled_dot_product_attention(shape):
    from ocean.models.components import ScaledDotProductAttention
    g = torch.Generator(device="cuda").manual_seed(1)
    m = ScaledDotProductAttention(48).cuda().eval()
    mask = torch.rand(2, *([1] if len(shape) == 4 else []), 70, 70, device="cuda", generator=g) < 0.7
    mask[..., torch.arange(70), torch.arange(70)] = True
    a, b = ([torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(s)).requires_grad_(True) for s in (2, 3, 4)] for _ in range(2))
    w = torch.randn(*shape, device="cuda", generator=g)
    out, none = m(*a, mask, need_weights=False)
    want, weights = m(*b, mask)
    assert none is None and weights is not None
    close(out, want, 1e-5)
    for x, y in zip(torch.autograd.grad(out, a, w), torch.autograd.grad(want, b, w)):
        close(x, y, 1e-4)


def block64(sd, x, y, heads, ok, bias=None, norms=True):
    """CrossModalAttention.forward (multi_factor_attention.py:190-215) in fp64"""
    D = x.shape[-1]
    d = D // heads
    lin = lambda n, t: F.linear(t, sd[n + ".weight"], sd[n + ".bias"])
    split = lambda t: t.view(t.shape[0], t.shape[1], heads, d).transpose(1, 2)
    p = "multihead_attention." if norms else ""
    q, k, v = split(lin(p + "w_q", x)), split(lin(p + "w_k", y)), split(lin(p + "w_v", y))
    s = q @ k.transpose(2, 3) / math.sqrt(d)
    if bias is not None:
        s = s + bias
    a = torch.softmax(s.masked_fill(~ok, -math.inf), -1) @ v
    a = lin(p + "w_o", a.transpose(1, 2).reshape(x.shape))
    if not norms:
        return a
    y1 = F.layer_norm(x + a, (D,), sd["layer_norm.weight"], sd["layer_norm.bias"])
    h = lin("feed_forward.3", torch.relu(lin("feed_forward.0", y1)))
    return F.layer_norm(y1 + h, (D,), sd["ff_layer_norm.weight"], sd["ff_layer_norm.bias"])


@pytest.mark.parametrize("D,heads,Lq,Lk", [(128, 8, 100, 100), (256, 2, 40, 1500), (1280, 10, 33, 70)])
def test_cross_modal_block(D, heads, Lq, Lk):
    """fp32 through four linear layers and two norms: outputs 1e-4 of their size, gradients 1e-3 as for the other form."""
    from ocean.models.components import CrossModalAttention
    torch.manual_seed(D)
    m = CrossModalAttention(D, heads, dropout=0.1).cuda().eval()
    sd = {k: v.detach().double().requires_grad_(True) for k, v in m.state_dict().items()}
    x, y = torch.randn(2, Lq, D, device="cuda"), torch.randn(2, Lk, D, device="cuda")
    n = torch.tensor([Lk, Lk // 3], dtype=torch.int32, device="cuda")
    ok, _ = ref.places(2, heads, Lq, Lk, lengths=n)
    xr, yr = (t.double().requires_grad_(True) for t in (x, y))
    want = block64(sd, xr, yr, heads, ok.cuda())
    xg, yg = (t.clone().requires_grad_(True) for t in (x, y))
    out, none = m(xg, yg, need_weights=False, key_lengths=n)
    assert none is None
    close(out, want, 1e-4)
    w = torch.randn(2, Lq, D, device="cuda")
    (want * w.double()).sum().backward()
    (out * w).sum().backward()
    close(xg.grad, xr.grad, 1e-3, "query")
    close(yg.grad, yr.grad, 1e-3, "key and value")
    for name, prm in m.named_parameters():
        # a constant on every key changes no softmax: the key projection's bias has no gradient but rounding
        if name.endswith("w_k.bias"):
            assert prm.grad.abs().max() <= 1e-4 * m.multihead_attention.w_k.weight.grad.abs().max()
        else:
            close(prm.grad, sd[name].grad, 1e-3, name)


def test_encoder_block_with_a_position_bias_trains_and_serves():
    """Attention with the bias, residual norm, and their gradients together, then the last position alone over the same keys."""
    from ocean import ops
    from ocean.models.components import MultiHeadAttention
    torch.manual_seed(3)
    B, L, D, H = 2, 90, 64, 4
    m = MultiHeadAttention(D, H, dropout=0.0).cuda()
    table = torch.nn.Parameter(0.3 * torch.randn(32, H, device="cuda"))
    weight, bias = torch.nn.Parameter(torch.rand(D, device="cuda") + 0.5), torch.nn.Parameter(torch.randn(D, device="cuda"))
    x = torch.randn(B, L, D, device="cuda", requires_grad=True)
    n = torch.tensor([90, 41], dtype=torch.int32, device="cuda")
    a, _ = m(x, x, x, need_weights=False, key_lengths=n, causal=True, position_table=table, bidirectional=False, max_distance=64)
    y, s = ops.add_layer_norm(x, a, weight, bias)
    w = torch.randn(B, L, D, device="cuda")
    leaves = [x, table, weight, bias, m.w_q.weight, m.w_v.bias]
    got = torch.autograd.grad(((y + 0.1 * s) * w).sum(), leaves)
    sd = {k: v.detach().double() for k, v in m.state_dict().items()}
    r = [t.detach().double().requires_grad_(True) for t in leaves]
    sd["w_q.weight"], sd["w_v.bias"] = r[4], r[5]
    ok, dist = ref.places(B, H, L, L, causal=True, lengths=n)
    lut = torch.tensor([ref.bucket(d, 32, 64, False) for d in range(-L, L + 1)], device="cuda")
    b64 = r[1][lut[dist.cuda() + L]].permute(0, 3, 1, 2)
    a64 = block64(sd, r[0], r[0], H, ok.cuda(), b64, norms=False)
    s64 = r[0] + a64
    want = torch.autograd.grad(((F.layer_norm(s64, (D,), r[2], r[3]) + 0.1 * s64) * w.double()).sum(), r)
    close(s, s64, 1e-5)
    for g, h, name in zip(got, want, ("x", "table", "weight", "bias", "w_q", "w_v.bias")):
        close(g, h, 1e-3, name)
    with torch.no_grad():
        last = torch.stack([x[i, int(n[i]) - 1] for i in range(B)]).unsqueeze(1)
        one, _ = m(last, x, x, need_weights=False, key_lengths=n, causal=True, query_start=n - 1, position_table=table, bidirectional=False, max_distance=64)
        for i in range(B):
            close(one[i, 0], a[i, int(n[i]) - 1], 1e-5)


def test_refusals():
    from ocean.models.components import CrossModalAttention, MultiHeadAttention, ScaledDotProductAttention
    x = torch.randn(2, 5, 32, device="cuda")
    for m in (ScaledDotProductAttention(32, 0.1).cuda().train(), MultiHeadAttention(32, 4, 0.1).cuda().train()):
        with pytest.raises(NotImplementedError):
            m(x, x, x, need_weights=False)
        with pytest.raises(ValueError):
            m(x, x, x, causal=True)
    with pytest.raises(NotImplementedError):
        CrossModalAttention(32, 4, 0.1).cuda().train()(x, x, need_weights=False)
    with pytest.raises(RuntimeError):
        MultiHeadAttention(32, 4).cuda().eval()(x, x[:1], x[:1], need_weights=False)


def test_second_derivatives_are_refused():
    from ocean.models.components import MultiHeadAttention
    m = MultiHeadAttention(32, 2, dropout=0.0).cuda()
    x = torch.randn(1, 5, 32, device="cuda")
    for p in m.parameters():
        p.requires_grad_(False)
    m.w_o.weight.requires_grad_(True)                       # its projection alone is on the way back
    with pytest.raises(RuntimeError, match="differentiated"):
        torch.autograd.grad(m(x, x, x, need_weights=False)[0].square().sum(), m.w_o.weight, create_graph=True)

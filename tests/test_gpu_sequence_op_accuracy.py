"""Digits that the sequence operators' kernels take care to keep, at the level of fp32 sums."""
import math

import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu


def plain_table_grad(q, k, v, table, dout, at, ok, scale):
    """The position table's gradient by the formulas in fp32, summed in 64 bits: [buckets, H]."""
    q, k, v, do = (t.detach().float().contiguous() for t in (q, k, v, dout))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale + table.detach()[at].permute(0, 3, 1, 2)
    s = s.masked_fill(~ok, -math.inf)
    p = torch.softmax(s, -1)
    o = torch.matmul(p, v)
    ds = p * (torch.matmul(do, v.transpose(2, 3).contiguous()) - (do * o).sum(-1, keepdim=True))
    return ref.table_grad(ds.double(), at, table.shape[0])


@pytest.mark.parametrize("B,H,L,lengths", [(16, 4, 512, True),       # many rows: an error to one side grows with them, rounding with their root
                                           (1, 1, 4096, False)])     # few tiles: the launch over queries is split, and its deltas joined
def test_position_bias_gradient_in_bf16_is_that_of_fp32_formulas(B, H, L, lengths):
    """Inputs in bf16 are exact, and this gradient is fp32 throughout: its distance from 64 bits has to be that of the formulas
    evaluated in fp32, within a factor of two for another order of the sums.  A delta from the rounded output would be some 2^-9
    / 2^-24 times as far off; products that start their sums elsewhere in one of the two launches three times."""
    from ocean import ops
    d, buckets, far = 64, 32, 128
    g = torch.Generator(device="cuda").manual_seed(L)
    q, k, v, dout = (torch.randn(B, L, H, d, device="cuda", generator=g).bfloat16().transpose(1, 2) for _ in range(4))
    table = (0.5 * torch.randn(buckets, H, device="cuda", generator=g)).requires_grad_(True)
    n = torch.tensor([L - b * L // (3 * B) for b in range(B)], dtype=torch.int32, device="cuda") if lengths else None
    ok, dist = ref.places(B, H, L, L, lengths=n)
    bias, at = ref.bias_of(table, dist, buckets, far, True)
    at = at.cuda()
    exact = ref.table_grad(ref.attention(q, k, v, ok, 1 / math.sqrt(d), dout, bias)["ds"], at, buckets)
    plain = plain_table_grad(q, k, v, table, dout, at, ok.cuda(), 1 / math.sqrt(d))
    got = torch.autograd.grad(ops.attention(q, k, v, key_lengths=n, position_table=table, max_distance=far), table, dout)[0].double()
    off, allowed = (got - exact).norm().item(), 2 * (plain - exact).norm().item()
    print(f"{off / exact.norm().item():.2e} of the norm, plain {allowed / 2 / exact.norm().item():.2e}")
    assert off <= allowed


@pytest.mark.parametrize("W", [24, 250, 1000, 6000, 20000])
def test_layer_norm_keeps_the_deviation_of_rows_far_from_zero(W):
    """Rows at 4096 with deviation 1.  A mean of at most 48 additions deep (16 in a lane, 16 waves, 6 steps between lanes, or 20 in a
    lane of the widest) is 48 half steps of 4096 off at most, e; x - mean is exact, so the rows' variance is too large by e^2 and
    48 half steps at most, and every y shifts by the same e / deviation."""
    from ocean import ops
    u = 2.0 ** -24
    x = torch.randn(50, W, device="cuda", generator=torch.Generator(device="cuda").manual_seed(W)) + 4096.0
    y = ops.layer_norm(x, eps=1e-5).double()
    xc = x.double() - x.double().mean(-1, keepdim=True)
    var = (xc * xc).mean(-1, keepdim=True)
    rstd = 1.0 / (var + 1e-5).sqrt()
    e = 48 * u * (4096.0 + 8.0)
    shift = y.mean(-1, keepdim=True)
    assert (shift.abs() <= e * rstd + u).all()
    rel = (e * e / var + 48 * u) / 2 + 4 * u                 # of the deviation's inverse; its root, quotient and product
    assert ((y - shift - xc * rstd).abs() <= rel * (xc * rstd).abs() + (rel + u) * e * rstd + u * y.abs() + 2 * u).all()


@pytest.mark.parametrize("B,H,Hk,Lq,Lk,d", [(1, 8, 2, 1, 257, 64), (3, 8, 1, 1, 5000, 128), (2, 4, 2, 9, 777, 40)])
def test_single_tokens_in_bf16_round_once(B, H, Hk, Lq, Lk, d):
    """The weights of few queries keep 16 bits (2^-16 of each), so only the output's own rounding is a bf16 one."""
    from ocean import ops
    g = torch.Generator(device="cuda").manual_seed(Lk)
    q, k, v = (torch.randn(B, h, n, d, device="cuda", generator=g).bfloat16() for h, n in ((H, Lq), (Hk, Lk), (Hk, Lk)))
    ok, _ = ref.places(B, H, Lq, Lk)
    r = ref.attention(q, k, v, ok, 1 / math.sqrt(d))
    limit = ref.tolerance("out", r, torch.float32, d, Lk) + 2.0 ** -16 * r["mag"]["out"]
    limit = limit + 2.0 ** -8 * (r["out"].abs() + limit)
    err = (ops.attention(q, k, v).double() - r["out"]).abs()
    assert (err <= limit).all(), f"{(err / limit).amax().item():.3g} times the bound"

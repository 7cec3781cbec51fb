"""The largest and smallest that the sequence operators take, and what they answer beyond."""
import ctypes

import pytest
import torch

from ocean import _hip
from test_sequence_op_refusals import attention_shape


@pytest.mark.parametrize("change,forward,backward", [
    (dict(B=1 << 24, H=1, Hk=1, Lq=1, Lk=1), 2, 2), (dict(B=(1 << 24) - 1, H=1, Hk=1, Lq=1, Lk=1), 4, 4), (dict(B=1 << 20, H=16, Hk=16, Lq=64, Lk=64), 2, 2),
    (dict(B=1 << 21, H=8, Hk=1, Lq=16, Lk=16), 2, 2), (dict(B=1 << 21, H=8, Hk=1, Lq=4, Lk=16), 4, 2), (dict(B=1, H=1, Hk=1, Lq=40, Lk=1 << 30), 4, 4),
    (dict(B=3, H=1, Hk=1, Lq=40, Lk=1 << 30), 4, 2), (dict(B=1, H=1, Hk=1, Lq=1 << 30, Lk=5), 4, 4), (dict(B=1, H=2, Hk=2, Lq=1 << 30, Lk=5, causal=1), 2, 2)])
def test_more_blocks_than_a_grid_has_threads_for(change, forward, backward):
    """2^24 blocks of 256 threads are 2^32, where a grid wraps around without an error.  A forward call that leaves lse is one that
    a backward call follows."""
    L, s = _hip.lib(), attention_shape(**change)
    none, lse = [None] * 7, ctypes.c_void_p(64)
    assert L.ocean_attention_fwd(ctypes.byref(s), *none, None, 0, None, None, None) == forward
    assert L.ocean_attention_fwd(ctypes.byref(s), *none, None, 0, None, lse, None) == max((forward, backward), key=lambda x: x == 2)
    assert L.ocean_attention_bwd(ctypes.byref(s), *none, None, None, None, None, 0, None, None, None, None, None) == backward


@pytest.mark.parametrize("scale,status", [(0.0, 1), (9e-31, 1), (1e-38, 1), (1.1e30, 1), (2.5e38, 1), (1e-30, 4), (1e30, 4)])
def test_scales_whose_log2_form_or_inverse_is_not_finite(scale, status):
    L, s = _hip.lib(), attention_shape(scale=scale)
    none = [None] * 7
    assert L.ocean_attention_fwd(ctypes.byref(s), *none, None, 0, None, None, None) == status
    assert L.ocean_attention_bwd(ctypes.byref(s), *none, None, None, None, None, 0, None, None, None, None, None) == status


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_smallest_scale(dtype):
    """Weights are all 1 / 200: the output is the values' mean and dv the gradient's."""
    from ocean import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    leaves = [torch.randn(1, 2, 200, 32, device="cuda", generator=g).to(dtype).requires_grad_(True) for _ in range(3)]
    w = torch.randn(1, 2, 200, 32, device="cuda", generator=g).to(dtype)
    for scale in (1e-38, 2.5e38):
        with pytest.raises(ValueError):
            ops.attention(*leaves, scale=scale)
    out = ops.attention(*leaves, scale=1e-30)
    u = torch.finfo(dtype).eps / 2                           # of the weights and of the result; 232 half steps of a sum of 200
    for got, x in ((out, leaves[2]), (torch.autograd.grad(out, leaves, w)[2], w)):
        x = x.detach().double()
        size = x.abs().mean(2, keepdim=True)
        assert ((got.double() - x.mean(2, keepdim=True)).abs() <= (232 * 2.0 ** -24 + 2 * u) * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lq", [1, 150])
def test_scaled_scores_of_nine_hundred_millions(dtype, Lq):
    """One key at 9.1e8, the others at half: its weight is 1, and the remaining exponent, a rounding of 1.3e9, is 64 at most."""
    from ocean import ops
    q = torch.full((1, 2, Lq, 32), 2.0 ** 14, device="cuda", dtype=dtype)
    k = torch.full((1, 1, 300, 32), 2.0 ** 9, device="cuda", dtype=dtype)
    k[:, :, 170] *= 2
    v = torch.randn(1, 1, 300, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    out = ops.attention(q, k, v, scale=1.7).double()
    want = v[:, :, 170:171].double()                         # (e v) / e: three roundings and their products, in bf16 of e and out too
    assert ((out - want).abs() <= (4 * 2.0 ** -24 + (0 if dtype == torch.float32 else 2.01 * 2.0 ** -8)) * want.abs()).all()


@pytest.mark.gpu
def test_the_largest_batch():
    from ocean import ops
    B = (1 << 24) - 1
    q, k, v, w = (torch.randn(8, device="cuda").bfloat16().expand(B, 1, 1, 8).contiguous() for _ in range(4))
    v[-1], w[-1] = 7.0, 5.0
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = ops.attention(*leaves)                             # one key: its weight is 1
    assert torch.equal(out, v)
    dq, dk, dv = torch.autograd.grad(out, leaves, w)
    # ds = p (dp - p dp) with p off from 1 by the rounding of the score t < 20 and of 2^x, (t + 2) 2^-24 at most; |dp| <= 280
    assert torch.equal(dv, w) and max(dq.abs().max(), dk.abs().max()) <= 22 * 2.0 ** -24 * 280 / 8 ** 0.5 * max(q.abs().max(), k.abs().max())
    with pytest.raises(_hip.OceanHipError, match="unsupported size"):
        one = q.detach()[:1].expand(B + 1, 1, 1, 8)
        ops.attention(one, one, one)


@pytest.mark.gpu
def test_a_large_batch_of_single_tokens_with_shared_key_heads():
    """2^24 query heads on 2^21 key heads: the forward call alone takes them, one that gradients follow does not."""
    from ocean import ops
    B = 1 << 21
    q = torch.randn(B, 8, 1, 8, device="cuda").bfloat16()
    k, v = (torch.randn(B, 1, 1, 8, device="cuda").bfloat16() for _ in range(2))
    assert torch.equal(ops.attention(q, k, v), v.expand(B, 8, 1, 8))
    with pytest.raises(_hip.OceanHipError, match="unsupported size"):
        ops.attention(q.requires_grad_(True), k, v)

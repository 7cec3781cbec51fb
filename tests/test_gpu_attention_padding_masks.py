"""Padding masks of ops.attention where the axis they do not have has one place anyway: one query over a padded cache, one key."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def spoiled(t, gone, fill):
    return t.masked_fill(gone, fill)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Hk,Lk", [(3, 4, 2, 130), (2, 2, 2, 1), (1, 1, 1, 70), (2, 8, 1, 2000)])
def test_one_query_reads_no_key_that_a_padding_mask_takes(dtype, B, H, Hk, Lk):
    from ocean import ops
    g = torch.Generator(device="cuda").manual_seed(Lk)
    rand = lambda h, n: torch.randn(B, h, n, 64, device="cuda", generator=g).to(dtype)
    q, k, v, w = rand(H, 1), rand(Hk, Lk), rand(Hk, Lk), rand(H, 1)
    mask = torch.rand(B, 1, 1, Lk, device="cuda", generator=g) < 0.6
    gone = ~mask.transpose(2, 3)
    sets = []
    for a, b in ((k, v), (spoiled(k, gone, float("inf")), spoiled(v, gone, float("nan")))):
        leaves = [x.clone().requires_grad_(True) for x in (q, a, b)]
        out = ops.attention(*leaves, mask=mask)
        assert torch.equal(out, ops.attention(*(x.detach() for x in leaves), mask=mask))
        sets.append([out, *torch.autograd.grad(out, leaves, w)])
    for a, b in zip(*sets):
        assert torch.isfinite(b).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lq", [1, 5, 140])
def test_one_key_and_queries_that_a_padding_mask_takes(dtype, Lq):
    from ocean import ops
    g = torch.Generator(device="cuda").manual_seed(Lq)
    rand = lambda h, n: torch.randn(4, h, n, 64, device="cuda", generator=g).to(dtype)
    q, k, v, w = rand(4, Lq), rand(2, 1), rand(2, 1), rand(4, Lq)
    mask = torch.rand(4, 1, Lq, 1, device="cuda", generator=g) < 0.5
    mask[0], mask[1] = False, True
    sets = []
    for a, b in ((q, w), (spoiled(q, ~mask, float("nan")), spoiled(w, ~mask, float("-inf")))):
        leaves = [x.clone().requires_grad_(True) for x in (a, k, v)]
        out = ops.attention(*leaves, mask=mask)
        assert torch.equal(out, ops.attention(*(x.detach() for x in leaves), mask=mask))
        sets.append([out, *torch.autograd.grad(out, leaves, b)])
    for a, b in zip(*sets):
        assert torch.isfinite(b).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_query_of_a_module_over_a_padded_cache(dtype):
    from ocean.models.components import ScaledDotProductAttention
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k, v = (torch.randn(2, n, 48, device="cuda", generator=g).to(dtype) for n in (1, 90, 90))
    mask = torch.ones(2, 1, 90, device="cuda")
    mask[0, :, 50:], mask[1, :, 7:] = 0, 0
    m = ScaledDotProductAttention(48).cuda().eval()
    want, _ = m(q, k, v, mask, need_weights=False)
    gone = mask.transpose(1, 2) == 0
    got, _ = m(q, spoiled(k, gone, float("nan")), spoiled(v, gone, float("inf")), mask, need_weights=False)
    assert torch.isfinite(want).all() and torch.equal(got, want)

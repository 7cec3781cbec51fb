"""ops.layer_norm / ops.add_layer_norm against their definition in 64 bits.  Bounds: half a step of the output's type for
each rounding (torch.finfo.eps / 2), fp32 sums of W (rows) terms add at most W (rows) half steps of the terms' sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0 ** -24


def exact(s, w, b, eps, dy=None, dsum=None):
    s = s.detach().double()
    W = s.shape[-1]
    mean = s.mean(-1, keepdim=True)
    xc = s - mean
    rstd = 1.0 / ((xc * xc).mean(-1, keepdim=True) + eps).sqrt()
    xh = xc * rstd
    w = torch.ones(W, device=s.device, dtype=torch.float64) if w is None else w.detach().double()
    b = torch.zeros(W, device=s.device, dtype=torch.float64) if b is None else b.detach().double()
    # error of xh: the mean's (W + 2 half steps of the mean size), the deviation's (W / 2 + 4, relative)
    size = s.abs().mean(-1, keepdim=True)
    e_xh = ((W + 4) * U32 * (size + s.abs()) * rstd) + (W + 8) * U32 * xh.abs()
    out = {"y": (xh * w + b, e_xh * w.abs() + 4 * U32 * ((xh * w).abs() + b.abs()))}
    if dy is not None:
        dy = dy.double()
        g = dy * w
        mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        dx = rstd * (g - mg - xh * mgx)
        ag, agx = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
        e = rstd * ((W + 8) * U32 * (g.abs() + ag + xh.abs() * agx) * 2 + e_xh * agx + xh.abs() * (g.abs() * e_xh).mean(-1, keepdim=True))
        e = e + (W + 8) * U32 * dx.abs()
        if dsum is not None:
            dx = dx + dsum.double()
            e = e + 2 * U32 * dsum.double().abs()
        R = s.numel() // W
        flat = lambda t: t.reshape(-1, W)
        out["dx"] = (dx, e)
        out["dw"] = (flat(dy * xh).sum(0), (R + 4) * U32 * flat((dy * xh).abs()).sum(0) + flat(dy.abs() * e_xh).sum(0))
        out["db"] = (flat(dy).sum(0), (R + 4) * U32 * flat(dy.abs()).sum(0))
    return out


def close(name, got, want):
    ref, e = want
    limit = e + torch.finfo(got.dtype).eps / 2 * (ref.abs() + e) + 2.0 ** -25 * (got.dtype == torch.float16) + 1e-30
    err = (got.detach().double() - ref).abs()
    assert got.shape == ref.shape
    assert (err <= limit).all(), f"{name}: {(err / limit).amax().item():.3g} times the bound, max err {err.amax().item():.3e}"


def rows(R, W, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(R, W, device="cuda", generator=g) * scale + shift).to(dtype)


WIDTHS = [1, 2, 3, 7, 8, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 768, 1000, 1023, 1025, 2047, 2049, 4095, 4097, 8191, 8193, 16384, 16385, 32769]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("W", WIDTHS)
def test_widths(W, dtype):
    from ocean import ops
    R = 1 if W % 5 == 0 else 37
    x, dy = rows(R, W, dtype, W, 1.5, 0.4), rows(R, W, dtype, W + 1)
    w, b = 1 + 0.3 * rows(1, W, torch.float32, 5)[0], rows(1, W, torch.float32, 6)[0]
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = ops.layer_norm(*leaves, 1e-5)
    want = exact(x, w, b, 1e-5, dy)
    close("y", y, want["y"])
    for n, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)):
        close(n, g, want[n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,W", [(1, 128), (5, 96), (300, 65), (4097, 24), (700, 2500), (3, 17000)])
def test_residual_sum_and_its_gradient(R, W, dtype):
    from ocean import ops
    x, r, dy, ds = (rows(R, W, dtype, s) for s in (1, 2, 3, 4))
    w, b = 1 + 0.3 * rows(1, W, torch.float32, 5)[0], rows(1, W, torch.float32, 6)[0]
    leaves = [t.requires_grad_(True) for t in (x, r, w, b)]
    y, s = ops.add_layer_norm(*leaves, 1e-5)
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    want = exact(s, w, b, 1e-5, dy, ds)
    close("y", y, want["y"])
    got = torch.autograd.grad([y, s], leaves, [dy, ds], retain_graph=True)
    assert torch.equal(got[0], got[1])
    for n, g in zip(("dx", "dw", "db"), (got[0], got[2], got[3])):
        close(n, g, want[n])
    only = exact(s, w, b, 1e-5, dy)
    close("dx without the sum's gradient", torch.autograd.grad(y, x, dy, retain_graph=True)[0], only["dx"])
    zero = torch.autograd.grad(s, leaves, ds)
    assert torch.equal(zero[0], ds) and torch.equal(zero[1], ds) and not zero[2].any() and not zero[3].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_types_and_absence(dtype):
    from ocean import ops
    x, dy = rows(50, 200, dtype, 1), rows(50, 200, dtype, 2)
    for w, b in ((None, None), (rows(1, 200, dtype, 3)[0], None), (None, rows(1, 200, torch.float32, 4)[0]), (rows(1, 200, dtype, 3)[0], rows(1, 200, dtype, 4)[0])):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
        y = ops.layer_norm(leaves[0], *(None if t is None else leaves[1 + (n if w is not None else 0)] for n, t in enumerate((w, b))), 1e-6)
        want = exact(x, w, b, 1e-6, dy)
        close("y", y, want["y"])
        got = torch.autograd.grad(y, leaves, dy)
        names = ["dx"] + (["dw"] if w is not None else []) + (["db"] if b is not None else [])
        for n, g in zip(names, got):
            ref, e = want[n]
            close(n, g, (ref, e + U32 * ref.abs()))


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_and_strides(dtype):
    from ocean import ops
    w, b = rows(1, 120, torch.float32, 3)[0], rows(1, 120, torch.float32, 4)[0]
    base = rows(60, 131, dtype, 1)
    for x in (base[:, 5:125], base[::2, 1:121], base[:, 5:125].reshape(3, 20, 120), base[:, 5:125].reshape(3, 20, 120).transpose(0, 1), base[:120, :60].t(),
              base[0, :120], base[:1, 3:123].expand(7, 120)):
        x = x if x.shape[-1] == 120 else rows(120, 40, dtype, 9).t()
        leaf = x.detach().requires_grad_(True)
        y = ops.layer_norm(leaf, w, b)
        want = exact(x, w, b, 1e-5, torch.ones_like(x))
        close("y", y, want["y"])
        close("dx", torch.autograd.grad(y.sum(), leaf)[0], want["dx"])
        assert y.shape == x.shape


def test_rows_without_spread_large_offsets_and_no_rows():
    from ocean import ops
    x = torch.full((5, 300), 7.25, device="cuda")
    assert not ops.layer_norm(x).any()                            # the mean is exact, xh = 0
    x = rows(20, 1000, torch.float32, 1) + 4096.0                 # centred sums: the deviation keeps its digits
    close("y", ops.layer_norm(x), exact(x, None, None, 1e-5)["y"])
    w = torch.ones(40, device="cuda", requires_grad=True)
    e = torch.empty(0, 40, device="cuda", requires_grad=True)
    y = ops.layer_norm(e, w)
    dx, dw = torch.autograd.grad(y, (e, w), torch.empty_like(y))
    assert y.shape == (0, 40) and dx.shape == (0, 40) and not dw.any()
    y, s = ops.add_layer_norm(e, e, w)
    assert y.shape == s.shape == (0, 40)
    x = rows(4, 64, torch.float32, 2)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y = ops.layer_norm(x)
    assert torch.isfinite(y[[0, 3]]).all() and torch.isnan(y[1]).all() and torch.isnan(y[2]).any()


def test_same_results_in_every_run_streams_and_replays():
    from ocean import _hip, ops
    x, dy = rows(5000, 768, torch.bfloat16, 1), rows(5000, 768, torch.bfloat16, 2)
    w, b = rows(1, 768, torch.float32, 3)[0], rows(1, 768, torch.float32, 4)[0]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y, s = ops.add_layer_norm(leaves[0], x, leaves[1], leaves[2])
        return [y.detach(), s.detach(), *torch.autograd.grad(y, leaves, dy)]

    first = step()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, other))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with _hip.capture(gr):
            outs = step()
        graphs.append((gr, outs))
    for it in range(3):
        x.copy_(x * 1.5)
        for gr, outs in graphs:
            gr.replay()
        want = step()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, c) for a, c in zip(outs, want))


def test_gradients_against_differences():
    """Central differences in fp32 inputs with fp64 sums of the outputs: at e = 1e-2 the third derivative's share and the
    rounding of the two values both stay below 1e-3 of the gradient's norm."""
    from ocean import ops
    x, w, b, c = rows(6, 50, torch.float32, 1), 1 + 0.2 * rows(1, 50, torch.float32, 2)[0], rows(1, 50, torch.float32, 3)[0], rows(6, 50, torch.float32, 4)
    f = lambda *t: (ops.layer_norm(*t).double() * c.double()).sum()
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(f(*leaves), leaves)
    for n in range(3):
        u = torch.randn(leaves[n].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
        u /= u.norm()
        lo, hi = ([t.detach() + (s * 1e-2 * u if m == n else 0) for m, t in enumerate(leaves)] for s in (-1, 1))
        num = ((f(*hi) - f(*lo)) / 2e-2).item()
        assert abs(num - (grads[n].double() * u.double()).sum().item()) <= 1e-3 * max(1.0, float(grads[n].norm()))

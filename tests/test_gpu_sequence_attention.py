"""ops.attention (no stored weights; backward by recomputation; position bias by buckets) against its definition in 64 bits.
Bounds: sequence_reference.tolerance."""
import math

import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def heads_view(B, H, L, d, dtype, seed, layout="rows", scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "rows":                       # [B, L, H * d] as a projection gives it
        return (torch.randn(B, L, H, d, device="cuda", generator=g) * scale).to(dtype).transpose(1, 2)
    if layout == "heads":
        return (torch.randn(B, H, L, d, device="cuda", generator=g) * scale).to(dtype)
    wide = (torch.randn(B, H, L, d + 3, device="cuda", generator=g) * scale).to(dtype)      # "odd": rows at no alignment
    return wide[..., 1:d + 1]


def run_case(B, H, Hk, Lq, Lk, d, dtype, causal=False, lengths=None, starts=None, start=None, mask=None, buckets=0, max_distance=128,
             both=True, layout="rows", scale=None, train=True, seed=0, spread=1.0):
    from ocean import ops
    q, k, v = (heads_view(B, h, L, d, dtype, 10 * seed + n, layout, spread) for n, (h, L) in enumerate(((H, Lq), (Hk, Lk), (Hk, Lk))))
    dout = heads_view(B, H, Lq, d, dtype, 10 * seed + 3, layout)
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    sc = 1.0 / math.sqrt(d) if scale is None else scale
    ok, dist = ref.places(B, H, Lq, Lk, causal, lengths, mask, starts, start)
    bias = table = at = None
    if buckets:
        table = torch.randn(buckets, H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 77)) * 0.7
        bias, at = ref.bias_of(table, dist, buckets, max_distance, both)
    r = ref.attention(q, k, v, ok, sc, dout if train else None, bias)
    leaves = [t.detach().requires_grad_(train) for t in (q, k, v)]
    if table is not None:
        leaves.append(table.requires_grad_(train))
    out = ops.attention(*leaves[:3], mask=None if mask is None else mask.cuda(), key_lengths=lengths, causal=causal, scale=scale,
                        query_start=starts if starts is not None else start, position_table=table, max_distance=max_distance,
                        bidirectional=both)
    ref.check("out", out, r, dtype, d, Lk)
    assert (out.detach()[~ok.any(-1).cuda()] == 0).all()
    if not train:
        return out
    grads = torch.autograd.grad(out, leaves, dout)
    for name, g, n in zip(("dq", "dk", "dv"), grads, (Lk, Lq * (H // Hk), Lq * (H // Hk))):
        ref.check(name, g, r, dtype, d, n)
    if table is not None:
        want, size = ref.table_grad(r["ds"], at, buckets), ref.table_grad(r["mag"]["ds"], at, buckets)
        u = 2.0 ** -8 if dtype == BF16 else 0.0              # delta from the rounded output
        limit = (2 * (d + 4) * 2.0 ** -24 * max(1.0, r["smax"]) + (Lk + d + 16) * 2.0 ** -24 + u) * size + 1e-30
        err = (grads[3].double() - want).abs()
        assert (err <= limit).all(), f"dtable {(err / limit).amax().item():.3g}"
    return out


SIZES = [(1, 1, 1, 1, 1, 8), (2, 3, 3, 5, 1, 16), (1, 2, 1, 31, 33, 32), (2, 4, 2, 32, 32, 64), (1, 2, 2, 33, 31, 49), (2, 2, 1, 127, 129, 64),
         (1, 3, 1, 128, 128, 128), (1, 2, 2, 129, 65, 96), (2, 8, 2, 100, 100, 16), (1, 2, 1, 257, 300, 80), (1, 1, 1, 64, 513, 128),
         (1, 4, 1, 300, 64, 33), (3, 2, 2, 70, 70, 127)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H,Hk,Lq,Lk,d", SIZES)
def test_sizes(B, H, Hk, Lq, Lk, d, dtype):
    run_case(B, H, Hk, Lq, Lk, d, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H,Hk,Lq,Lk,d", [(2, 2, 1, 127, 127, 64), (1, 2, 2, 130, 300, 32), (2, 2, 1, 300, 130, 128), (1, 4, 2, 257, 257, 96), (2, 6, 3, 1, 40, 64),
                                            (1, 2, 2, 7, 129, 40)])
def test_causal(B, H, Hk, Lq, Lk, d, dtype):
    run_case(B, H, Hk, Lq, Lk, d, dtype, causal=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_of_zero_one_and_beyond(dtype, causal):
    run_case(6, 4, 2, 150, 150, 64, dtype, causal=causal, lengths=[0, 1, 33, 64, 150, 149])
    from ocean import ops
    q, k, v = (heads_view(3, 2, 40, 32, dtype, s) for s in (1, 2, 3))
    n = torch.tensor([-5, 1000, 40], dtype=torch.int32, device="cuda")          # clamped to 0..keys
    out = ops.attention(q, k, v, key_lengths=n)
    same = ops.attention(q, k, v, key_lengths=torch.tensor([0, 40, 40], dtype=torch.int32, device="cuda"))
    assert torch.equal(out, same) and (out[0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_positions_of_the_first_query(dtype):
    run_case(4, 2, 2, 50, 90, 64, dtype, causal=True, starts=[-70, -20, 0, 200])       # a whole sample, some rows, none empty
    run_case(2, 2, 1, 50, 90, 64, dtype, causal=True, start=13)
    run_case(2, 2, 1, 3, 90, 32, dtype, causal=True, start=-2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 1, 70, 150), (2, 4, 70, 150), (1, 1, 1, 150), (2, 1, 1, 150), (1, 4, 70, 1)])
def test_masks(dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    mask = torch.rand(shape, generator=g) < 0.7
    if shape[2] > 1:
        mask[:, :, 5::13] = False                                                   # rows that see nothing
    mask = mask.expand(2, 4, 70, 150)
    run_case(2, 4, 2, 70, 150, 64, dtype, mask=mask)
    run_case(2, 4, 2, 70, 150, 40, dtype, mask=mask, causal=True, lengths=[150, 77])
    run_case(2, 4, 4, 2, 150, 40, dtype, mask=mask[:, :, :2], causal=True, lengths=[150, 77])


def test_mask_types_and_odd_strides():
    from ocean import ops
    q, k, v = (heads_view(2, 2, 65, 32, F32, s) for s in (1, 2, 3))
    g = torch.Generator(device="cuda").manual_seed(5)
    m = (torch.rand(2, 2, 65, 130, device="cuda", generator=g) < 0.6)[..., ::2]
    a = ops.attention(q, k, v, mask=m)
    assert torch.equal(a, ops.attention(q, k, v, mask=m.contiguous()))
    assert torch.equal(a, ops.attention(q, k, v, mask=m.to(torch.uint8) * 7))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["heads", "odd"])
@pytest.mark.parametrize("d", [8, 17, 64, 128])
def test_layouts(dtype, layout, d):
    run_case(2, 4, 2, 70, 90, d, dtype, layout=layout)
    run_case(2, 4, 2, 3, 90, d, dtype, layout=layout, lengths=[90, 31])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [1, 3, 5, 7])
def test_few_features(dtype, d):
    run_case(2, 2, 1, 40, 50, d, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H,Hk,Lq,Lk,d", [(1, 8, 2, 1, 257, 64), (3, 8, 1, 1, 2000, 128), (2, 12, 12, 1, 1000, 64), (1, 32, 2, 1, 4097, 96), (2, 4, 2, 9, 777, 32),
                                            (1, 1, 1, 32, 3000, 128), (40, 16, 8, 1, 300, 128)])
def test_few_queries_over_long_keys(dtype, B, H, Hk, Lq, Lk, d):
    lengths = [max(1, Lk - 97 * b) for b in range(B)]
    run_case(B, H, Hk, Lq, Lk, d, dtype, train=False)
    run_case(B, H, Hk, Lq, Lk, d, dtype, lengths=lengths, starts=[n - Lq for n in lengths], causal=True, buckets=16, both=False, max_distance=50)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("buckets,max_distance,both", [(32, 128, True), (4, 20, True), (2, 2, False), (17, 33, False), (128, 256, True), (64, 1024, False)])
def test_position_bias(dtype, buckets, max_distance, both):
    run_case(2, 3, 3, 150, 150, 64, dtype, buckets=buckets, max_distance=max_distance, both=both, causal=not both)
    run_case(2, 4, 2, 70, 333, 40, dtype, buckets=buckets, max_distance=max_distance, both=both, lengths=[333, 100], starts=[263, 30])


def test_position_bias_far_from_the_diagonal_and_on_every_bucket():
    run_case(1, 1, 1, 700, 700, 32, F32, buckets=32, max_distance=64)
    from ocean import ops
    # one query, one-hot values: the weights themselves tell every key's bucket
    for both, nb, md in ((True, 32, 128), (False, 32, 128), (True, 24, 100), (False, 7, 300), (True, 128, 1024), (False, 128, 1023)):
        Lk, at = 2 * md + 40, md + 20
        table = torch.linspace(-2.0, 2.0, nb, device="cuda").view(nb, 1).contiguous()
        p = torch.softmax(table.view(-1).double().cpu()[torch.tensor([ref.bucket(j - at, nb, md, both) for j in range(Lk)])], 0)
        q, k = torch.zeros(1, 1, 1, 32, device="cuda"), torch.zeros(1, 1, Lk, 32, device="cuda")
        for c in range(0, Lk, 32):
            m = min(32, Lk - c)
            v = torch.zeros(1, 1, Lk, 32, device="cuda")
            v[0, 0, torch.arange(c, c + m), torch.arange(m)] = 1.0
            w = ops.attention(q, k, v, position_table=table, max_distance=md, bidirectional=both, query_start=at)[0, 0, 0, :m].double().cpu()
            # the buckets' weights are at least exp(4 / 127) = 3 % apart; a weight is a quotient of sums of Lk terms
            assert ((w - p[c:c + m]).abs() <= (2 * Lk + 32) * 2.0 ** -24 * p[c:c + m]).all(), (both, nb, md, c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales_and_large_scores(dtype):
    run_case(1, 2, 2, 70, 90, 64, dtype, scale=1.7)
    run_case(1, 2, 2, 70, 90, 64, dtype, scale=1e-3)
    from ocean import ops
    # one key far above the rest: the running maximum jumps late, everything before it vanishes
    k = torch.zeros(1, 1, 200, 32, device="cuda", dtype=dtype)
    k[:, :, 150] = 10.0
    q = torch.ones(1, 1, 40, 32, device="cuda", dtype=dtype)
    v = torch.randn(1, 1, 200, 32, device="cuda").to(dtype)
    # the remaining weight is e = 2^t with t the rounding of the scaled maximum, so the row is (e v) / e: the product, the
    # reciprocal and the last product round once each, at most 3 half steps of fp32 (4 with their products)
    for out in (ops.attention(q, k, v, scale=1.0), ops.attention(q[:, :, :1], k, v, scale=1.0)):
        want = v[:, :, 150:151].double()
        assert ((out.double() - want).abs() <= (4 * 2.0 ** -24 + (0 if dtype == F32 else 2.0 ** -8)) * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq", [1, 140])
def test_what_lies_behind_a_sample_is_not_read(dtype, Lq):
    from ocean import ops
    n = torch.tensor([140, 37, 64, 0], dtype=torch.int32, device="cuda")
    q, k, v = (heads_view(4, 4 if s == 1 else 2, Lq if s == 1 else 140, 64, dtype, s).detach() for s in (1, 2, 3))
    dirty = [k.clone(), v.clone()]
    for t, fill in zip(dirty, (float("nan"), float("inf"))):
        for b in range(4):
            t[b, :, int(n[b]):] = fill
    args = [[t.requires_grad_(True) for t in (q.clone(), a, b)] for a, b in ((k.clone(), v.clone()), dirty)]
    outs = [ops.attention(*a, key_lengths=n) for a in args]
    assert torch.equal(outs[0], outs[1])
    for x, y in zip(*(torch.autograd.grad(o, a, torch.ones_like(o)) for o, a in zip(outs, args))):
        assert torch.equal(x, y) and torch.isfinite(x).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq", [2, 140])
def test_what_a_padding_mask_takes_is_not_read(dtype, Lq):
    """NaN and infinities in keys and values that a mask [batch, 1, 1, keys] takes, in queries and in the arriving gradient where one
    of [batch, 1, queries, 1] does."""
    from ocean import ops
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v, w = (heads_view(3, 4 if s in (1, 4) else 2, Lq if s in (1, 4) else 130, 64, dtype, s).detach() for s in (1, 2, 3, 4))
    by_key = torch.rand(3, 1, 1, 130, device="cuda", generator=g) < 0.7
    by_query = torch.rand(3, 1, Lq, 1, device="cuda", generator=g) < 0.5
    for mask, dirty in ((by_key, (1, 2)), (by_query, (0, 3))):
        sets = []
        for spoil in (False, True):
            t = [x.clone() for x in (q, k, v, w)]
            if spoil:
                gone = ~(mask.transpose(2, 3) if dirty[0] else mask)
                for n, fill in zip(dirty, (float("nan"), float("-inf"))):
                    t[n] = t[n].masked_fill(gone, fill)
            leaves = [x.requires_grad_(True) for x in t[:3]]
            out = ops.attention(*leaves, mask=mask)
            sets.append([out, *torch.autograd.grad(out, leaves, t[3])])
            assert torch.equal(out, ops.attention(*(x.detach() for x in leaves), mask=mask))
        for a, b in zip(*sets):
            assert torch.isfinite(b).all() and torch.equal(a, b)


def test_second_derivatives_are_refused():
    from ocean import ops
    q = torch.randn(1, 1, 4, 16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="differentiated"):
        torch.autograd.grad(ops.attention(q, q, q).sum(), q, create_graph=True)
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="differentiated"):
        torch.autograd.grad(ops.layer_norm(x).sum(), x, create_graph=True)


def test_nothing_to_attend_to():
    from ocean import ops
    for Lq, Lk, B in ((3, 0, 2), (0, 5, 2), (3, 5, 0)):
        leaves = [torch.randn(B, 2, L, 16, device="cuda", requires_grad=True) for L in (Lq, Lk, Lk)]
        out = ops.attention(*leaves)
        assert out.shape == (B, 2, Lq, 16) and (out == 0).all()
        for g, t in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), leaves):
            assert g.shape == t.shape and (g == 0).all()


def test_gradients_of_broadcast_inputs_and_partial_requests():
    from ocean import ops
    q = heads_view(3, 4, 50, 32, F32, 1).detach().requires_grad_(True)
    k1, v1 = (heads_view(1, 2, 60, 32, F32, s).detach().requires_grad_(True) for s in (2, 3))
    w = torch.randn(3, 4, 50, 32, device="cuda")
    out = ops.attention(q, k1.expand(3, 2, 60, 32), v1.expand(3, 2, 60, 32))
    got = torch.autograd.grad(out, (q, k1, v1), w)
    full = [t.detach().expand(3, 2, 60, 32).contiguous().requires_grad_(True) for t in (k1, v1)]
    out2 = ops.attention(q, *full)
    want = torch.autograd.grad(out2, (q, *full), w)
    assert torch.equal(out, out2) and torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
        assert torch.allclose(a, b.sum(0, keepdim=True), rtol=1e-6, atol=1e-6 * float(b.abs().max()))
    for pick in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(n in pick) for n, t in enumerate((q, *full))]
        g = torch.autograd.grad(ops.attention(*leaves), [leaves[n] for n in pick], w)
        for n, x in zip(pick, g):
            assert torch.equal(x, want[n])
    # the gradient that arrives may be a broadcast
    assert torch.equal(torch.autograd.grad(ops.attention(q, *full).sum(), q)[0],
                       torch.autograd.grad(ops.attention(q, *full), q, torch.ones_like(out))[0])


def test_gradients_against_differences():
    """f(x + e u) - f(x - e u) over 2 e along a random direction.  The third derivative's share is e^2 |f'''| / 6 and the
    difference's rounding 2^-24 |f| sqrt(n) / e: at e = 1e-2 both stay below 1e-3 of the derivatives' scale here."""
    from ocean import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = [rand(1, 2, 20, 16), rand(1, 1, 40, 16), rand(1, 1, 40, 16), rand(8, 2)]
    w = rand(1, 2, 20, 16)
    f = lambda a: (ops.attention(a[0], a[1], a[2], position_table=a[3], max_distance=10).double() * w.double()).sum()
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(f(leaves), leaves)
    for n in range(4):
        u = rand(*x[n].shape)
        u /= u.norm()
        e = 1e-2
        moved = [[t + (sgn * e * u if m == n else 0) for m, t in enumerate(x)] for sgn in (1, -1)]
        num = ((f(moved[0]) - f(moved[1])) / (2 * e)).item()
        ana = (grads[n].double() * u.double()).sum().item()
        assert abs(num - ana) <= 1e-3 * max(1.0, float(grads[n].norm())), (n, num, ana)


def test_same_results_in_every_run():
    from ocean import ops
    leaves = [heads_view(2, h, 300, 64, BF16, s).detach().requires_grad_(True) for s, h in ((1, 8), (2, 2), (3, 2))]
    leaves.append(torch.randn(32, 8, device="cuda", requires_grad=True))
    w = heads_view(2, 8, 300, 64, BF16, 9)
    step = lambda: (lambda o: [o, *torch.autograd.grad(o, leaves, w)])(ops.attention(*leaves[:3], position_table=leaves[3], max_distance=64))
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    tok = lambda: ops.attention(leaves[0][:, :, :1], leaves[1], leaves[2])
    t = tok().detach()
    assert torch.equal(t, tok())


def test_another_stream_and_two_at_once():
    from ocean import ops
    q, k, v = (heads_view(2, 4, 200, 64, F32, s) for s in (1, 2, 3))
    want, want1 = ops.attention(q, k, v), ops.attention(q[:, :, :1], k, v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                outs.append((ops.attention(q, k, v), ops.attention(q[:, :, :1], k, v)))
    torch.cuda.synchronize()
    for a, b in outs:
        assert torch.equal(a, want) and torch.equal(b, want1)


def test_captured_and_replayed():
    """Two graphs of the same operators, replayed in turn with eager work between; inputs change under them."""
    from ocean import _hip, ops
    g = torch.Generator(device="cuda").manual_seed(1)
    src = [torch.randn(2, 4, 130, 64, device="cuda", generator=g).to(BF16) for _ in range(4)]
    n = torch.tensor([130, 50], dtype=torch.int32, device="cuda")

    def step(bufs):
        leaves = [t.detach().requires_grad_(True) for t in bufs[:3]]
        o = ops.attention(*leaves, key_lengths=n, causal=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, bufs[3]), ops.attention(leaves[0].detach()[:, :, :1], *[t.detach() for t in leaves[1:]], key_lengths=n)]

    graphs = []
    side = torch.cuda.Stream()
    for k in range(2):
        bufs = [t.clone() for t in src]
        with torch.cuda.stream(side):
            step(bufs)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with _hip.capture(gr):
            outs = step(bufs)
        graphs.append((gr, bufs, outs))
    for it in range(4):
        for k, (gr, bufs, outs) in enumerate(graphs):
            for b, s in zip(bufs, src):
                b.copy_(s * (1 + 0.25 * (it + k)))
            n.copy_(torch.tensor([130 - 7 * it, 50 + it], dtype=torch.int32))
            gr.replay()
            want = step([b.clone() for b in bufs])
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """A cache whose last rows lie more than 2^32 elements behind its first."""
    from ocean import ops
    Lk, gap = 70, (1 << 32) // 64 + 1000
    base = torch.zeros((Lk - 1) * gap + 64, device="cuda", dtype=BF16)
    k = base.as_strided((1, 1, Lk, 64), (0, 0, gap, 1))
    small = torch.randn(1, 1, Lk, 64, device="cuda").to(BF16)
    k.copy_(small)
    q = torch.randn(1, 1, 40, 64, device="cuda").to(BF16)
    assert torch.equal(ops.attention(q, k, k), ops.attention(q, small, small))
    assert torch.equal(ops.attention(q[:, :, :1], k, k), ops.attention(q[:, :, :1], small, small))

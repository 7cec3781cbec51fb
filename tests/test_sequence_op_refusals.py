"""What the sequence operators refuse, in Python and at the C ABI: nothing here launches a kernel."""
import ctypes

import pytest
import torch

from ocean import _hip, ops


def qkv(B=2, H=4, Hk=2, Lq=3, Lk=5, d=16, dtype=torch.float32):
    return torch.zeros(B, H, Lq, d, dtype=dtype), torch.zeros(B, Hk, Lk, d, dtype=dtype), torch.zeros(B, Hk, Lk, d, dtype=dtype)


@pytest.mark.parametrize("change", [
    dict(H=3), dict(d=0), dict(d=129), dict(dtype=torch.float64), dict(dtype=torch.float16)])
def test_attention_shapes_and_types(change):
    with pytest.raises(ValueError):
        ops.attention(*qkv(**change))


def test_attention_arguments():
    q, k, v = qkv()
    with pytest.raises(ValueError):
        ops.attention(q[0], k, v)
    with pytest.raises(ValueError):
        ops.attention(q, k, v[:, :, :-1])
    with pytest.raises(ValueError):
        ops.attention(q, k[:1], v[:1])
    with pytest.raises(ValueError):
        ops.attention(q, k.bfloat16(), v.bfloat16())
    with pytest.raises(_hip.OceanHipError):
        ops.attention(q, k, v)                                # no CPU path
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(()))
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(_hip.OceanHipError):
        ops.layer_norm(torch.zeros(3, 4))


@pytest.mark.gpu
def test_arguments_with_the_tensors_on_the_gpu():
    q, k, v = (t.cuda() for t in qkv())
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = torch.zeros(32, 4, device="cuda")
    bad = [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(mask=torch.ones(2, 1, 3, 5, device="cuda")),
           dict(key_lengths=torch.tensor([1, 2], device="cuda")), dict(key_lengths=i32(1, 2, 3)), dict(query_start=i32(1)),
           dict(query_start=1 << 31), dict(position_table=table[:, :3]), dict(position_table=table[:31]), dict(position_table=table[:2]),
           dict(position_table=table[:1], bidirectional=False), dict(position_table=table, max_distance=8),
           dict(position_table=table, max_distance=1025), dict(position_table=torch.zeros(130, 4, device="cuda"))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.attention(q, k, v, **kw)
    for kw in (dict(mask=torch.ones(2, 1, 3, 5, dtype=torch.bool)), dict(key_lengths=torch.tensor([1, 2], dtype=torch.int32)),
               dict(position_table=table.cpu())):
        with pytest.raises(_hip.OceanHipError):
            ops.attention(q, k, v, **kw)
    with pytest.raises(RuntimeError):
        ops.attention(q, k, v, mask=torch.ones(2, 1, 4, 5, dtype=torch.bool, device="cuda"))
    x = torch.zeros(3, 8, device="cuda")
    for args in ((x, x[:, :7].contiguous()[0]), (x, None, x[0, :3])):
        with pytest.raises(ValueError):
            ops.layer_norm(*args)
    with pytest.raises(ValueError):
        ops.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        ops.add_layer_norm(x, x[:2])
    with pytest.raises(ValueError):
        ops.add_layer_norm(x, x.bfloat16())


def attention_shape(**change):
    s = _hip.AttentionShape()
    for k, v in dict(dict(B=2, H=4, Hk=2, Lq=3, Lk=5, d=16, scale=1.0), **change).items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("change,status", [
    (dict(B=0), 1), (dict(H=3), 1), (dict(Lq=0), 1), (dict(Lk=-1), 1), (dict(dtype=2), 1), (dict(scale=0.0), 1), (dict(scale=float("nan")), 1),
    (dict(d=129), 2), (dict(d=3), 2), (dict(d=7, dtype=1), 2), (dict(query_start=(1 << 30) + 1), 2), (dict(num_buckets=7, bidirectional=1, max_distance=9), 1),
    (dict(num_buckets=8, max_distance=4), 1), (dict(num_buckets=130, max_distance=200), 2), (dict(num_buckets=8, max_distance=1025), 2), (dict(), 4)])
def test_attention_status_codes(change, status):
    L, s = _hip.lib(), attention_shape(**change)
    none = [None] * 8
    assert L.ocean_attention_fwd(ctypes.byref(s), *none[:7], None, 0, None, None, None) == status
    assert L.ocean_attention_bwd(ctypes.byref(s), *none[:7], None, None, None, None, 0, None, None, None, None, None) == status
    p = ctypes.c_void_p(64)                                   # never followed: a missing table, output or workspace is found first
    if status == 4:
        assert L.ocean_attention_fwd(ctypes.byref(s), p, p, p, None, None, None, None, None, 0, None, None, None) == 4
        assert L.ocean_attention_fwd(ctypes.byref(s), p, p, p, None, None, None, p, None, 0, p, None, None) == 4
        assert L.ocean_attention_bwd(ctypes.byref(s), p, p, p, None, None, None, None, p, p, p, p, 1, p, p, p, None, None) == 3
        long = attention_shape(Lq=1, Lk=100000)
        n = L.ocean_attention_fwd_workspace(ctypes.byref(long))
        assert n > 0
        assert L.ocean_attention_fwd(ctypes.byref(long), p, p, p, None, None, None, None, None, n, p, None, None) == 4
        assert L.ocean_attention_fwd(ctypes.byref(long), p, p, p, None, None, None, None, p, n - 1, p, None, None) == 3
    else:
        assert L.ocean_attention_bwd_workspace(ctypes.byref(s)) == 0


def test_layer_norm_status_codes():
    L = _hip.lib()
    p = ctypes.c_void_p(64)

    def shape(rows=4, width=8, dtype=0, **kw):
        s = _hip.LayerNormShape()
        s.rows, s.width, s.dtype, s.eps, s.x_stride, s.dy_stride = rows, width, dtype, 1e-5, width, width
        for k, v in kw.items():
            setattr(s, k, v)
        return s

    for s, status in ((shape(rows=0), 1), (shape(width=0), 1), (shape(dtype=3), 1), (shape(x_stride=7), 1), (shape(rows=1 << 31), 2), (shape(width=(1 << 24) + 1), 2)):
        assert L.ocean_layer_norm_fwd(ctypes.byref(s), p, None, None, None, p, None, None, None) == status
        assert L.ocean_layer_norm_bwd(ctypes.byref(s), p, p, None, p, None, p, 1 << 20, p, p, p, None) == status
    s = shape()
    assert L.ocean_layer_norm_fwd(ctypes.byref(s), None, None, None, None, p, None, None, None) == 4
    assert L.ocean_layer_norm_fwd(ctypes.byref(s), p, p, None, None, p, None, None, None) == 4
    assert L.ocean_layer_norm_fwd(ctypes.byref(s), p, p, None, None, p, p, None, None) == 1
    assert L.ocean_layer_norm_bwd(ctypes.byref(s), p, p, None, p, None, None, 0, p, p, None, None) == 4
    assert L.ocean_layer_norm_bwd(ctypes.byref(s), p, p, None, p, None, p, L.ocean_layer_norm_bwd_workspace(ctypes.byref(s)) - 1, p, p, None, None) == 3
    assert L.ocean_layer_norm_bwd(ctypes.byref(shape(dy_stride=7)), p, p, None, p, None, None, 0, p, None, None, None) == 1

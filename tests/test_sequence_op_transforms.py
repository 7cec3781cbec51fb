"""The sequence operators under tracing and forward-mode differentiation.  The first half runs without a GPU, over a stand-in for
the library whose operators copy their first input to the output."""
import ctypes
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ocean import _hip, ops


class Copying:
    """Layer norm and attention that copy: 8 values a call (x, or q, to y, or out)."""

    def ocean_layer_norm_fwd(self, sh, x, residual, w, b, y, total, stats, stream):
        ctypes.memmove(y, x, 32)
        if total:
            ctypes.memmove(total, x, 32)
        return 0

    def ocean_attention_fwd_workspace(self, sh):
        return 0

    def ocean_attention_fwd(self, sh, q, k, v, mask, lengths, starts, table, ws, n, out, lse, stream):
        ctypes.memmove(out, q, 32)
        return 0


@pytest.fixture
def copying(monkeypatch):
    monkeypatch.setattr(_hip, "lib", lambda: Copying())
    monkeypatch.setattr(ops, "_gpu", lambda t, name, index=None: 0)
    monkeypatch.setattr(ops, "_stream_of", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


CALLS = {"layer_norm": (lambda x: ops.layer_norm(x), (2, 4)),
         "add_layer_norm": (lambda x: ops.add_layer_norm(x, x)[0], (2, 4)),
         "attention": (lambda x: ops.attention(x, x, x), (1, 1, 2, 4)),
         "attention over one tensor": (lambda x: ops.attention(x, torch.ones(1, 1, 3, 4, device=x.device), torch.ones(1, 1, 3, 4, device=x.device)), (1, 1, 2, 4))}


def traced(f, example):
    with warnings.catch_warnings():                          # of sizes that a trace fixes
        warnings.simplefilter("ignore")
        return torch.jit.trace(f, (example,), check_trace=False)


@pytest.mark.parametrize("name", list(CALLS))
def test_a_trace_holds_the_operator(copying, name):
    f, shape = CALLS[name]
    t = traced(f, torch.zeros(shape))
    x = torch.arange(8.0).reshape(shape) + 1
    assert torch.equal(t(x), x)


@pytest.mark.parametrize("name", list(CALLS))
def test_a_forward_mode_tangent_is_refused_not_lost(copying, name):
    f, shape = CALLS[name]
    with fwAD.dual_level():
        with pytest.raises(RuntimeError):
            f(fwAD.make_dual(torch.ones(shape), torch.ones(shape)))
    with fwAD.dual_level():                                  # no tangent, nothing to lose
        assert torch.equal(f(torch.ones(shape)), torch.ones(shape))
    assert torch.equal(f(torch.ones(shape)), torch.ones(shape))


@pytest.mark.gpu
def test_traces_and_tangents_on_the_gpu():
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(2, h, n, 32, device="cuda", generator=g) for h, n in ((4, 40), (2, 60), (2, 60)))
    n = torch.tensor([60, 13], dtype=torch.int32, device="cuda")
    x, w = torch.randn(6, 50, device="cuda", generator=g), torch.rand(50, device="cuda", generator=g)
    for f, args in ((lambda a, b, c: ops.attention(a, b, c, key_lengths=n, causal=True), (q, k, v)),
                    (lambda a, b: ops.layer_norm(a, b), (x, w)), (lambda a, b: ops.add_layer_norm(a, a, b), (x, w))):
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            t = torch.jit.trace(f, args, check_trace=False)
        args = tuple(a * 1.5 for a in args)
        want, got = f(*args), t(*args)
        for a, b in zip(*(r if isinstance(r, tuple) else (r,) for r in (want, got))):
            assert torch.equal(a, b)
        with fwAD.dual_level():
            with pytest.raises(RuntimeError):
                f(fwAD.make_dual(args[0], torch.ones_like(args[0])), *args[1:])

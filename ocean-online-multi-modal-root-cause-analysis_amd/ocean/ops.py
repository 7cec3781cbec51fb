"""Autograd wrappers over single C-ABI entry points (losses and small glue).

Each function validates shapes on the host, allocates outputs / workspaces
through torch's caching allocator and enqueues the HIP work on the current
stream.  None of them has a CPU path.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _hip


class _InfoNce(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, positive, negatives, tau, label_offset, mean_rows):
        L = _hip.lib()
        sh = _hip.InfoNceShape()
        sh.B, sh.P = anchor.shape
        sh.Bp = positive.shape[0]
        sh.K = 0 if negatives is None else negatives.shape[0]
        sh.label_offset, sh.mean_rows, sh.tau = label_offset, mean_rows, tau
        ws = torch.empty(L.ocean_infonce_workspace(ctypes.byref(sh)), device=anchor.device, dtype=torch.float32)
        loss = torch.zeros((), device=anchor.device, dtype=torch.float32)
        _hip.check(L.ocean_infonce_fwd(ctypes.byref(sh), _hip.dev_ptr(anchor, "anchor"), _hip.dev_ptr(positive, "positive"),
                                       _hip.dev_ptr(negatives, "negatives"), _hip.dev_ptr(ws), ws.numel(), _hip.dev_ptr(loss),
                                       _hip.stream()), "ocean_infonce_fwd")
        ctx.sh = sh
        ctx.save_for_backward(anchor, positive, ws)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        L = _hip.lib()
        anchor, positive, ws = ctx.saved_tensors
        sh = ctx.sh
        wb = torch.empty(L.ocean_infonce_bwd_workspace(ctypes.byref(sh)), device=anchor.device, dtype=torch.float32)
        da, dp = torch.empty_like(anchor), torch.empty_like(positive)
        _hip.check(L.ocean_infonce_bwd(ctypes.byref(sh), _hip.dev_ptr(anchor), _hip.dev_ptr(positive), _hip.dev_ptr(ws),
                                       _hip.dev_ptr(wb), wb.numel(), _hip.dev_ptr(dloss.contiguous().float(), "dloss"),
                                       _hip.dev_ptr(da), _hip.dev_ptr(dp), _hip.stream()), "ocean_infonce_bwd")
        return da, dp, None, None, None, None


class _InfoNceRows(torch.autograd.Function):
    """reduction='none': one loss per anchor row."""

    @staticmethod
    def forward(ctx, anchor, positive, negatives, tau, label_offset):
        L = _hip.lib()
        sh = _hip.InfoNceShape()
        sh.B, sh.P = anchor.shape
        sh.Bp = positive.shape[0]
        sh.K = 0 if negatives is None else negatives.shape[0]
        sh.label_offset, sh.mean_rows, sh.tau = label_offset, 0, tau
        ws = torch.empty(L.ocean_infonce_workspace(ctypes.byref(sh)), device=anchor.device, dtype=torch.float32)
        rows = torch.empty(sh.B, device=anchor.device, dtype=torch.float32)
        _hip.check(L.ocean_infonce_rows_fwd(ctypes.byref(sh), _hip.dev_ptr(anchor, "anchor"), _hip.dev_ptr(positive, "positive"),
                                            _hip.dev_ptr(negatives, "negatives"), _hip.dev_ptr(ws), ws.numel(), _hip.dev_ptr(rows),
                                            _hip.stream()), "ocean_infonce_rows_fwd")
        ctx.sh = sh
        ctx.save_for_backward(anchor, positive, ws)
        return rows

    @staticmethod
    def backward(ctx, drows):
        L = _hip.lib()
        anchor, positive, ws = ctx.saved_tensors
        sh = ctx.sh
        wb = torch.empty(L.ocean_infonce_bwd_workspace(ctypes.byref(sh)), device=anchor.device, dtype=torch.float32)
        da, dp = torch.empty_like(anchor), torch.empty_like(positive)
        ws = ws.clone()                          # the backward pass rewrites the saved similarities
        _hip.check(L.ocean_infonce_rows_bwd(ctypes.byref(sh), _hip.dev_ptr(anchor), _hip.dev_ptr(positive), _hip.dev_ptr(ws),
                                            _hip.dev_ptr(wb), wb.numel(), _hip.dev_ptr(drows.contiguous().float(), "d_row_loss"),
                                            _hip.dev_ptr(da), _hip.dev_ptr(dp), _hip.stream()), "ocean_infonce_rows_bwd")
        return da, dp, None, None, None


def infonce(anchor: torch.Tensor, positive: torch.Tensor, negatives: Optional[torch.Tensor] = None,
            temperature: float = 0.1, label_offset: int = 0, mean_rows: int = 0, per_row: bool = False) -> torch.Tensor:
    """InfoNCELoss.forward (graph_fusion.py:112-162): the mean over rows, or with `per_row` (reduction='none') one
    value per anchor row.  negatives given: memory-bank branch; None: in-batch branch where row b of
    `anchor` is matched with row label_offset + b of `positive`."""
    if anchor.dim() != 2 or positive.dim() != 2 or anchor.shape[1] != positive.shape[1]:
        raise ValueError("anchor and positive must be [B, dim] with equal dim")
    if negatives is not None:
        if positive.shape[0] != anchor.shape[0]:
            raise ValueError("anchor and positive must have the same batch size")
        negatives = negatives.detach().contiguous().float()
    if per_row:
        return _InfoNceRows.apply(anchor.contiguous().float(), positive.contiguous().float(), negatives, float(temperature),
                                  int(label_offset))
    return _InfoNce.apply(anchor.contiguous().float(), positive.contiguous().float(), negatives, float(temperature),
                          int(label_offset), int(mean_rows))


class _InfoNce3(torch.autograd.Function):
    @staticmethod
    def forward(ctx, Z, G, tau, label_offset):
        L = _hip.lib()
        sh = _hip.InfoNce3Shape()
        _, sh.B, sh.P = Z.shape
        sh.tau = tau
        sh.Bp = 0 if G is None else G.shape[1]
        sh.label_offset = label_offset
        ws = torch.empty(L.ocean_infonce3_workspace(ctypes.byref(sh)), device=Z.device, dtype=torch.float32)
        if ws.numel() == 0:
            raise ValueError("infonce_pairs: label_offset + local rows must fit the gathered rows")
        losses = torch.zeros(3, device=Z.device, dtype=torch.float32)
        _hip.check(L.ocean_infonce3_fwd(ctypes.byref(sh), _hip.dev_ptr(Z, "projections"), _hip.dev_ptr(G, "gathered projections"),
                                        _hip.dev_ptr(ws), ws.numel(), _hip.dev_ptr(losses), _hip.stream()), "ocean_infonce3_fwd")
        ctx.sh = sh
        ctx.save_for_backward(ws)
        ctx.shapes = (Z.shape, None if G is None else G.shape)
        return losses

    @staticmethod
    def backward(ctx, dlosses):
        L = _hip.lib()
        (ws,) = ctx.saved_tensors
        sh = ctx.sh
        wb = torch.empty(L.ocean_infonce3_bwd_workspace(ctypes.byref(sh)), device=ws.device, dtype=torch.float32)
        dZ = torch.empty(ctx.shapes[0], device=ws.device, dtype=torch.float32)
        dG = None if ctx.shapes[1] is None else torch.empty(ctx.shapes[1], device=ws.device, dtype=torch.float32)
        _hip.check(L.ocean_infonce3_bwd(ctypes.byref(sh), _hip.dev_ptr(ws), _hip.dev_ptr(wb), wb.numel(),
                                        _hip.dev_ptr(dlosses.contiguous().float(), "dlosses"), _hip.dev_ptr(dZ), _hip.dev_ptr(dG),
                                        _hip.stream()), "ocean_infonce3_bwd")
        return dZ, dG, None, None


def infonce_pairs(projections: torch.Tensor, temperature: float = 0.1, gathered: Optional[torch.Tensor] = None,
                  label_offset: int = 0) -> torch.Tensor:
    """The in-batch InfoNCE losses of the pairs (0,1), (0,2), (1,2) of `projections` [3, B, P] as one [3] tensor: what
    three InfoNCELoss.forward(anchor, positive) calls return (graph_fusion.py:112-162, 231-249), from one normalisation,
    one batched similarity launch and one row pass.  `gathered` [3, B_all, P] (data parallel): the projections of every
    rank, whose rows serve as positives; local row r then pairs with gathered row label_offset + r.  The backward pass
    consumes the saved state: differentiate once."""
    if projections.dim() != 3 or projections.shape[0] != 3:
        raise ValueError("projections must be [3, B, dim]")
    if gathered is not None:
        if gathered.dim() != 3 or gathered.shape[0] != 3 or gathered.shape[2] != projections.shape[2]:
            raise ValueError("gathered must be [3, B_all, dim]")
        gathered = gathered.contiguous().float()
    return _InfoNce3.apply(projections.contiguous().float(), gathered, float(temperature), int(label_offset))


class StackedLosses(dict):
    """A dictionary of scalar losses that may also carry them as ONE tensor, `stacked` [n] in the dictionary's order
    (None when the entries are separate tensors): combine_losses then reads one operand and its backward writes one."""
    stacked: Optional[torch.Tensor] = None


class LossDict(dict):
    """compute_loss's result; `vec` (or None) holds [total, prediction, contrastive] as one device tensor, so that the
    learner's read-back needs no stacking launch."""
    vec: Optional[torch.Tensor] = None


class _CombineLosses(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, stacked, wp, wc):
        out = torch.empty(3, device=pred.device, dtype=torch.float32)
        n = 0 if stacked is None else stacked.numel()
        _hip.check(_hip.lib().ocean_loss_combine_fwd(_hip.dev_ptr(pred, "prediction loss"), _hip.dev_ptr(stacked, "contrastive losses"), n,
                                                     wp, wc, _hip.dev_ptr(out), _hip.stream()), "ocean_loss_combine_fwd")
        ctx.cfg = (wp, wc, n, None if stacked is None else stacked.shape)
        ctx.set_materialize_grads(False)
        total, csum = out[0], out[2]
        ctx.mark_non_differentiable(out)
        return total, csum, out

    @staticmethod
    def backward(ctx, d_total, d_csum, _d_out):
        wp, wc, n, shape = ctx.cfg
        ref = d_total if d_total is not None else d_csum
        if ref is None:
            return None, None, None, None
        d_pred = torch.empty((), device=ref.device, dtype=torch.float32)
        d_c = None if n == 0 else torch.empty(shape, device=ref.device, dtype=torch.float32)
        f = lambda g: None if g is None else g.contiguous().float()
        _hip.check(_hip.lib().ocean_loss_combine_bwd(_hip.dev_ptr(f(d_total)), _hip.dev_ptr(f(d_csum)), n, wp, wc, _hip.dev_ptr(d_pred),
                                                     _hip.dev_ptr(d_c), _hip.stream()), "ocean_loss_combine_bwd")
        return d_pred, d_c, None, None


def combine_losses(pred: torch.Tensor, stacked: Optional[torch.Tensor], wp: float, wc: float):
    """(total, contrastive sum, [total, pred, contrastive sum]) with total = wp * pred + wc * (0 + stacked[0] + ...),
    the arithmetic of OCEANModel.compute_loss (ocean_model.py:257-266) in one launch (one more in backward)."""
    if pred.dim() != 0 or pred.dtype != torch.float32 or (stacked is not None and (stacked.dim() != 1 or stacked.dtype != torch.float32)):
        raise ValueError("combine_losses takes an fp32 scalar and an fp32 vector")
    return _CombineLosses.apply(pred, None if stacked is None else stacked.contiguous(), float(wp), float(wc))


_loss_states = {}


def _loss_state(device) -> torch.Tensor:
    """The zero-initialised ocean_loss_state of `device` (per-block sums and the finished-block counter of
    ocean_pred_total_fwd), made on first use and kept: the kernel leaves the counter at zero."""
    key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
    t = _loss_states.get(key)
    if t is None:
        t = _loss_states[key] = torch.zeros(512 + 4, device=device, dtype=torch.float32)
    return t


class _PredTotal(torch.autograd.Function):
    @staticmethod
    def forward(ctx, probs, targets, mean_n, stacked, wp, wc):
        out = torch.empty(3, device=probs.device, dtype=torch.float32)
        n_c = 0 if stacked is None else stacked.numel()
        _hip.check(_hip.lib().ocean_pred_total_fwd(_hip.dev_ptr(probs, "probs"), _hip.dev_ptr(targets, "targets"), probs.numel(), mean_n,
                                                   _hip.dev_ptr(stacked, "contrastive losses"), n_c, wp, wc,
                                                   _hip.dev_ptr(_loss_state(probs.device)), _hip.dev_ptr(out), _hip.stream()),
                   "ocean_pred_total_fwd")
        ctx.cfg = (mean_n, wp, wc, n_c, None if stacked is None else stacked.shape)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(probs, targets)
        total, pred, csum = out[0], out[1], out[2]
        ctx.mark_non_differentiable(out)
        return total, pred, csum, out

    @staticmethod
    def backward(ctx, d_total, d_pred, d_csum, _d_out):
        mean_n, wp, wc, n_c, shape = ctx.cfg
        probs, targets = ctx.saved_tensors
        if d_total is None and d_pred is None and d_csum is None:
            return None, None, None, None, None, None
        dp = torch.empty_like(probs)
        d_c = None if n_c == 0 else torch.empty(shape, device=probs.device, dtype=torch.float32)
        f = lambda g: None if g is None else g.contiguous().float()
        _hip.check(_hip.lib().ocean_pred_total_bwd(_hip.dev_ptr(probs), _hip.dev_ptr(targets), _hip.dev_ptr(f(d_total)), _hip.dev_ptr(f(d_csum)),
                                                   _hip.dev_ptr(f(d_pred)), probs.numel(), mean_n, n_c, wp, wc, _hip.dev_ptr(dp),
                                                   _hip.dev_ptr(d_c), _hip.stream()), "ocean_pred_total_bwd")
        return dp, None, None, d_c, None, None


def prediction_and_total(probs: torch.Tensor, targets: torch.Tensor, reduction: str, stacked: Optional[torch.Tensor], wp: float,
                         wc: float):
    """(total, prediction loss, contrastive sum, [total, prediction, contrastive sum]): binary_cross_entropy(probs,
    targets, reduction) followed by combine_losses, as OCEANModel.compute_loss applies them (ocean_model.py:249-266), in
    one launch (one more in backward).  reduction 'mean' or 'sum'."""
    if probs.shape != targets.shape:
        raise ValueError(f"Using a target size ({tuple(targets.shape)}) that is different to the input size "
                         f"({tuple(probs.shape)}) is deprecated. Please ensure they have the same size.")
    if reduction not in ("mean", "sum"):
        raise ValueError(f"{reduction} is not a valid value for reduction")
    if stacked is not None and (stacked.dim() != 1 or stacked.dtype != torch.float32):
        raise ValueError("prediction_and_total takes the contrastive losses as one fp32 vector")
    return _PredTotal.apply(probs.contiguous().float(), targets.to(probs.device).contiguous().float(),
                            0 if reduction == "mean" else 1, None if stacked is None else stacked.contiguous(), float(wp), float(wc))


class _Bce(torch.autograd.Function):
    @staticmethod
    def forward(ctx, probs, targets, mean_n):
        loss = torch.zeros((), device=probs.device, dtype=torch.float32)
        _hip.check(_hip.lib().ocean_bce_fwd(_hip.dev_ptr(probs, "probs"), _hip.dev_ptr(targets, "targets"), probs.numel(),
                                            mean_n, _hip.dev_ptr(loss), _hip.stream()), "ocean_bce_fwd")
        ctx.mean_n = mean_n
        ctx.save_for_backward(probs, targets)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        probs, targets = ctx.saved_tensors
        dp = torch.empty_like(probs)
        _hip.check(_hip.lib().ocean_bce_bwd(_hip.dev_ptr(probs), _hip.dev_ptr(targets), _hip.dev_ptr(dloss.contiguous().float()),
                                            probs.numel(), ctx.mean_n, _hip.dev_ptr(dp), _hip.stream()), "ocean_bce_bwd")
        return dp, None, None


class _BceElem(torch.autograd.Function):
    """reduction='none': the per-element loss, same shape as the input."""

    @staticmethod
    def forward(ctx, probs, targets):
        out = torch.empty_like(probs)
        _hip.check(_hip.lib().ocean_bce_elem_fwd(_hip.dev_ptr(probs, "probs"), _hip.dev_ptr(targets, "targets"), probs.numel(),
                                                 _hip.dev_ptr(out), _hip.stream()), "ocean_bce_elem_fwd")
        ctx.save_for_backward(probs, targets)
        return out

    @staticmethod
    def backward(ctx, dout):
        probs, targets = ctx.saved_tensors
        dp = torch.empty_like(probs)
        _hip.check(_hip.lib().ocean_bce_elem_bwd(_hip.dev_ptr(probs), _hip.dev_ptr(targets), _hip.dev_ptr(dout.contiguous().float()),
                                                 probs.numel(), _hip.dev_ptr(dp), _hip.stream()), "ocean_bce_elem_bwd")
        return dp, None


def binary_cross_entropy(probs: torch.Tensor, targets: torch.Tensor, reduction: str = "mean") -> torch.Tensor:
    """F.binary_cross_entropy on probabilities (ocean_model.py:249-253), log terms clamped at -100."""
    if probs.shape != targets.shape:
        raise ValueError(f"Using a target size ({tuple(targets.shape)}) that is different to the input size "
                         f"({tuple(probs.shape)}) is deprecated. Please ensure they have the same size.")
    if reduction == "none":
        return _BceElem.apply(probs.contiguous().float(), targets.to(probs.device).contiguous().float())
    if reduction not in ("mean", "sum"):
        raise ValueError(f"{reduction} is not a valid value for reduction")
    loss = _Bce.apply(probs.contiguous().float(), targets.to(probs.device).contiguous().float(),
                      0 if reduction == "mean" else 1)
    return loss


def mean_tokens(x: torch.Tensor) -> torch.Tensor:
    """[B,L,C] -> [B,C] mean over L (log-embedding sequences, ocean_model.py:179-181).  Inputs only: no gradient."""
    if x.dim() != 3:
        raise ValueError("expected [batch, tokens, dim]")
    if x.requires_grad:
        raise NotImplementedError("mean_tokens is applied to model inputs and carries no gradient")
    x = x.contiguous().float()
    out = torch.empty(x.shape[0], x.shape[2], device=x.device, dtype=torch.float32)
    _hip.check(_hip.lib().ocean_mean_mid_f32(_hip.dev_ptr(x, "logs"), _hip.dev_ptr(out), x.shape[0], x.shape[1], x.shape[2],
                                             _hip.stream()), "ocean_mean_mid_f32")
    return out


class _Mse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b):
        loss = torch.zeros((), device=a.device, dtype=torch.float32)
        _hip.check(_hip.lib().ocean_mse_fwd(_hip.dev_ptr(a), _hip.dev_ptr(b), a.numel(), _hip.dev_ptr(loss), _hip.stream()), "ocean_mse_fwd")
        ctx.save_for_backward(a, b)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        a, b = ctx.saved_tensors
        da = torch.empty_like(a)
        _hip.check(_hip.lib().ocean_mse_bwd(_hip.dev_ptr(a), _hip.dev_ptr(b), _hip.dev_ptr(dloss.contiguous().float()), a.numel(),
                                            _hip.dev_ptr(da), _hip.stream()), "ocean_mse_bwd")
        return da, None


def mse_loss(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """nn.MSELoss()(a, b) with the gradient flowing to `a` (trainer.py:94: b is the detached previous batch)."""
    if a.shape != b.shape:
        raise ValueError(f"mse_loss needs equal shapes, got {tuple(a.shape)} and {tuple(b.shape)}")
    return _Mse.apply(a.contiguous().float(), b.detach().contiguous().float())


class _Diversity(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        L = _hip.lib()
        B, E = x.shape
        ws = torch.empty(L.ocean_diversity_workspace(B, E), device=x.device, dtype=torch.float32)
        loss = torch.zeros((), device=x.device, dtype=torch.float32)
        _hip.check(L.ocean_diversity_fwd(_hip.dev_ptr(x), B, E, _hip.dev_ptr(ws), ws.numel(), _hip.dev_ptr(loss), _hip.stream()),
                   "ocean_diversity_fwd")
        ctx.shape = (B, E)
        ctx.save_for_backward(ws)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        (ws,) = ctx.saved_tensors
        B, E = ctx.shape
        dx = torch.empty(B, E, device=ws.device, dtype=torch.float32)
        ws = ws.clone()                      # backward overwrites the similarity matrix; keep double-backward-free reuse safe
        _hip.check(_hip.lib().ocean_diversity_bwd(B, E, _hip.dev_ptr(ws), _hip.dev_ptr(dloss.contiguous().float()), _hip.dev_ptr(dx),
                                                  _hip.stream()), "ocean_diversity_bwd")
        return dx


def diversity_loss(x: torch.Tensor) -> torch.Tensor:
    """mean over i != j of |cos(x_i, x_j)| (trainer.py:97-108)."""
    if x.dim() != 2:
        raise ValueError("expected [batch, dim]")
    return _Diversity.apply(x.contiguous().float())


# ---------------------------------------------------------------- sequences: attention without stored weights, layer norm
# Small calls are bound by what the host does for them, so these two functions pack their shape structures in one step, ask
# for the raw stream handle, and go around autograd where nothing needs a gradient, outside traces and forward-mode levels.
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_pack_attention = struct.Struct("@9if4i28l").pack            # ocean_attention_shape
_pack_norm = struct.Struct("@l2if4x4l").pack                 # ocean_layer_norm_shape


def _stream_of(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _gpu(t: torch.Tensor, name: str, index: Optional[int] = None) -> int:
    """The GPU `t` lives on, which must be number `index` if that is given."""
    at = t.get_device()
    if at < 0:
        raise _hip.OceanHipError(f"{name} must live on the GPU (got {t.device}); the HIP path has no CPU fallback")
    if index is not None and at != index:
        raise ValueError(f"{name} lives on {t.device}, the other inputs on cuda:{index}")
    return at


def _fp32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.float().contiguous()


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised tensor in t's memory order, features innermost."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _once() -> None:
    if torch.is_grad_enabled():
        raise RuntimeError("the backward pass of this operator cannot itself be differentiated (create_graph=True)")


def _through_autograd(grad: bool) -> bool:
    """Whether a call has to go through its autograd function: for a gradient, in a trace (which records the function but would
    miss what the library writes) and inside a forward-mode level (where the function refuses a tangent that would be lost)."""
    return (grad and torch.is_grad_enabled()) or torch._C._get_tracing_state() is not None or forward_ad._current_level >= 0


_NO_STRIDES = (0, 0, 0)


def _attention_forward(q, k, v, mask, lengths, starts, table, cfg, want_lse):
    """(out, lse or None, what the backward call packs again)"""
    causal, start, scale, max_distance, both = cfg
    out = _like(q)
    if out.numel() == 0 or k.numel() == 0:
        return out.zero_(), None, None
    L = _hip.lib()
    B, H, Lq, d = q.shape
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    head = (B, H, k.shape[1], Lq, k.shape[2], d, _DTYPES[q.dtype], causal, start, scale, 0 if table is None else table.shape[0], max_distance, both)
    loose = (qp % 16 != 0) | (kp % 16 != 0) << 1 | (vp % 16 != 0) << 2
    strides = (*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3])
    mask_strides = (0, 0, 0, 0) if mask is None else mask.stride()
    sh = _pack_attention(*head, loose, *strides, *_NO_STRIDES, *_NO_STRIDES, *_NO_STRIDES, *_NO_STRIDES, *mask_strides)
    dev = q.device
    lse = torch.empty((B, H, Lq), device=dev, dtype=torch.float32) if want_lse else None
    n = L.ocean_attention_fwd_workspace(sh)
    ws = torch.empty(n, device=dev, dtype=torch.float32) if n else None
    rc = L.ocean_attention_fwd(sh, qp, kp, vp, _at(mask), _at(lengths), _at(starts), _at(table), _at(ws), n, out.data_ptr(), _at(lse), _stream_of(dev))
    if rc:
        _hip.check(rc, "ocean_attention_fwd")
    return out, lse, (head, loose, strides, mask_strides)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, lengths, starts, table, cfg):
        out, lse, ctx.packed = _attention_forward(q, k, v, mask, lengths, starts, table, cfg, True)
        ctx.save_for_backward(q, k, v, mask, lengths, starts, table, out, lse)
        return out

    @staticmethod
    def backward(ctx, d_out):
        _once()
        q, k, v, mask, lengths, starts, table, out, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        if lse is None:                                       # no query or no key: nothing depends on anything
            dq, dk, dv, dt = (torch.zeros_like(t) if need[n] else None for n, t in ((0, q), (1, k), (2, v), (6, table)))
            return dq, dk, dv, None, None, None, dt, None
        L = _hip.lib()
        dev = q.device
        if dev.index != torch.cuda.current_device():
            with torch.cuda.device(dev):
                return _Attention.backward(ctx, d_out)
        if d_out.stride(3) != 1:
            d_out = d_out.contiguous()
        dq, dk, dv, dt = (_like(t) if need[n] else None for n, t in ((0, q), (1, k), (2, v), (6, table)))
        head, loose, strides, mask_strides = ctx.packed
        gp = d_out.data_ptr()
        st = lambda t: _NO_STRIDES if t is None else t.stride()[:3]
        sh = _pack_attention(*head, loose | (gp % 16 != 0) << 3, *strides, *d_out.stride()[:3], *st(dq), *st(dk), *st(dv), *mask_strides)
        n = L.ocean_attention_bwd_workspace(sh)
        ws = lse.new_empty(n)
        rc = L.ocean_attention_bwd(sh, q.data_ptr(), k.data_ptr(), v.data_ptr(), _at(mask), _at(lengths), _at(starts), _at(table), out.data_ptr(),
                                   lse.data_ptr(), gp, ws.data_ptr(), n, _at(dq), _at(dk), _at(dv), _at(dt), _stream_of(dev))
        if rc:
            _hip.check(rc, "ocean_attention_bwd")
        return dq, dk, dv, None, None, None, dt, None


def _attention(q, k, v, mask, lengths, starts, table, cfg):
    if _through_autograd(q.requires_grad or k.requires_grad or v.requires_grad or (table is not None and table.requires_grad)):
        return _Attention.apply(q, k, v, mask, lengths, starts, table, cfg)
    return _attention_forward(q, k, v, mask, lengths, starts, table, cfg, False)[0]


def _per_sample(t: torch.Tensor, name: str, B: int, index: int) -> torch.Tensor:
    _gpu(t, name, index)
    if t.dtype != torch.int32 or t.shape != (B,):
        raise ValueError(f"{name} must be an int32 tensor of shape ({B},), got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, mask: Optional[torch.Tensor] = None,
              key_lengths: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
              query_start: Union[int, torch.Tensor, None] = None, position_table: Optional[torch.Tensor] = None,
              max_distance: int = 128, bidirectional: bool = True) -> torch.Tensor:
    """softmax(scale * Q K^T + position bias) V without the weights in memory, for training (the backward pass recomputes
    them) and serving (single tokens over a long cache); ScaledDotProductAttention (multi_factor_attention.py:34-65) is the form
    that returns the weights.

    query [batch, heads, queries, d], key / value [batch, key heads, keys, d] in fp32 or bf16, d at most 128, any strides (a
    transposed view of a projection's [batch, length, heads * d] needs no copy; the result has the query's memory order).
    Query heads share key heads in equal groups; batch * heads * ceil(queries / 128), and the same of key heads and keys, are below
    2^24 (without gradients only the first, or batch * key heads for up to 32 queries a key head).  Products and sums accumulate in fp32; the probabilities enter the second
    product in the inputs' type.

    mask: bool or uint8, broadcastable to [batch, heads, queries, keys], nonzero = allowed.  key_lengths: int32 [batch] on the
    GPU, each sample's key count (clamped to 0..keys); what lies behind is never read, its gradient is zero.  The same holds for
    keys that a mask without a query axis takes (size 1 there; with shared key heads without a head axis too), and for queries
    that one without a key axis takes.  Any other place that a mask or `causal` takes away still enters sums, with weight zero:
    its key, value, query and the gradient that arrives have to be finite.  A query with no allowed key gets zeros, and passes
    no gradient.
    query_start: position of the first query among the keys, an int or int32 [batch] on the GPU; default keys - queries (the
    queries are the last keys).  It places `causal` (keys up to the query's own position) and the position bias.
    position_table [buckets, heads]: the learned bias of the distance key - query position, added to the scaled scores.
    bidirectional: half of the buckets for each sign; else keys after the query count as distance 0.  With E = half of one
    side's buckets, distances below E have a bucket each, the others share the rest in logarithmic steps up to max_distance
    (at most 1024; 128 buckets at most)."""
    if query.dim() != 4 or key.dim() != 4 or value.shape != key.shape:
        raise ValueError(f"query [batch, heads, queries, d] and key, value [batch, key heads, keys, d] expected, got {tuple(query.shape)}, "
                         f"{tuple(key.shape)}, {tuple(value.shape)}")
    B, H, Lq, d = query.shape
    Hk, Lk = key.shape[1], key.shape[2]
    if key.shape[0] != B or key.shape[3] != d or Hk == 0 or H == 0 or H % Hk != 0:
        raise ValueError(f"key heads must divide the heads, batch and d must agree: query {tuple(query.shape)}, key {tuple(key.shape)}")
    if query.dtype not in (torch.float32, torch.bfloat16) or key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError(f"attention takes fp32 or bf16 inputs of one type, got {query.dtype}, {key.dtype}, {value.dtype}")
    if not 1 <= d <= 128:
        raise ValueError(f"attention takes 1 to 128 features a head, got {d}")
    index = _gpu(query, "query")
    _gpu(key, "key", index)
    _gpu(value, "value", index)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"scale must be from 1e-30 to 1e30, got {scale}")
    if mask is not None:
        _gpu(mask, "mask", index)
        if mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"mask must be bool or uint8 (nonzero = allowed), got {mask.dtype}")
        mask = mask.view(torch.uint8).expand(B, H, Lq, Lk)
    if key_lengths is not None:
        key_lengths = _per_sample(key_lengths, "key_lengths", B, index)
    starts, start = None, Lk - Lq
    if isinstance(query_start, torch.Tensor):
        starts = _per_sample(query_start, "query_start", B, index)
    elif query_start is not None:
        start = int(query_start)
    if not -(1 << 30) <= start <= (1 << 30):
        raise ValueError(f"query_start must be within 2^30, got {start}")
    if position_table is not None:
        _gpu(position_table, "position_table", index)
        if position_table.dim() != 2 or position_table.shape[1] != H or not position_table.is_floating_point():
            raise ValueError(f"position_table must be [buckets, {H}], got {tuple(position_table.shape)} {position_table.dtype}")
        nb = position_table.shape[0]
        side = nb // 2 if bidirectional else nb
        if side < 2 or nb > 128 or (bidirectional and nb % 2):
            raise ValueError(f"2 to 128 buckets expected (an even number, 4 at least, when bidirectional), got {nb}")
        if not side // 2 < max_distance <= 1024:
            raise ValueError(f"max_distance must be above {side // 2} and at most 1024, got {max_distance}")
        position_table = _fp32(position_table)
    least = 4 if query.dtype == torch.float32 else 8
    if d < least:                                             # the kernels read 16 bytes at a time
        pad = lambda t: torch.nn.functional.pad(t, (0, least - d))
        query, key, value = pad(query), pad(key), pad(value)
    q, k, v = (t if t.stride(3) == 1 else t.contiguous() for t in (query, key, value))
    cfg = (int(bool(causal)), start, scale, int(max_distance), int(bool(bidirectional)))
    args = (q, k, v, mask, key_lengths, starts, position_table, cfg)
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            out = _attention(*args)
    else:
        out = _attention(*args)
    return out[..., :d] if d < least else out


def _row_stride(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """`t` (or a dense copy) as rows of its last dimension at one stride."""
    W = t.shape[-1]
    rows = t.numel() // W
    if t.is_contiguous():
        return t, W
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= W:
        return t, t.stride(0) if rows > 1 else W
    return t.contiguous(), W


def _norm_forward(x, residual, weight, bias, eps, want_stats):
    """(y, sum or None, the normalised rows, their stride, statistics or None)"""
    W = x.shape[-1]
    dev = x.device
    y = x.new_empty(x.shape)
    total = None if residual is None else x.new_empty(x.shape)
    rows = x.numel() // W
    if rows == 0:
        return y, total, x, W, None
    x, ldx = _row_stride(x)
    residual, ldr = (None, 0) if residual is None else _row_stride(residual)
    stats = torch.empty((rows, 2), device=dev, dtype=torch.float32) if want_stats else None
    rc = _hip.lib().ocean_layer_norm_fwd(_pack_norm(rows, W, _DTYPES[y.dtype], eps, ldx, ldr, 0, 0), x.data_ptr(), _at(residual), _at(weight), _at(bias),
                                         y.data_ptr(), _at(total), _at(stats), _stream_of(dev))
    if rc:
        _hip.check(rc, "ocean_layer_norm_fwd")
    return (y, total, x, ldx, stats) if total is None else (y, total, total, W, stats)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        ctx.set_materialize_grads(False)
        y, total, rows, ctx.ldx, stats = _norm_forward(x, residual, weight, bias, eps, True)
        ctx.save_for_backward(rows, stats, weight)
        ctx.shape, ctx.eps = x.shape, eps
        return y if total is None else (y, total)

    @staticmethod
    def backward(ctx, dy, d_sum=None):
        _once()
        need_x, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        if dy is None and d_sum is None:
            return None, None, None, None, None
        x, stats, weight = ctx.saved_tensors
        W, dev = ctx.shape[-1], x.device
        if dy is None or stats is None:                       # only the sum was used, or there are no rows
            zeros = lambda n: torch.zeros(W, device=dev, dtype=torch.float32) if n else None
            dx = d_sum if dy is None else torch.zeros(ctx.shape, device=dev, dtype=x.dtype)
            return dx if need_x else None, dx if need_r else None, zeros(need_w), zeros(need_b), None
        if dev.index != torch.cuda.current_device():
            with torch.cuda.device(dev):
                return _LayerNorm.backward(ctx, dy, d_sum)
        L = _hip.lib()
        dx = x.new_empty(ctx.shape) if need_x or need_r else None
        dw = stats.new_empty(W) if need_w else None
        db = stats.new_empty(W) if need_b else None
        dy, ldy = _row_stride(dy)
        d_sum, lds = (None, 0) if d_sum is None else _row_stride(d_sum)
        sh = _pack_norm(x.numel() // W, W, _DTYPES[x.dtype], ctx.eps, ctx.ldx, 0, ldy, lds)
        n = L.ocean_layer_norm_bwd_workspace(sh) if need_w or need_b else 0
        ws = stats.new_empty(n) if n else None
        rc = L.ocean_layer_norm_bwd(sh, x.data_ptr(), stats.data_ptr(), _at(weight), dy.data_ptr(), _at(d_sum), _at(ws), n, _at(dx), _at(dw), _at(db),
                                    _stream_of(dev))
        if rc:
            _hip.check(rc, "ocean_layer_norm_bwd")
        return dx if need_x else None, dx if need_r else None, dw, db, None


def _norm_parameter(t: torch.Tensor, name: str, W: int, index: int) -> torch.Tensor:
    _gpu(t, name, index)
    if t.dim() != 1 or t.shape[0] != W or not t.is_floating_point():
        raise ValueError(f"{name} must be [{W}], got {tuple(t.shape)} {t.dtype}")
    return _fp32(t)


def _norm(x, residual, weight, bias, eps):
    W = x.shape[-1] if x.dim() else 0
    if not 1 <= W <= 1 << 24:
        raise ValueError(f"layer_norm takes [..., width] with 1 to 2^24 columns, got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"layer_norm takes fp32, bf16 or fp16 rows, got {x.dtype}")
    index = _gpu(x, "x")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    grad = x.requires_grad
    if residual is not None:
        _gpu(residual, "residual", index)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"x and residual must agree in shape and type, got {tuple(x.shape)} {x.dtype}, {tuple(residual.shape)} {residual.dtype}")
        grad = grad or residual.requires_grad
    if weight is not None:
        weight = _norm_parameter(weight, "weight", W, index)
        grad = grad or weight.requires_grad
    if bias is not None:
        bias = _norm_parameter(bias, "bias", W, index)
        grad = grad or bias.requires_grad
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _norm_call(x, residual, weight, bias, float(eps), grad)
    return _norm_call(x, residual, weight, bias, float(eps), grad)


def _norm_call(x, residual, weight, bias, eps, grad):
    if _through_autograd(grad):
        return _LayerNorm.apply(x, residual, weight, bias, eps)
    y, total = _norm_forward(x, residual, weight, bias, eps, False)[:2]
    return y if total is None else (y, total)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension, any width, fp32, bf16 or fp16 (statistics and
    the weights' gradients in fp32, the latter summed in a fixed order); weight and bias [width] in any floating type, or None."""
    return _norm(x, None, weight, bias, eps)


def add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """(layer_norm(s), s) with s = x + residual, rounded to their type, in one pass; the gradient of s joins the norm's."""
    return _norm(x, residual, weight, bias, eps)

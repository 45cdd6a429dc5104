"""The SAE and the router as functions of torch.autograd (an extension).

Same results as the functions of the same purpose elsewhere in the package,
and gradients by the kernels of ``backward`` and ``routing``:

    topk_sae_forward(X, W_enc, b_enc, W_dec, b_dec, k) -> x_hat, vals, idxs
    topk_sae_encode(X, W_enc, b_enc, k)                -> vals, idxs
    topk_sae_decode(vals, idxs, W_dec, b_dec)          -> x_hat
    route_experts(logits, k, ...)                      -> weights, experts

idxs and experts have no gradient; gradients of gradients are not supported.

These are for eager programs.  Under CUDA-graph capture they refuse: autograd
adds a leaf's gradient on the stream where the leaf was first used, and a
capture that joins work of an eager graph's stream cannot be ended cleanly.
Capture the explicit calls instead (``train.TopkSAETrainer`` does).
"""
from __future__ import annotations

import torch

from . import backward as _bw
from . import decode as _decode
from . import ops as _ops
from . import routing as _routing
from .native import _require


def _not_capturing(device):
    if device.type == "cuda":
        with torch.cuda.device(device):
            _require(not torch.cuda.is_current_stream_capturing(),
                     "autograd functions cannot be captured in a CUDA graph; capture the explicit *_backward calls")


def _grad(want, t):
    return t if want else None


class _Forward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, W_enc, b_enc, W_dec, b_dec, k):
        _not_capturing(X.device)
        _require(W_enc.dtype == X.dtype and W_dec.dtype == X.dtype and W_dec.shape == W_enc.shape,
                 "X, W_enc and W_dec must have one dtype, W_enc and W_dec one shape")
        x_hat, vals, idxs = _decode.topk_sae_forward(X, W_enc, b_enc, W_dec, b_dec, k)
        ctx.save_for_backward(X, W_enc, W_dec, vals, idxs)
        ctx.bias_dtypes = b_enc.dtype, None if b_dec is None else b_dec.dtype
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(idxs)
        return x_hat, vals, idxs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, gv, _):
        X, W_enc, W_dec, vals, idxs = ctx.saved_tensors
        _not_capturing(X.device)
        if g is None:
            g = torch.zeros(X.shape, dtype=torch.float32, device=X.device)
        r = _bw.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, grad_vals=gv, need_dx=ctx.needs_input_grad[0])
        need, (be, bd) = ctx.needs_input_grad, ctx.bias_dtypes
        return (r.X, _grad(need[1], r.W_enc), _grad(need[2], r.b_enc.to(be)), _grad(need[3], r.W_dec),
                _grad(need[4], None if bd is None else r.b_dec.to(bd)), None)


class _Encode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, W_enc, b_enc, k):
        _not_capturing(X.device)
        vals, idxs = _ops.topk_sae_cuda_exact(X, W_enc, b_enc, k)
        ctx.save_for_backward(X, W_enc, idxs)
        ctx.bias_dtype = b_enc.dtype
        ctx.mark_non_differentiable(idxs)
        return vals, idxs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gv, _):
        X, W_enc, idxs = ctx.saved_tensors
        _not_capturing(X.device)
        dX, dW, db = _bw.topk_sae_encode_backward(gv, idxs, X, W_enc, need_dx=ctx.needs_input_grad[0])
        need = ctx.needs_input_grad
        return dX, _grad(need[1], dW), _grad(need[2], db.to(ctx.bias_dtype)), None


class _Decode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, vals, idxs, W_dec, b_dec):
        _not_capturing(vals.device)
        ctx.save_for_backward(vals, idxs, W_dec)
        ctx.bias_dtype = None if b_dec is None else b_dec.dtype
        return _decode.topk_sae_decode(vals, idxs, W_dec, b_dec)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        vals, idxs, W_dec = ctx.saved_tensors
        _not_capturing(vals.device)
        dv, dW, db = _bw.topk_sae_decode_backward(g, vals, idxs, W_dec)
        need = ctx.needs_input_grad
        return (_grad(need[0], dv.to(vals.dtype)), None, _grad(need[2], dW),
                None if ctx.bias_dtype is None else _grad(need[3], db.to(ctx.bias_dtype)))


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, how, select):
        _not_capturing(logits.device)
        weights, experts = _routing.route_experts(logits, k, **how, **select)
        ctx.save_for_backward(logits, experts)
        ctx.how = how
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gw, _):
        logits, experts = ctx.saved_tensors
        _not_capturing(logits.device)
        return _routing.route_experts_backward(gw, logits, experts, **ctx.how), None, None, None


def topk_sae_forward(X, W_enc, b_enc, W_dec, b_dec, k):
    """(x_hat (B, d) fp32, vals (B, k) fp32, idxs (B, k) int32): encode by exact top-k, then decode.
    X, W_enc and W_dec have one dtype; b_dec may be None; k is one that ``topk_sae_cuda_exact`` takes."""
    return _Forward.apply(X, W_enc, b_enc, W_dec, b_dec, int(k))


def topk_sae_encode(X, W_enc, b_enc, k):
    """(vals, idxs) of ``topk_sae_cuda_exact``, vals differentiable in X, W_enc and b_enc."""
    return _Encode.apply(X, W_enc, b_enc, int(k))


def topk_sae_decode(vals, idxs, W_dec, b_dec=None):
    """x_hat of ``topk_sae_decode``, differentiable in vals, W_dec and b_dec."""
    return _Decode.apply(vals, idxs, W_dec, b_dec)


def route_experts(logits, k, *, score="softmax", bias=None, n_groups=1, topk_groups=1, renormalize=True, scale=1.0,
                  row_mask=None):
    """(weights, experts) of ``routing.route_experts``, weights differentiable in logits (not in bias)."""
    return _Route.apply(logits, k, {"score": score, "renormalize": renormalize, "scale": scale},
                        {"bias": None if bias is None else bias.detach(), "n_groups": n_groups,
                         "topk_groups": topk_groups, "row_mask": row_mask})

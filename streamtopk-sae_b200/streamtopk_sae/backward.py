"""Gradients of the top-k SAE over its sparse codes (an extension: the
reference does not train).

    x_hat = b_dec + sum_j vals[:, j] W_dec[idxs[:, j]]
    vals  = X . W_enc[idxs] + b_enc[idxs]          (idxs: no gradient)

``topk_sae_backward`` is the gradient of ``topk_sae_forward``: given dL/dx_hat it
returns those of X, W_enc, b_enc, W_dec, b_dec and vals from one walk over the
dictionary (stk_sae_backward).  ``topk_sae_decode_backward`` and
``topk_sae_encode_backward`` are its halves, for programs that do something to
the codes in between.  All are explicit calls that allocate their outputs and
can be captured in a CUDA graph; ``autograd`` has them as functions of
torch.autograd.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _capi
from .native import _DTYPE_CODE, _int32_indices, _launch, _require


class SAEGradients(NamedTuple):
    """Gradients by the name of what they belong to."""
    X: Optional[torch.Tensor]
    W_enc: Optional[torch.Tensor]
    b_enc: Optional[torch.Tensor]
    W_dec: Optional[torch.Tensor]
    b_dec: Optional[torch.Tensor]
    vals: Optional[torch.Tensor]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run(g, X, W_enc, W_dec, vals, idxs, gv, F, d, dtype, need_dx):
    dev = idxs.device
    B, k = idxs.shape
    _require(k >= 1, "vals and idxs must be (B, k) with k >= 1")
    dec, enc = W_dec is not None, W_enc is not None

    # (sizes one by one: as a tuple each allocation takes 0.7 us more)
    out = SAEGradients(torch.empty(B, d, dtype=dtype, device=dev) if need_dx else None,
                       torch.empty(F, d, dtype=dtype, device=dev) if enc else None,
                       torch.empty(F, dtype=torch.float32, device=dev) if enc else None,
                       torch.empty(F, d, dtype=dtype, device=dev) if dec else None,
                       torch.empty(d, dtype=torch.float32, device=dev) if dec else None,
                       torch.empty(B, k, dtype=torch.float32, device=dev) if dec else None)
    nbytes = _capi.sae_backward_workspace_bytes(B, k, F, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(dev, _capi.load().stk_sae_backward,
            _ptr(g), _ptr(X), _ptr(W_enc) if need_dx else None, _ptr(W_dec), _ptr(vals), idxs.data_ptr(), _ptr(gv),
            _ptr(out.W_enc), _ptr(out.b_enc), _ptr(out.W_dec), _ptr(out.b_dec), _ptr(out.vals), _ptr(out.X), B, k, F, d,
            _DTYPE_CODE[dtype], ws.data_ptr(), nbytes)
    return out


def _codes(vals, idxs):
    if idxs.dim() != 2 or vals.shape != idxs.shape:
        raise RuntimeError("vals and idxs must be (B, k)")
    return vals.float().contiguous(), _int32_indices(idxs)


def _same_device(first, *others):
    at = first.get_device()
    for t in (first, *others):
        if t is not None and t.get_device() != at or at < 0:
            raise RuntimeError("inputs must be on CUDA" if at < 0 or not t.is_cuda else "inputs must be on the same device")


def topk_sae_backward(grad_x_hat, X, W_enc, W_dec, vals, idxs, *, grad_vals=None, need_dx=False):
    """SAEGradients of ``topk_sae_forward`` from dL/dx_hat (B, d).

    X (B, d), W_enc and W_dec (F, d) in one dtype (fp32, fp16 or bf16); vals and
    idxs (B, k) as the forward call returned them (indices < 0 are passed over);
    grad_vals (B, k): dL/dvals other than through x_hat, e.g. of a penalty.
    Gradients of X (where need_dx), W_enc and W_dec have their dtype, the others
    are fp32; sums are fp32 and the same in every call.
    """
    _same_device(grad_x_hat, X, W_enc, W_dec, vals, idxs, grad_vals)
    _require(X.dim() == 2 and W_enc.dim() == 2 and W_enc.shape == W_dec.shape and W_enc.shape[1] == X.shape[1],
             "W_enc and W_dec must be (F, d), X (B, d)")
    _require(X.dtype in _DTYPE_CODE and W_enc.dtype == X.dtype and W_dec.dtype == X.dtype,
             "X, W_enc and W_dec must have one dtype: fp32, fp16, or bf16")
    vals, idxs = _codes(vals, idxs)
    _require(grad_x_hat.shape == X.shape and idxs.shape[0] == X.shape[0], "grad_x_hat must be (B, d), idxs (B, k)")
    _require(grad_vals is None or grad_vals.shape == idxs.shape, "grad_vals must be (B, k)")
    g = grad_x_hat.float().contiguous()
    gv = None if grad_vals is None else grad_vals.float().contiguous()
    F, d = W_dec.shape
    return _run(g, X.contiguous(), W_enc.contiguous(), W_dec.contiguous(), vals, idxs, gv, F, d, X.dtype, need_dx)


def topk_sae_decode_backward(grad_x_hat, vals, idxs, W_dec):
    """Gradients of ``topk_sae_decode``: (vals (B, k) fp32, W_dec (F, d) in its dtype, b_dec (d,) fp32)."""
    _same_device(grad_x_hat, vals, idxs, W_dec)
    _require(W_dec.dim() == 2 and W_dec.dtype in _DTYPE_CODE, "W_dec must be (F, d) fp32, fp16 or bf16")
    vals, idxs = _codes(vals, idxs)
    F, d = W_dec.shape
    _require(grad_x_hat.shape == (idxs.shape[0], d), "grad_x_hat must be (B, d)")
    r = _run(grad_x_hat.float().contiguous(), None, None, W_dec.contiguous(), vals, idxs, None, F, d, W_dec.dtype, False)
    return r.vals, r.W_dec, r.b_dec


def topk_sae_encode_backward(grad_vals, idxs, X, W_enc, *, need_dx=True):
    """Gradients of the encoder's vals at fixed idxs: (X (B, d) or None, W_enc (F, d), both in X's dtype, b_enc (F,)
    fp32), of vals[b, j] = X[b] . W_enc[idxs[b, j]] + b_enc[idxs[b, j]]."""
    _same_device(grad_vals, idxs, X, W_enc)
    _require(X.dim() == 2 and W_enc.dim() == 2 and W_enc.shape[1] == X.shape[1], "W_enc must be (F, d), X (B, d)")
    _require(X.dtype in _DTYPE_CODE and W_enc.dtype == X.dtype, "X and W_enc must have one dtype: fp32, fp16, or bf16")
    grad_vals, idxs = _codes(grad_vals, idxs)
    _require(idxs.shape[0] == X.shape[0], "idxs must be (B, k)")
    F, d = W_enc.shape
    r = _run(None, X.contiguous(), W_enc.contiguous(), None, None, idxs, grad_vals, F, d, X.dtype, need_dx)
    return r.X, r.W_enc, r.b_enc

"""Training steps of a top-k SAE on its reconstruction error (an extension).

    x_hat = topk_sae_forward(X, W_enc, b_enc, W_dec, b_dec, k)
    loss  = mean over the batch of |x_hat - X|^2
    gradients by topk_sae_backward, the four tensors' step by AdamW

The weights learn in fp32; the encoder and decoder read copies in ``dtype``.  The
AdamW step writes the copies along with the weights, and each step first takes
them from the weights again: they are the user's tensors, and what a program
does to them between steps (rows brought back to length 1, features started
anew, a checkpoint loaded) leaves no sign that could be relied on -- writes
through ``.data`` and replayed graphs count no version.  That reads and
writes 6 bytes an element of the dictionaries: with k=64, d=2048, F=65536 a step
of 4096 rows takes 3.32 ms instead of 3.06, with k=32, d=768 one of 128 rows 506
us instead of 414.
No part of a step waits for the GPU, so steps of one batch shape can be captured
in a CUDA graph and replayed (``capturable=True``).
"""
from __future__ import annotations

import torch

from .backward import topk_sae_backward
from .decode import topk_sae_forward
from .native import _require
from .optim import AdamW


class TopkSAETrainer:
    """W_enc, W_dec (F, d), b_enc (F,), b_dec (d,): fp32 CUDA tensors, updated in place, which may be changed in place
    between steps; k is one that ``topk_sae_cuda_exact`` takes.  Further arguments are AdamW's.  ``trainer.W_enc`` and
    ``.W_dec`` are the weights in ``dtype`` as the last step left them."""

    def __init__(self, W_enc, b_enc, W_dec, b_dec, k, *, dtype=torch.bfloat16, **adamw):
        self.params = (W_enc, b_enc, W_dec, b_dec)
        _require(all(p.dtype == torch.float32 and p.is_contiguous() for p in self.params),
                 "weights and biases must be contiguous fp32")
        _require(W_enc.dim() == 2 and W_enc.shape == W_dec.shape and b_enc.shape == W_enc.shape[:1]
                 and b_dec.shape == W_enc.shape[1:], "W_enc and W_dec must be (F, d), b_enc (F,), b_dec (d,)")
        self.k, self.dtype = int(k), dtype
        low = dtype != torch.float32
        with torch.inference_mode(False), torch.no_grad():  # steps inside and outside of inference mode write them
            self.W_enc, self.W_dec = (W.to(dtype) if low else W for W in (W_enc, W_dec))
        self.optimizer = AdamW(self.params, copies={W_enc: self.W_enc, W_dec: self.W_dec} if low else None, **adamw)

    @torch.no_grad()
    def step(self, X):
        """One step on X (B, d), in ``dtype``; returns the loss before it, as an fp32 CUDA scalar."""
        _require(X.dtype == self.dtype, "X must have the trainer's dtype")
        _require(X.dim() == 2 and X.shape[0] > 0, "X must be (B, d) with B >= 1")
        W_enc, b_enc, W_dec, b_dec = self.params
        if self.dtype != torch.float32:
            self.W_enc.copy_(W_enc)
            self.W_dec.copy_(W_dec)
        x_hat, vals, idxs = topk_sae_forward(X, self.W_enc, b_enc, self.W_dec, b_dec, self.k)
        error = x_hat.sub_(X)
        loss = error.square().sum() / X.shape[0]
        g = topk_sae_backward(error.mul_(2.0 / X.shape[0]), X, self.W_enc, self.W_dec, vals, idxs)
        self.optimizer.step([g.W_enc, g.b_enc, g.W_dec, g.b_dec])
        return loss

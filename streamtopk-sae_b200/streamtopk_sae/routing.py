"""Routing rows to experts: the router of a routed (switch) SAE, whose
dictionary is split over experts and each row encoded by a few of them (an
extension: the reference has one dictionary).

    s       = softmax(logits) or sigmoid(logits)
    experts = the k largest of logits, or of s + bias, per row
    weights = scale * s[experts], divided by their sum where renormalize

``route_experts`` (stk_route_forward) returns weights fp32 (N, k) and experts
int32 (N, k) like the top-k ops: best first, ties to the lower index, -1 with
weight 0 where nothing is left.  ``route_experts_backward`` is the weights'
gradient; ``autograd.route_experts`` joins the two.
``topk_sae_routed_encode`` routes a batch and encodes each row with its experts'
dictionaries; its codes index all dictionaries as one, so ``topk_sae_decode``
and ``topk_sae_backward`` take them as they are.
"""
from __future__ import annotations

import torch

from . import _capi
from .native import _DTYPE_CODE, _launch, _require

_SCORES = {"softmax": _capi.STK_SCORE_SOFTMAX, "sigmoid": _capi.STK_SCORE_SIGMOID}


def _logits(logits, score):
    if not logits.is_cuda:
        raise RuntimeError("logits must be on CUDA")
    if logits.dim() != 2 or logits.dtype not in _DTYPE_CODE:
        raise RuntimeError("logits must be (N, E) fp32, fp16 or bf16")
    if score not in _SCORES:
        raise RuntimeError("score must be 'softmax' or 'sigmoid'")
    N, E = logits.shape
    if not 1 <= E <= 1024:
        raise RuntimeError("need 1 <= E <= 1024 experts")
    if logits.is_contiguous():
        return logits, N, E, E
    if E > 1 and logits.stride(1) != 1 or N > 1 and logits.stride(0) < E:
        logits = logits.contiguous()
    return logits, N, E, logits.stride(0) if N > 1 else E


def route_experts(logits, k, *, score="softmax", bias=None, n_groups=1, topk_groups=1, renormalize=True, scale=1.0,
                  row_mask=None, return_counts=False):
    """(weights (N, k) fp32, experts (N, k) int32[, counts (E,) int32]) of router logits (N, E).

    bias (E,): added to the scores for the choice alone (load balance).
    n_groups, topk_groups: experts are chosen from the topk_groups groups of
    E / n_groups neighbours whose two best choices have the largest sums.
    row_mask (N,) bool: rows that are False get experts -1 and weights 0, and
    their logits are not used.  Experts with a logit of -inf or NaN are not
    chosen.  E <= 1024, k <= 32, n_groups <= 32.
    """
    logits, N, E, ld = _logits(logits, score)
    k, n_groups, topk_groups = int(k), int(n_groups), int(topk_groups)
    _require(1 <= topk_groups <= n_groups <= 32 and E % n_groups == 0,
             "need 1 <= topk_groups <= n_groups <= 32 and E a multiple of n_groups")
    _require(1 <= k <= min(32, topk_groups * (E // n_groups)), "k out of range")
    dev = logits.device
    if bias is not None:
        _require(bias.shape == (E,) and bias.device == dev, "bias must be (E,) on logits' device")
        bias = bias.float().contiguous()
    if row_mask is not None:
        _require(row_mask.shape == (N,) and row_mask.device == dev and row_mask.dtype == torch.bool,
                 "row_mask must be (N,) bool on logits' device")
        row_mask = row_mask.contiguous()
    weights = torch.empty(N, k, dtype=torch.float32, device=dev)
    experts = torch.empty(N, k, dtype=torch.int32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev) if return_counts else None
    _launch(dev, _capi.load().stk_route_forward,
            logits.data_ptr(), _DTYPE_CODE[logits.dtype], ld, None if bias is None else bias.data_ptr(),
            None if row_mask is None else row_mask.data_ptr(), weights.data_ptr(), experts.data_ptr(),
            None if counts is None else counts.data_ptr(), N, E, k, _SCORES[score], n_groups, topk_groups,
            bool(renormalize), scale)
    return (weights, experts, counts) if return_counts else (weights, experts)


def route_experts_backward(grad_weights, logits, experts, *, score="softmax", renormalize=True, scale=1.0):
    """Gradient (N, E), in logits' dtype, of route_experts' weights; experts as that call returned them."""
    logits, N, E, ld = _logits(logits, score)
    dev = logits.device
    _require(experts.dim() == 2 and experts.shape[0] == N and 1 <= experts.shape[1] <= min(32, E)
             and grad_weights.shape == experts.shape, "grad_weights and experts must be (N, k)")
    _require(experts.dtype == torch.int32, "experts must be int32")
    _require(experts.device == dev and grad_weights.device == dev, "inputs must be on the same device")
    experts = experts.contiguous()
    grad_weights = grad_weights.float().contiguous()
    grad = torch.empty(N, E, dtype=logits.dtype, device=dev)
    _launch(dev, _capi.load().stk_route_backward,
            grad_weights.data_ptr(), logits.data_ptr(), _DTYPE_CODE[logits.dtype], ld, experts.data_ptr(),
            grad.data_ptr(), N, E, experts.shape[1], _SCORES[score], bool(renormalize), scale)
    return grad


def topk_sae_routed_encode(X, logits, W_enc, b_enc, k, top_experts=1, **router):
    """Routed exact top-k encode.

    X (B, d), logits (B, E) of the router, W_enc (E, Fe, d) and b_enc (E, Fe):
    each row goes to its ``top_experts`` dictionaries (``router``: keyword
    arguments of ``route_experts``) and gets the k best features of each, by
    ``topk_sae_cuda_exact`` (k is one that it takes).  Returns (vals (B, top_experts * k) fp32, not yet
    weighted, idxs (B, top_experts * k) int32 into the dictionaries as one of
    E * Fe features, weights (B, top_experts) fp32, experts (B, top_experts)
    int32).  Codes of a row that is routed nowhere are 0 with index -1.  Reads
    the experts' loads back to the host, so it cannot be captured in a graph.
    """
    from .ops import topk_sae_cuda_exact
    _require(X.dim() == 2 and W_enc.dim() == 3 and W_enc.shape[2] == X.shape[1], "W_enc must be (E, Fe, d), X (B, d)")
    _require(b_enc.shape == W_enc.shape[:2], "b_enc must be (E, Fe)")
    _require(logits.shape == (X.shape[0], W_enc.shape[0]), "logits must be (B, E)")
    _require(W_enc.shape[0] * W_enc.shape[1] < 2 ** 31, "E * Fe features must fit int32 indices")
    _require(not router.get("return_counts", False), "return_counts is not an option here")
    B, m, Fe = X.shape[0], int(top_experts), W_enc.shape[1]
    weights, experts, counts = route_experts(logits, m, return_counts=True, **router)
    vals = torch.zeros((B * m, k), dtype=torch.float32, device=X.device)
    idxs = torch.full((B * m, k), -1, dtype=torch.int32, device=X.device)
    order = torch.argsort(experts.reshape(-1), stable=True)  # slots by expert; those routed nowhere (-1) first
    at = B * m - int(counts.sum())
    for e, n in enumerate(counts.tolist()):
        if n:
            slots = order[at:at + n]
            v, i = topk_sae_cuda_exact(X[slots // m], W_enc[e], b_enc[e], k)
            vals[slots] = v
            idxs[slots] = i + e * Fe
            at += n
    return vals.view(B, m * k), idxs.view(B, m * k), weights, experts

"""AdamW over many tensors in one launch, with states in 32 or 8 bits (an
extension: the reference does not train).

    m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

``adamw_step`` is the operator (stk_adamw_step); ``AdamW`` keeps the states and
calls it.  8-bit states are E4M3 codes of m and sqrt(v) with one fp32 scale for
every 256 consecutive elements of a tensor: 2.03 bytes an element instead of 8.
``copies`` are further outputs of the updated parameters in another type, e.g.
the bf16 weights that the encoder reads beside fp32 parameters that learn.

A step may be captured in a CUDA graph: give ``step`` (int64) and, where it
changes, ``lr`` (fp32) as one-element CUDA tensors, and advance ``step`` inside
the graph (``AdamW(capturable=True)`` does).
"""
from __future__ import annotations

import ctypes
from array import array
from itertools import chain
from operator import attrgetter

import torch

from . import _capi
from .native import _DTYPE_CODE, _launch, _require

E4M3 = torch.float8_e4m3fn
BLOCK = 256
_dtype, _shape = attrgetter("dtype"), attrgetter("shape")
_contiguous, _numel = torch.Tensor.is_contiguous, torch.Tensor.numel
_data_ptr, _get_device = torch.Tensor.data_ptr, torch.Tensor.get_device
_increment_version = torch.autograd.graph.increment_version


class _Args(ctypes.Structure):
    _fields_ = [("lr", ctypes.c_double), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double),
                ("eps", ctypes.c_double), ("weight_decay", ctypes.c_double), ("step", ctypes.c_int64),
                ("lr_dev", ctypes.c_void_p), ("step_dev", ctypes.c_void_p), ("grad_scale", ctypes.c_void_p)]


def state_blocks(numel: int) -> int:
    """Scales of an 8-bit state of `numel` elements."""
    return -(-numel // BLOCK)


def _scalar(t, dtype, device, name):
    _require(t.dtype == dtype and t.numel() == 1 and t.device == device,
             f"{name} must be one {str(dtype).removeprefix('torch.')} value on the params' device")
    return t.data_ptr()


def _checked(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, exp_avg_scales, exp_avg_sq_scales,
             copies, grad_scale):
    """The arguments of adamw_step as a call that can be issued, nothing written yet: RuntimeError where the lists do
    not fit.  (None for no tensors.)"""
    n = len(params)
    _require(len(grads) == n and len(exp_avgs) == n and len(exp_avg_sqs) == n,
             "params, grads, exp_avgs and exp_avg_sqs must have the same length")
    if n == 0:
        return None
    dev, pdt, gdt, sdt = params[0].device, params[0].dtype, grads[0].dtype, exp_avgs[0].dtype
    _require(dev.type == "cuda", "params must be on CUDA")
    _require(pdt in _DTYPE_CODE and gdt in _DTYPE_CODE, "params and grads must be fp32, fp16, or bf16")
    _require(sdt in (torch.float32, E4M3), "states must be fp32 or float8_e4m3fn")
    eight = sdt == E4M3
    _require(eight == (exp_avg_scales is not None) and eight == (exp_avg_sq_scales is not None),
             "float8_e4m3fn states need exp_avg_scales and exp_avg_sq_scales, fp32 states take none")
    _require(not eight or (len(exp_avg_scales) == n and len(exp_avg_sq_scales) == n), "one scale tensor per state")
    cdt = None
    if copies is not None:
        _require(len(copies) == n, "one copy per param")
        cdt = copies[0].dtype
        _require(cdt in _DTYPE_CODE, "copies must be fp32, fp16, or bf16")
    # (map over unbound methods: a third of the time of a loop over 96 tensors, which took longer than the kernel)
    if not all(map(_contiguous, grads)):
        grads = [g.contiguous() for g in grads]
    states = [*exp_avgs, *exp_avg_sqs]
    sizes = list(map(_numel, params))
    _require(set(map(_dtype, params)) == {pdt} and set(map(_dtype, grads)) == {gdt} and set(map(_dtype, states)) == {sdt},
             "params, grads and states must each have one dtype")
    given = [*params, *grads, *states]
    _require(list(map(_shape, grads)) == list(map(_shape, params)) and list(map(_numel, states)) == sizes + sizes,
             "grads and states must have their param's shape")
    _require(all(map(_contiguous, params)) and all(map(_contiguous, states)), "params and states must be contiguous")
    pointers = list(map(_data_ptr, given))
    p, g, m, v = (pointers[i * n:(i + 1) * n] for i in range(4))
    ms = vs = cp = [0] * n
    if eight:
        scales = [*exp_avg_scales, *exp_avg_sq_scales]
        blocks = list(map(state_blocks, sizes))
        _require(set(map(_dtype, scales)) == {torch.float32} and all(map(_contiguous, scales))
                 and list(map(_numel, scales)) == blocks + blocks,
                 "scales must be contiguous fp32, one for every 256 elements, on the params' device")
        given += scales
        pointers = list(map(_data_ptr, scales))
        ms, vs = pointers[:n], pointers[n:]
    if cdt is not None:
        _require(set(map(_dtype, copies)) == {cdt} and all(map(_contiguous, copies)) and list(map(_numel, copies)) == sizes,
                 "copies must be contiguous, of one dtype, with their param's size, on its device")
        given += copies
        cp = list(map(_data_ptr, copies))
    _require(set(map(_get_device, given)) == {dev.index}, "all tensors must be on one device")
    written = [q for f in (p, m, v, ms, vs, cp) for q in f if q]
    _require(len(set(written)) == len(written), "the same tensor was given twice")
    # the stk_adamw_tensor of each (as an array of ctypes it took 8 us instead of one)
    table = array("q", chain.from_iterable(zip(p, g, m, v, ms, vs, cp, sizes)))
    a = _Args()
    a.beta1, a.beta2 = betas
    a.eps, a.weight_decay = eps, weight_decay
    if isinstance(lr, torch.Tensor):
        a.lr_dev = _scalar(lr, torch.float32, dev, "lr")
    else:
        a.lr = lr
    if isinstance(step, torch.Tensor):
        a.step_dev = _scalar(step, torch.int64, dev, "step")
    else:
        a.step = step
    if grad_scale is not None:
        a.grad_scale = _scalar(grad_scale, torch.float32, dev, "grad_scale")
    # (grads: a copy made contiguous above is to live until the launch)
    types = _DTYPE_CODE[pdt], _DTYPE_CODE[gdt], -1 if cdt is None else _DTYPE_CODE[cdt], 8 if eight else 32
    return dev, table, n, types, a, params, copies, grads


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
               exp_avg_scales=None, exp_avg_sq_scales=None, copies=None, grad_scale=None):
    """One AdamW step, in place, over lists of CUDA tensors on one device.

    params (fp32, fp16 or bf16, contiguous, one type for all), grads (one type
    for all, same shapes), exp_avgs / exp_avg_sqs (contiguous; fp32 m and v, or
    float8_e4m3fn codes of m and sqrt(v) with their fp32 scales in
    exp_avg_scales / exp_avg_sq_scales, ceil(numel / 256) values a tensor);
    copies: tensors that get the updated params in their own type.  step counts
    from 1.  grad_scale: one fp32 CUDA value that multiplies every gradient
    (clipping, loss scaling) without a host read.  Tensors must not overlap.
    To autograd the step is an operation in place on params and copies (a graph
    that saved them refuses its backward pass); states and their scales, which no
    forward pass reads, count no version.
    """
    _issue(_checked(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, exp_avg_scales,
                    exp_avg_sq_scales, copies, grad_scale))


def _issue(call):
    """Launch what ``_checked`` returned."""
    if call is None:
        return
    dev, table, n, types, args, params, copies, _ = call
    _launch(dev, _capi.load().stk_adamw_step, table.buffer_info()[0], n, *types, ctypes.byref(args))
    # The kernel writes by address: autograd is to notice that tensors which it saved have changed.  (Tensors of
    # inference mode have no version and are passed over there.  With the states and their scales this took 37 instead
    # of 8 us for 96 tensors, on the host, where such a call is bound.)
    _increment_version([*params, *(copies or ())])


class AdamW:
    """AdamW that keeps the states of `params` and steps them from their ``.grad``, or from gradients given to ``step``
    (in the params' order, None for a param that has none; bf16 gradients of fp32 params, say).

    state_bits 32 or 8; copies: {param: tensor} to be written with the updated
    param.  Params without a gradient are passed over, and each counts its own
    steps.  capturable: the step count lives on the GPU and ``step`` advances
    it there, so that a captured ``step`` can be replayed; every param then has
    to have a gradient, and ``lr`` may be a one-element fp32 CUDA tensor.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=32, copies=None,
                 capturable=False):
        self.params = list(params)
        _require(state_bits in (8, 32), "state_bits must be 8 or 32")
        _require(len({id(p) for p in self.params}) == len(self.params), "the same tensor was given twice")
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self.state_bits, self.capturable = state_bits, capturable
        _require(not capturable or len({p.device for p in self.params}) <= 1,
                 "capturable: all params must be on one device, where the step count lives")
        copies = copies or {}
        known = {id(p) for p in self.params}
        _require(all(id(p) in known for p in copies), "copies must be of params of this optimizer")
        self.copies = [copies.get(p) for p in self.params]
        self.state = [self._new_state(p) for p in self.params]
        self.step_dev = (torch.zeros((), dtype=torch.int64, device=self.params[0].device)
                         if capturable and self.params else None)

    def _new_state(self, p):
        dt = E4M3 if self.state_bits == 8 else torch.float32
        s = {"step": 0, "exp_avg": torch.zeros(p.shape, dtype=dt, device=p.device),
             "exp_avg_sq": torch.zeros(p.shape, dtype=dt, device=p.device)}
        if self.state_bits == 8:
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                s[name] = torch.ones(state_blocks(p.numel()), dtype=torch.float32, device=p.device)
        return s

    @torch.no_grad()
    def step(self, grads=None, *, grad_scale=None):
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        _require(len(grads) == len(self.params), "one gradient per param")
        capturing = bool(self.params) and self.params[0].is_cuda and torch.cuda.is_current_stream_capturing()
        _require(self.capturable or not capturing, "capturing a step needs AdamW(capturable=True)")
        _require(not self.capturable or all(g is not None for g in grads), "capturable: every param needs a gradient")
        groups = {}
        for i, p in enumerate(self.params):
            if grads[i] is None:
                continue
            c = self.copies[i]
            key = (p.device, p.dtype, grads[i].dtype, None if c is None else c.dtype, self.state[i]["step"] + 1)
            groups.setdefault(key, []).append(i)
        # All groups are checked before anything is written: a step that is refused has changed nothing.
        calls = []
        for (_, _, _, cdt, t), at in groups.items():
            st = [self.state[i] for i in at]
            eight = self.state_bits == 8
            calls.append(_checked([self.params[i] for i in at], [grads[i] for i in at], [s["exp_avg"] for s in st],
                                  [s["exp_avg_sq"] for s in st], self.step_dev if self.capturable else t, self.lr,
                                  self.betas, self.eps, self.weight_decay,
                                  [s["exp_avg_scale"] for s in st] if eight else None,
                                  [s["exp_avg_sq_scale"] for s in st] if eight else None,
                                  None if cdt is None else [self.copies[i] for i in at], grad_scale))
        if self.capturable and calls:
            dev, _, _, types, args, *_ = calls[0]  # the C entry point's own checks, with no tensors: lr, betas, eps, ...
            _launch(dev, _capi.load().stk_adamw_step, None, 0, *types, ctypes.byref(args))
            self.step_dev.add_(1)
        for call, ((_, _, _, _, t), at) in zip(calls, groups.items()):
            _issue(call)
            if not self.capturable:
                for i in at:
                    self.state[i]["step"] = t

    def zero_grad(self):
        """Drop the gradients (``.grad = None``)."""
        for p in self.params:
            p.grad = None

    def state_dict(self):
        """The states in params' order (their own tensors, not copies) and the step counts."""
        return {"state": [dict(s) for s in self.state], "state_bits": self.state_bits,
                "step": None if self.step_dev is None else self.step_dev}

    def load_state_dict(self, d):
        """Copy the values of ``state_dict()`` of an optimizer with the same params, state_bits and capturable."""
        _require(d["state_bits"] == self.state_bits and len(d["state"]) == len(self.state)
                 and (d["step"] is None) == (self.step_dev is None),
                 "the state is of an optimizer with other params, state_bits or capturable")
        for mine, s in zip(self.state, d["state"]):
            _require(all(s[k].shape == v.shape and s[k].dtype == v.dtype
                         for k, v in mine.items() if isinstance(v, torch.Tensor)), "a state has another shape or dtype")
        for mine, s in zip(self.state, d["state"]):
            for k, v in mine.items():
                if isinstance(v, torch.Tensor):
                    v.copy_(s[k])
                else:
                    mine[k] = s[k]
        if self.step_dev is not None:
            self.step_dev.copy_(d["step"])

"""Argument checks of the training operators' entry points, without a GPU: the
C ABI refuses before it touches a device, and so do the Python functions."""
import ctypes
import math

import pytest
import torch

from streamtopk_sae import _capi, optim


class Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "m", "v", "ms", "vs", "copy")] + [("n", ctypes.c_int64)]


def _adamw(count=1, pdt=_capi.STK_F32, gdt=_capi.STK_F32, cdt=-1, bits=32, null_args=False, n=8, ptr=4096, **kw):
    lib = _capi.load()
    a = optim._Args(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, step=1)
    for k, v in kw.items():
        setattr(a, k, v)
    t = (Tensor * max(count, 1))()
    for x in t:
        x.param = x.grad = x.m = x.v = ptr
        x.n = n
    rc = lib.stk_adamw_step(t, count, pdt, gdt, cdt, bits, None if null_args else ctypes.byref(a), None)
    return rc, lib.stk_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(pdt=9), "fp32, fp16 or bf16"), (dict(gdt=_capi.STK_E4M3), "fp32, fp16 or bf16"),
    (dict(cdt=7), "fp32, fp16 or bf16"), (dict(bits=16), "8 or 32"), (dict(null_args=True), "need args"),
    (dict(count=-1), "need args"), (dict(beta1=1.0), "betas"), (dict(beta2=-0.1), "betas"),
    (dict(beta2=math.nan), "betas"), (dict(eps=-1.0), "eps"), (dict(lr=math.nan), "lr must"),
    (dict(weight_decay=-1.0), "weight_decay"), (dict(step=0), "step must"), (dict(n=-1), "out of range"),
    (dict(ptr=None), "null tensor"), (dict(ptr=4097), "not aligned"), (dict(bits=8), "null tensor"),
    (dict(cdt=_capi.STK_BF16), "null tensor")])
def test_adamw_refusals(kw, msg):
    rc, said = _adamw(**kw)
    assert rc == _capi.STK_EINVAL and msg in said


def test_adamw_nothing_to_do():
    assert _adamw(count=0)[0] == _capi.STK_OK
    assert _adamw(n=0, ptr=None)[0] == _capi.STK_OK
    assert optim.adamw_step([], [], [], [], step=1, lr=0.1) is None


def test_adamw_python_refusals():
    x = torch.zeros(4)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        optim.adamw_step([x], [x], [x], [x], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="same length"):
        optim.adamw_step([x], [], [x], [x], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="8 or 32"):
        optim.AdamW([x], state_bits=16)
    with pytest.raises(RuntimeError, match="given twice"):
        optim.AdamW([x, x])

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
    (dict(beta2=math.nan), "betas"), (dict(eps=-1.0), "eps"), (dict(eps=1e-40), "eps"), (dict(lr=math.nan), "lr must"),
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


def _route(dtype=_capi.STK_F32, ld=64, N=4, E=64, k=2, score=0, G=1, top=1, scale=1.0, ptr=4096, out=4096):
    lib = _capi.load()
    rc = lib.stk_route_forward(ptr, dtype, ld, None, None, out, out, None, N, E, k, score, G, top, 1, scale, None)
    return rc, lib.stk_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=_capi.STK_E4M3), "logits must be"), (dict(score=2), "unknown score"), (dict(N=-1), "need N"),
    (dict(E=0), "need N"), (dict(E=1025, ld=1025), "need N"), (dict(k=0), "need 1 <= k"), (dict(k=33), "need 1 <= k"),
    (dict(E=2, k=3), "need 1 <= k"), (dict(ld=63), "row stride"), (dict(scale=math.nan), "scale must"),
    (dict(G=0), "n_groups"), (dict(G=7), "n_groups"), (dict(G=64), "n_groups"), (dict(G=8, top=9), "n_groups"),
    (dict(G=32, top=1, k=3), "k exceeds"), (dict(ptr=None), "null"), (dict(out=None), "null"),
    (dict(ptr=4098), "not aligned"), (dict(out=4098), "not aligned")])
def test_route_refusals(kw, msg):
    rc, said = _route(**kw)
    assert rc == _capi.STK_EINVAL and msg in said


def test_route_backward_refusals():
    lib = _capi.load()

    def call(gw=4096, x=4096, e=4096, out=4096, dtype=_capi.STK_BF16, N=4, k=2):
        return lib.stk_route_backward(gw, x, dtype, 64, e, out, N, 64, k, 0, 1, 1.0, None)

    assert call(N=0) == _capi.STK_OK
    for kw in (dict(gw=None), dict(x=None), dict(e=None), dict(out=None), dict(dtype=9), dict(k=65), dict(gw=4098),
               dict(out=4097)):
        assert call(**kw) == _capi.STK_EINVAL
    assert "stk_route_backward" in lib.stk_last_error().decode()


def test_routing_python_refusals():
    import streamtopk_sae as stk
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        stk.route_experts(torch.zeros(2, 4), 1)
    with pytest.raises(RuntimeError, match=r"W_enc must be \(E, Fe, d\)"):
        stk.topk_sae_routed_encode(torch.zeros(2, 4), torch.zeros(2, 3), torch.zeros(3, 5), torch.zeros(3, 5), 1)


def _sae(dec=True, enc=True, B=4, k=2, F=10, d=8, dtype=_capi.STK_BF16, ws=None, n=0, **kw):
    lib = _capi.load()
    p = 4096
    a = dict(g=p if dec else None, X=p if enc else None, We=None, Wd=p if dec else None, V=p if dec else None, I=p,
             gv=None if dec else p, dWe=p if enc else None, dbe=p if enc else None, dWd=p if dec else None,
             dbd=p if dec else None, dv=p if dec else None, dX=None)
    a.update(kw)
    rc = lib.stk_sae_backward(*a.values(), B, k, F, d, dtype, ws, n, None)
    return rc, lib.stk_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=_capi.STK_E4M3), "fp32, fp16, or bf16"), (dict(B=-1), "need B"), (dict(k=0), "need B"),
    (dict(F=0), "need B"), (dict(d=0), "need B"), (dict(F=2 ** 31), "need B"), (dict(B=2 ** 20, k=2 ** 20), "need B"),
    (dict(dec=False, enc=False), "one of dW_enc and dW_dec"), (dict(dbe=None), "go together"),
    (dict(dec=False, dv=4096), "need dW_dec"), (dict(enc=False, dX=4096), "dX needs dW_enc"),
    (dict(I=None), "null"), (dict(g=None), "null"), (dict(Wd=None), "null"), (dict(V=None), "null"),
    (dict(X=None), "null"), (dict(dec=False, gv=None), "null"), (dict(dX=4096), "null"),
    (dict(dX=4096, We=4096, dv=None), "null"), (dict(X=4097), "not aligned"), (dict(dv=4098), "not aligned")])
def test_sae_backward_refusals(kw, msg):
    rc, said = _sae(**kw)
    assert rc == _capi.STK_EINVAL and msg in said


def test_sae_backward_workspace():
    rc, said = _sae()
    assert rc == _capi.STK_ENOSPACE and "workspace" in said
    need = _capi.sae_backward_workspace_bytes(4, 2, 10, 8)
    assert _sae(ws=4096, n=need - 1)[0] == _capi.STK_ENOSPACE
    assert _sae(ws=4112, n=need)[0] == _capi.STK_EINVAL
    # grows with the codes, holds sorted codes and the parts of long lists
    big = _capi.sae_backward_workspace_bytes(4096, 64, 65536, 2048)
    N = 4096 * 64
    assert big >= 4 * 4 * N + 4 * 65537 + 2 * (N // 256) * 2 * 4 * 2048
    with pytest.raises(RuntimeError, match="need B"):
        _capi.sae_backward_workspace_bytes(1, 0, 1, 1)


def test_sae_backward_python_refusals():
    import streamtopk_sae as stk
    x = torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        stk.topk_sae_backward(x, x, x, x, x, x.int())
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        stk.topk_sae_encode_backward(x, x.int(), x, x)
    with pytest.raises(RuntimeError, match="contiguous fp32"):
        stk.TopkSAETrainer(x.half(), x, x, x, 1)

"""Arguments at the ends of what the training operators' arithmetic holds, without a GPU."""
import ctypes
import math

import pytest
import torch

from streamtopk_sae import _capi, optim


@pytest.mark.parametrize("eps,ok", [(0.0, True), (2.0 ** -126, True), (1e-8, True), (1.0, True), (2.0 ** 125, True),
                                    (2.0 ** 126, False), (1e300, False), (math.inf, False), (math.nan, False)])
def test_adamw_eps(eps, ok):
    """The update divides by root + eps with a reciprocal that has to be a normal fp32 value."""
    lib = _capi.load()
    a = optim._Args(lr=1e-3, beta1=0.9, beta2=0.99, eps=eps, weight_decay=0.0, step=1)
    rc = lib.stk_adamw_step(None, 0, _capi.STK_F32, _capi.STK_F32, -1, 32, ctypes.byref(a), None)
    assert rc == (_capi.STK_OK if ok else _capi.STK_EINVAL)
    if not ok:
        assert "eps" in lib.stk_last_error().decode()


def test_routed_encode_of_more_features_than_int32_counts():
    import streamtopk_sae as stk
    W = torch.zeros(1, 1, 8).expand(2, 2 ** 30, 8)
    b = torch.zeros(1, 1).expand(2, 2 ** 30)
    with pytest.raises(RuntimeError, match=r"E \* Fe"):
        stk.topk_sae_routed_encode(torch.zeros(3, 8), torch.zeros(3, 2), W, b, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        stk.topk_sae_routed_encode(torch.zeros(3, 8), torch.zeros(3, 2), W[:, :-1], b[:, :-1], 4)

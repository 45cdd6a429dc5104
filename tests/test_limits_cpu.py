"""Arguments at the ends of what the training operators' arithmetic holds, without a GPU."""
import ctypes
import math

import pytest

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

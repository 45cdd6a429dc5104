"""Indices of codes given as int64: those that no int32 holds are passed over like all outside [0, F), not taken modulo 2^32."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FAR = [2 ** 32 + 3, -2 ** 32 + 3, 2 ** 31, 2 ** 63 - 1, -2 ** 63, -2 ** 31 - 1, 2 ** 40]


def codes(B=9, d=32, F=20, k=8):
    r = torch.Generator(device="cuda").manual_seed(3)
    X, g = (torch.randn(B, d, generator=r, device="cuda") for _ in range(2))
    W_enc, W_dec = (torch.randn(F, d, generator=r, device="cuda") for _ in range(2))
    vals = torch.randn(B, k, generator=r, device="cuda")
    idxs = torch.randint(0, F, (B, k), generator=r, device="cuda")
    near = idxs.clone()
    for n, far in enumerate(FAR):
        idxs[n, n], near[n, n] = far, -1
    return X, g, W_enc, W_dec, vals, idxs, near.int()


def test_decode():
    import streamtopk_sae as stk
    _, _, _, W_dec, vals, idxs, near = codes()
    assert torch.equal(stk.topk_sae_decode(vals, idxs, W_dec), stk.topk_sae_decode(vals, near, W_dec))


def test_gradients():
    import streamtopk_sae as stk
    X, g, W_enc, W_dec, vals, idxs, near = codes()
    pairs = [[stk.topk_sae_backward(g, X, W_enc, W_dec, vals, i, need_dx=True) for i in (idxs, near)],
             [stk.topk_sae_decode_backward(g, vals, i, W_dec) for i in (idxs, near)],
             [stk.topk_sae_encode_backward(vals, i, X, W_enc) for i in (idxs, near)]]
    for a, b in pairs:
        for x, y in zip(a, b):
            assert torch.equal(x, y)

"""The SAE's gradient where its plan is another: parts of 128 and 256 codes, three radix passes, wide rows.

Tolerances as in test_sae_backward_gpu, of chains of at most 256 codes and of at most n / 128 of them (parts are of 128 or
256 codes here): (256 + n / 128 + 2) u of the sum of the magnitudes, dvals (16 + d / 64) u, half a step of 16 bits.
"""
import pytest
import torch
from test_sae_backward_gpu import U, check, check_all, gen, make, want

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def dense(at, v, F):
    return torch.zeros(at.shape[0], F, dtype=torch.float64, device=at.device).scatter_add_(1, at, v)


@pytest.mark.parametrize("B,dtype", [(8192, torch.bfloat16), (16384, torch.float32)])
def test_few_features_and_many_codes(B, dtype):
    """2 * N / part * d above 2^25: parts of 128 (B=8192) and of 256 codes, beside lists of 1, 8, 9, 255, 256, 257 codes."""
    import streamtopk_sae as stk
    d, k, F = 4096, 64, 70
    r = gen(B)
    X, g = (torch.randn(B, d, generator=r, device="cuda") for _ in range(2))
    X = X.to(dtype)
    W_enc, W_dec = ((torch.randn(F, d, generator=r, device="cuda") * d ** -0.5).to(dtype) for _ in range(2))
    vals = torch.randn(B, k, generator=r, device="cuda")
    idxs = torch.randint(0, 64, (B, k), generator=r, device="cuda", dtype=torch.int32)
    place = torch.randperm(B * k, generator=r, device="cuda")
    used = 0
    for f, n in zip(range(64, 70), (1, 8, 9, 255, 256, 257)):
        idxs.view(-1)[place[used:used + n]] = f
        used += n
    idxs.view(-1)[place[used:used + 1000]] = -1
    out = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    live, at = idxs >= 0, idxs.clamp_min(0).long()
    g64, x64, we, wd = (t.double() for t in (g, X, W_enc, W_dec))
    v = torch.where(live, vals.double(), 0.0)
    dv = torch.where(live, (g64 @ wd.T).gather(1, at), 0.0)
    ev = torch.where(live, (g64.abs() @ wd.abs().T).gather(1, at), 0.0) * (16 + d / 64) * U
    n = torch.bincount(at[live], minlength=F).double()
    assert n[64:].tolist() == [1, 8, 9, 255, 256, 257]
    chain = ((n.clamp(max=256) + n / 128 + 2) * U)[:, None]
    check(out.vals, dv, ev)
    check(out.W_dec, dense(at, v, F).T @ g64, chain * (dense(at, v.abs(), F).T @ g64.abs()))
    codes, most, off = dense(at, dv, F), dense(at, dv.abs(), F), dense(at, ev, F)
    check(out.W_enc, codes.T @ x64, chain * ((most + off).T @ x64.abs()) + off.T @ x64.abs())
    check(out.b_enc, codes.sum(0), chain[:, 0] * (most + off).sum(0) + off.sum(0))
    check(out.b_dec, g64.sum(0), B * U * g64.abs().sum(0))
    check(out.X, codes @ we, (most * (k + 2) * U + off) @ we.abs())
    again = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    for a, b in zip(out, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B,d,F,k,hot,dtype", [
    (300, 8, 5_000_000, 40, 0.1, torch.float32), (300, 8, 4_194_304, 40, 0, torch.bfloat16),  # 23 bits of key: three passes
    (5, 70001, 40, 3, 0, torch.float32), (2101, 20008, 30, 4, 0.2, torch.bfloat16), (2101, 5001, 30, 4, 0.2, torch.float16)])
def test_many_features_and_wide_rows(B, d, F, k, hot, dtype):
    import streamtopk_sae as stk
    t = make(B, d, F, k, dtype, seed=B + d, hot=hot, invalid=True)
    X, W_enc, W_dec, vals, idxs, g = t
    idxs[1, 0], idxs[1, 1] = 0, F - 1
    check_all(stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True), want(*t))

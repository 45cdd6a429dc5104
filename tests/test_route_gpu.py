"""The router (stk_route_forward / stk_route_backward) against plain 64-bit
forms of its definition: the chosen experts have to be equal, ties included.

Tolerances, u = 2^-24: a weight is a ratio of fp32 exponentials (two units in
the last place each, and the rounding of x - top, which adds at most |x - top|
u), a sum of at most E of them (log2 32 + E / 32 roundings), a division and the
scale: within (16 + E / 32 + max |x - top|) u of its value for softmax.  A
gradient is a sum of k products of such values: within the same times the sum
of the magnitudes of its terms, and half a step of its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def scores64(logits, score):
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    if score == "sigmoid":
        return x, torch.sigmoid(x)
    top = x.amax(1, keepdim=True)
    e = torch.where(x == top, 1.0, torch.exp(x - top))
    e = torch.where(x == -math.inf, 0.0, e)
    return x, e / e.sum(1, keepdim=True).clamp_min(1e-300)


def plain(logits, k, score="softmax", bias=None, n_groups=1, topk_groups=1, renormalize=True, scale=1.0, row_mask=None):
    """(weights in 64 bits, experts) row by row, pick by pick."""
    x, s = scores64(logits, score)
    x, s = x.cpu(), s.cpu()
    b = None if bias is None else bias.double().cpu()
    N, E = x.shape
    per = E // n_groups
    experts = torch.full((N, k), -1, dtype=torch.int32)
    for n in range(N):
        if row_mask is not None and not bool(row_mask[n]):
            continue
        choice = x[n].clone() if b is None else torch.where(x[n] > -math.inf, s[n] + b, -math.inf)
        choice = torch.where(choice.isnan(), -math.inf, choice)
        each = torch.where(choice > -math.inf, s[n] if b is None else choice, -math.inf)
        if topk_groups < n_groups:
            total = []
            for g in range(n_groups):
                best = sorted((v for v in each[g * per:(g + 1) * per].tolist() if v > -math.inf), reverse=True)[:2]
                total.append(sum(best) if best else -math.inf)
            kept = sorted(range(n_groups), key=lambda g: (-total[g], g))[:topk_groups]
            for g in range(n_groups):
                if g not in kept:
                    choice[g * per:(g + 1) * per] = -math.inf
        c = choice.tolist()
        order = sorted((e for e in range(E) if c[e] > -math.inf), key=lambda e: (-c[e], e))[:k]
        experts[n, : len(order)] = torch.tensor(order, dtype=torch.int32)
    live = experts >= 0
    w = torch.where(live, s.gather(1, experts.clamp_min(0).long()), 0.0)
    if renormalize:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300 if score == "softmax" else 1e-20)
    return scale * w, experts


def close(weights, want, logits, score):
    E = logits.shape[1]
    x = logits.double()
    x = torch.where(x.isfinite(), x, 0.0)
    span = float((x.amax(1) - x.amin(1)).max()) if score == "softmax" else float(x.abs().max())
    tol = (16 + E / 32 + 2 * span) * U
    assert torch.all((weights.cpu().double() - want).abs() <= tol * want + 1e-37)


def run(logits, k, **kw):
    import streamtopk_sae as stk
    w, e, c = stk.route_experts(logits, k, return_counts=True, **kw)
    torch.cuda.synchronize()
    assert w.dtype == torch.float32 and e.dtype == torch.int32 and c.dtype == torch.int32
    want = torch.bincount(e[e >= 0].long(), minlength=logits.shape[1])
    assert torch.equal(c.long(), want)
    return w, e


def both(logits, k, **kw):
    w, e = run(logits, k, **kw)
    pw, pe = plain(logits, k, **kw)
    assert torch.equal(e.cpu(), pe)
    close(w, pw, logits, kw.get("score", "softmax"))
    return w, e


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("N,E,k,dtype", [
    (1, 1, 1, torch.float32), (1, 8, 3, torch.bfloat16), (37, 32, 32, torch.float16), (130, 33, 5, torch.float32),
    (64, 64, 4, torch.bfloat16), (50, 100, 2, torch.float32), (40, 256, 8, torch.float32), (9, 1000, 32, torch.float16),
    (5, 1024, 1, torch.float32)])
def test_matches_plain(score, renormalize, N, E, k, dtype):
    both(randn(N, E, seed=E + k, dtype=dtype) * 2, k, score=score, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,k", [(2, 2), (8, 4), (8, 8), (13, 5), (16, 2), (30, 7), (32, 8), (33, 4), (60, 6), (128, 3),
                                 (200, 8), (256, 4), (256, 9), (300, 4)])
def test_16_bit_picks(E, k, dtype):
    """Few picks of 16-bit logits are merged from sorted lists: ties, masked experts, rows that are partly empty."""
    x = (randn(67, E, seed=E + k) * 3).to(dtype)
    x[5:20] = (x[5:20].float() / 2).round().to(dtype)          # many equal logits, zeros of both signs
    x[20:30, ::3] = -math.inf
    x[30, 1:] = -math.inf
    x[31, :] = math.nan
    x[32, E // 2] = math.nan
    x[33, E - 1] = math.inf
    mask = torch.ones(67, dtype=torch.bool, device="cuda")
    mask[60:] = False
    for renormalize in (True, False):
        run_and_compare = dict(renormalize=renormalize, row_mask=mask)
        w, e = run(x, k, **run_and_compare)
        pw, pe = plain(x, k, **run_and_compare)
        assert torch.equal(e.cpu(), pe)
        # logits within 15 of one another: (16 + E / 32 + 2 * 30) u
        assert torch.all((w.cpu().double() - pw).abs() <= (76 + E / 32) * U * pw + 1e-37)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,G,top,use_bias,dtype", [
    (64, 6, 1, 1, True, torch.bfloat16), (256, 8, 8, 4, True, torch.float32), (256, 8, 8, 4, False, torch.bfloat16),
    (160, 6, 8, 3, False, torch.float32), (60, 4, 20, 7, True, torch.float16), (32, 3, 32, 5, True, torch.float32),
    (24, 3, 8, 1, False, torch.float32), (512, 16, 4, 4, True, torch.float32)])
def test_bias_and_groups_match_plain(score, E, k, G, top, use_bias, dtype):
    both(randn(120, E, seed=E, dtype=dtype), k, score=score, bias=randn(E, seed=1) * 0.1 if use_bias else None,
         n_groups=G, topk_groups=top)


@pytest.mark.parametrize("N", [200, 4100])
def test_large_biases_that_cancel_in_a_group(N):
    """Group totals whose two terms are far larger than they are, and nearly equal from group to group."""
    E, G = 64, 4
    logits = randn(N, E, seed=50) * 1e-3
    bias = torch.full((E,), -1000.0, device="cuda")
    bias[0::16], bias[1::16] = 500.0, -499.5
    for sign in (1, -1):
        b = bias + sign * torch.rand(E, generator=torch.Generator(device="cuda").manual_seed(51), device="cuda") * 1e-3
        w, e = run(logits, 3, score="sigmoid", bias=b, n_groups=G, topk_groups=2)
        at = torch.arange(0, N, max(1, N // 200), device="cuda")
        pw, pe = plain(logits[at], 3, score="sigmoid", bias=b, n_groups=G, topk_groups=2)
        assert torch.equal(e[at].cpu(), pe)
        close(w[at], pw, logits[at], "sigmoid")


@pytest.mark.parametrize("E,k,G,top,dtype", [(40, 32, 1, 1, torch.float32), (64, 4, 4, 2, torch.bfloat16),
                                             (128, 8, 8, 4, torch.float32), (100, 5, 1, 1, torch.float16),
                                             (256, 8, 8, 4, torch.float32), (200, 6, 1, 1, torch.bfloat16)])
def test_many_rows_with_bias(E, k, G, top, dtype):
    """Sixteen experts a lane (from 4096 rows on): the choices of a sample of rows, and those of every row against a
    call with few rows, whose lanes hold eight."""
    import streamtopk_sae as stk
    logits = randn(4100, E, seed=E, dtype=dtype)
    logits[:200] = (logits[:200].float() * 2).round().to(dtype)    # ties
    logits[200:220, ::2] = -math.inf
    bias = randn(E, seed=1) * 0.05
    bias[::7] = 0.25
    for score in ("softmax", "sigmoid"):
        how = dict(score=score, bias=bias, n_groups=G, topk_groups=top)
        w, e = run(logits, k, **how)
        sample = torch.arange(0, 4100, 37, device="cuda")
        pw, pe = plain(logits[sample], k, **how)
        assert torch.equal(e[sample].cpu(), pe)
        close(w[sample], pw, logits[sample], score)
        for n in range(0, 4100, 1025):
            ww, ee = stk.route_experts(logits[n:n + 1025], k, **how)
            assert torch.equal(e[n:n + 1025], ee)


@pytest.mark.parametrize("N", [300, 4200])
@pytest.mark.parametrize("spread", [0.0, 3e-7, 3e-6])
def test_choice_is_that_of_64_bits(N, spread):
    """Choices that differ by less than fp32 can tell, or by a few of its steps: s + bias equal to within 2^-30 or so,
    or spread over `spread`; with 8 and with 16 experts a lane."""
    E, k = 64, 8
    logits = randn(N, E, seed=3)
    s = torch.sigmoid(logits[0].double())
    # rows 0 .. 200: every choice 0.7 to within fp32 and the spread
    bias = (0.7 + spread * torch.rand(E, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") - s).float()
    logits[1:200] = logits[0] + randn(199, 1, seed=4) * 1e-6
    logits[200:230] = logits[0]
    logits[200:230, ::2] -= 1e-6
    for kw in ({}, {"n_groups": 8, "topk_groups": 3}, {"n_groups": 4, "topk_groups": 2}):
        w, e = run(logits, k, score="sigmoid", bias=bias, **kw)
        at = torch.cat([torch.arange(230), torch.arange(230, N, 50)]).cuda()
        pw, pe = plain(logits[at], k, score="sigmoid", bias=bias, **kw)
        assert torch.equal(e[at].cpu(), pe)
        close(w[at], pw, logits[at], "sigmoid")
        if not kw:
            assert len({tuple(r) for r in e[:200].tolist()}) > 1


@pytest.mark.parametrize("kw", [{}, {"bias": True}, {"n_groups": 8, "topk_groups": 3}, {"score": "sigmoid", "bias": True}])
def test_ties_go_to_the_lower_index(kw):
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.zeros(64, device="cuda")
    flat = torch.zeros(5, 64, device="cuda")
    _, e = both(flat, 6, **kw)
    assert torch.equal(e.cpu(), torch.arange(6, dtype=torch.int32).expand(5, 6))
    coarse = (randn(200, 64, seed=9) * 2).round().to(torch.bfloat16)   # many equal logits
    both(coarse, 8, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("use_bias,G,top", [(False, 1, 1), (True, 1, 1), (True, 4, 2), (False, 4, 2)])
def test_masked_experts_rows_and_infinities(score, use_bias, G, top):
    N, E, k = 40, 48, 6
    logits = randn(N, E, seed=2)
    logits[0] = -math.inf                          # nothing left
    logits[1] = math.nan
    logits[2, 3:] = -math.inf                      # fewer than k
    logits[3, ::2] = math.nan
    logits[4, 7] = math.inf
    logits[5, 7] = logits[5, 20] = math.inf
    logits[6] = torch.finfo(torch.float32).min     # the type's lowest value is a logit like any other
    logits[7, :40] = torch.finfo(torch.float32).min
    logits[8, 13:] = -math.inf
    bias = None
    if use_bias:
        bias = randn(E, seed=5) * 0.05
        bias[11], bias[12], bias[30] = -math.inf, math.nan, math.inf
    mask = torch.ones(N, dtype=torch.bool, device="cuda")
    mask[30:] = False
    logits[31] = math.nan
    w, e = run(logits, k, score=score, bias=bias, n_groups=G, topk_groups=top, row_mask=mask)
    pw, pe = plain(logits, k, score=score, bias=bias, n_groups=G, topk_groups=top, row_mask=mask)
    assert torch.equal(e.cpu(), pe)
    # the lowest fp32 values make spans beyond exp's range, where a score is 0 or 1
    assert torch.all((w.cpu().double() - pw).abs() <= 64 * U * pw + 1e-37)
    assert torch.all(e[30:] == -1) and torch.all(w[30:] == 0) and torch.all(e[:2] == -1) and torch.all(w[:2] == 0)


def test_strided_logits_no_rows_and_other_stream():
    import streamtopk_sae as stk
    wide = randn(70, 100, seed=6)
    a = both(wide[:, 10:74], 4)
    b = both(wide.T.contiguous().T[:, 10:74], 4)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    both(wide[:1].expand(30, 100), 4)
    w, e, c = stk.route_experts(wide[:0], 4, return_counts=True)
    assert w.shape == (0, 4) and e.shape == (0, 4) and not c.any()
    assert stk.route_experts_backward(w, wide[:0], e).shape == (0, 100)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        w, e = stk.route_experts(wide[:, 10:74], 4)
    s.synchronize()
    assert torch.equal(w, a[0]) and torch.equal(e, a[1])


def test_many_rows_each_counted():
    logits = randn(20011, 70, seed=8, dtype=torch.bfloat16)
    w, e = run(logits, 3)
    x, s = scores64(logits, "softmax")
    order = x.sort(dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(e.long(), order)


def grad64(gw, logits, experts, score, renormalize, scale):
    """By differentiating the formula in 64 bits."""
    x, _ = scores64(logits, score)
    leaf = x.clone().requires_grad_()
    live = experts >= 0
    if score == "sigmoid":
        s = torch.sigmoid(leaf)
    else:
        s = torch.softmax(leaf, 1)
    s = torch.where(live, s.gather(1, experts.clamp_min(0).long()), 0.0)
    if renormalize:
        s = s / s.sum(1, keepdim=True).clamp_min(1e-300 if score == "softmax" else 1e-20)
    (torch.where(live, scale * s, 0.0) * gw.double()).sum().backward()
    return torch.where(live.any(1, keepdim=True), leaf.grad.nan_to_num(0.0), 0.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("N,E,k,dtype", [
    (1, 1, 1, torch.float32), (1, 8, 3, torch.bfloat16), (37, 32, 32, torch.float16), (130, 33, 5, torch.float32),
    (300, 128, 1, torch.float32), (40, 256, 8, torch.bfloat16), (9, 1000, 32, torch.float32)])
def test_backward_matches_differentiation(score, renormalize, N, E, k, dtype):
    import streamtopk_sae as stk
    logits = randn(N, E, seed=E + k, dtype=dtype) * 2
    if N > 20:
        logits[3, 2:] = -math.inf
        logits[4] = -math.inf
        logits[5, 0] = 30.0                          # nearly certain: 1 - s must not cancel
    how = dict(score=score, renormalize=renormalize, scale=1.5)
    mask = torch.arange(N, device="cuda") < max(1, N - N // 10)
    _, experts = stk.route_experts(logits, k, row_mask=mask, **how)
    gw = randn(N, k, seed=1)
    got = stk.route_experts_backward(gw, logits, experts, **how)
    want = grad64(gw, logits, experts, **how)
    assert got.dtype == dtype and got.shape == (N, E)
    # magnitudes of the terms: |g| s_e for each, and s_e times the chosen ones' |g| s
    _, s = scores64(logits, score)
    live = experts >= 0
    sk = torch.where(live, s.gather(1, experts.clamp_min(0).long()), 0.0)
    norm = sk.sum(1, keepdim=True).clamp_min(1e-20) if renormalize else 1.0
    p = sk / norm
    g = torch.where(live, 1.5 * gw.double(), 0.0)
    own = torch.zeros_like(s).scatter_add_(1, experts.clamp_min(0).long(), g.abs() * (1 if not renormalize else 1 / norm))
    terms = s * (own + (g.abs() * p).sum(1, keepdim=True) / norm)
    span = float(torch.where(logits.isfinite(), logits.float(), 0.0).abs().max()) * 2
    tol = 4 * (16 + E / 32 + 2 * span + k) * U * terms
    half = torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * 2.0 ** -10
    assert torch.all((got.double() - want).abs() <= tol + half)
    assert torch.all(got[~live.any(1)] == 0)


def test_backward_of_a_certain_choice_keeps_its_digits():
    """s near 1: the gradient s (1 - s) g must be right relative to itself, not to g."""
    import streamtopk_sae as stk
    logits = torch.zeros(1, 4, device="cuda")
    logits[0, 1] = 20.0
    gw = torch.ones(1, 1, device="cuda")
    for score in ("softmax", "sigmoid"):
        w, e = stk.route_experts(logits, 1, score=score, renormalize=False)
        got = stk.route_experts_backward(gw, logits, e, score=score, renormalize=False)
        want = grad64(gw, logits, e, score, False, 1.0)
        assert torch.all((got.double() - want).abs() <= 200 * U * want.abs())


@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_backward_matches_differences(score, renormalize):
    """Central differences of the plain 64-bit weights at fixed experts."""
    import streamtopk_sae as stk
    logits = randn(3, 12, seed=21)
    how = dict(score=score, renormalize=renormalize, scale=1.0)
    _, experts = stk.route_experts(logits, 4, **how)
    gw = randn(3, 4, seed=22)
    got = stk.route_experts_backward(gw, logits, experts, **how).double()

    def loss(x):
        s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, 1)
        s = s.gather(1, experts.long())
        return ((s / s.sum(1, keepdim=True) if renormalize else s) * gw.double()).sum(1)

    h = 1e-5
    for e in range(12):
        d = torch.zeros(3, 12, dtype=torch.float64, device="cuda")
        d[:, e] = h
        diff = (loss(logits.double() + d) - loss(logits.double() - d)) / (2 * h)
        # differences are good to h^2 = 1e-10, the kernel to some 40 u of terms below |gw|
        assert torch.all((got[:, e] - diff).abs() <= 64 * U * gw.abs().sum(1) + 1e-9)


def test_captured_and_replayed():
    import streamtopk_sae as stk
    logits = randn(64, 64, seed=30)
    bias = randn(64, seed=31) * 0.1
    stk.route_experts(logits, 4, bias=bias, return_counts=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, e, c = stk.route_experts(logits, 4, bias=bias, return_counts=True)
    for seed in (32, 33):
        logits.copy_(randn(64, 64, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        ww, ee, cc = stk.route_experts(logits, 4, bias=bias, return_counts=True)
        assert torch.equal(w, ww) and torch.equal(e, ee) and torch.equal(c, cc)


def test_routed_encode_matches_each_dictionary():
    import streamtopk_sae as stk
    E, Fe, d, B, k, m = 5, 700, 64, 90, 8, 2
    X, W, b = stk.make_inputs(B, d, E * Fe, dtype=torch.bfloat16, seed=4, device="cuda")
    W, b = W.view(E, Fe, d), b.view(E, Fe)
    logits = randn(B, E, seed=41)
    mask = torch.arange(B, device="cuda") < 80
    vals, idxs, weights, experts = stk.topk_sae_routed_encode(X, logits, W, b, k, m, row_mask=mask)
    w, e = stk.route_experts(logits, m, row_mask=mask)
    assert torch.equal(weights, w) and torch.equal(experts, e)
    assert torch.all(idxs[80:] == -1) and torch.all(vals[80:] == 0)
    for n in range(0, 80, 7):
        for j in range(m):
            at = int(e[n, j])
            v, i = stk.topk_sae_cuda_exact(X[n:n + 1], W[at], b[at], k)
            assert torch.equal(idxs[n, j * k:(j + 1) * k], i[0] + at * Fe)
            # the same scores from another tiling of the batch: fp32 sums of d terms
            assert torch.all((vals[n, j * k:(j + 1) * k] - v[0]).abs() <= 2 * d * U * v[0].abs().max())


def test_refusals():
    import streamtopk_sae as stk
    x = randn(4, 64)
    for kw, msg in ((dict(k=0), "k out of range"), (dict(k=33), "k out of range"),
                    (dict(k=9, n_groups=8, topk_groups=1), "k out of range"),
                    (dict(k=1, n_groups=7), "multiple of n_groups"), (dict(k=1, n_groups=64, topk_groups=1), "n_groups"),
                    (dict(k=1, score="tanh"), "score must be"), (dict(k=1, bias=randn(63)), "bias must be"),
                    (dict(k=1, row_mask=torch.ones(4, device="cuda")), "row_mask must be"),
                    (dict(k=1, scale=math.inf), "scale must be finite")):
        with pytest.raises(RuntimeError, match=msg):
            stk.route_experts(x, **kw)
    with pytest.raises(RuntimeError, match="1024"):
        stk.route_experts(randn(2, 1025), 1)
    with pytest.raises(RuntimeError, match="fp32, fp16 or bf16"):
        stk.route_experts(x.double(), 1)
    w, e = stk.route_experts(x, 2)
    with pytest.raises(RuntimeError, match="int32"):
        stk.route_experts_backward(w, x, e.long())
    with pytest.raises(RuntimeError, match=r"\(N, k\)"):
        stk.route_experts_backward(w[:2], x, e)

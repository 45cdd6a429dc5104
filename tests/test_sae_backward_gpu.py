"""The SAE's gradient (stk_sae_backward) against its formulas in 64 bits.

Tolerances, u = 2^-24, from the roundings that a sum of products can meet in
the orders the kernel may take:  dvals sums d products, in 64 chains of fused
multiply-adds (d / 64 each) that a warp adds in 6 steps, or with those steps for
every 256 columns (4 + 6 + d / 256): within (16 + d / 64) u of the sum of the
magnitudes.  dW sums a feature's n codes in
chains of at most 256 and then over the chains: (min(n, 256) + n / 256 + 2) u,
and dW_enc, db_enc and dX carry the error of dvals.  Column sums of g: B u / 8
at most in a row, loosely B u.  Gradients in 16 bits add half a step of theirs.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(B, d, F, k, dtype, seed=0, hot=0.0, invalid=False):
    """X, W_enc, W_dec, vals, idxs, g; `hot`: share of codes that go to one feature."""
    r = gen(seed)
    X = torch.randn(B, d, generator=r, device="cuda").to(dtype)
    W_enc = (torch.randn(F, d, generator=r, device="cuda") * d ** -0.5).to(dtype)
    W_dec = (torch.randn(F, d, generator=r, device="cuda") * d ** -0.5).to(dtype)
    vals = torch.randn(B, k, generator=r, device="cuda")
    idxs = torch.randint(0, F, (B, k), generator=r, device="cuda", dtype=torch.int32)
    if hot:
        idxs[torch.rand(B, k, generator=r, device="cuda") < hot] = F // 2
    if invalid:
        idxs[B // 2, :] = -1
        idxs[0, 0] = -7
        idxs[B - 1, k - 1] = F
        idxs[B - 1, 0] = 2 ** 31 - 1
    g = torch.randn(B, d, generator=r, device="cuda")
    return X, W_enc, W_dec, vals, idxs, g


def want(X, W_enc, W_dec, vals, idxs, g, gv=None):
    """The formulas in 64 bits, and the magnitudes that the tolerances go by."""
    F, d = W_dec.shape
    live = (idxs >= 0) & (idxs < F)
    at = torch.where(live, idxs, 0).long()
    flat = at.reshape(-1)
    g, x = g.double(), X.double()
    v = torch.where(live, vals.double(), 0.0)
    k = idxs.shape[1]
    dv, mv = torch.zeros_like(v), torch.zeros_like(v)
    dx, mx = torch.zeros_like(x), torch.zeros_like(x)
    ext = 0.0 if gv is None else gv.double()
    for j in range(k):
        w = W_dec[at[:, j]].double()
        dv[:, j] = (w * g).sum(1)
        mv[:, j] = (w * g).abs().sum(1)
    dv, mv = torch.where(live, dv + ext, 0.0), torch.where(live, mv + (ext.abs() if gv is not None else 0.0), 0.0)
    ev = (16 + d / 64) * U * mv
    out = {}
    zero = torch.zeros(F, d, dtype=torch.float64, device=X.device)
    n = torch.zeros(F, dtype=torch.float64, device=X.device).index_add_(0, flat, live.double().reshape(-1))
    chain = ((n.clamp(max=256) + n / 256 + 2) * U)[:, None]
    dec, mdec, enc, menc, eenc = (zero.clone() for _ in range(5))
    for j in range(k):
        for to, a, b in ((dec, v[:, j], g), (mdec, v[:, j].abs(), g.abs()), (enc, dv[:, j], x),
                         (menc, dv[:, j].abs(), x.abs()), (eenc, ev[:, j], x.abs())):
            to.index_add_(0, at[:, j], a[:, None] * b)
        we = W_enc[at[:, j]].double()
        dx += dv[:, j:j + 1] * we
        mx += (dv[:, j:j + 1].abs() * (k + 2) * U + ev[:, j:j + 1]) * we.abs()
    bz = torch.zeros(F, dtype=torch.float64, device=X.device)
    b = bz.clone().index_add_(0, flat, dv.reshape(-1))
    mb = bz.clone().index_add_(0, flat, dv.abs().reshape(-1))
    eb = bz.clone().index_add_(0, flat, ev.reshape(-1))
    out["vals"] = dv, ev
    out["W_dec"] = dec, chain * mdec
    out["W_enc"] = enc, chain * (menc + eenc) + eenc
    out["b_enc"] = b, chain[:, 0] * (mb + eb) + eb
    out["b_dec"] = g.sum(0), g.shape[0] * U * g.abs().sum(0)
    out["X"] = dx, mx
    return out


def check(got, ref, tol):
    assert got.shape == ref.shape
    half = 0.0
    if got.dtype != torch.float32:
        fi = torch.finfo(got.dtype)
        half = fi.eps / 2 * (ref.abs() + tol) + fi.smallest_normal * fi.eps / 2
    assert torch.all((got.double() - ref).abs() <= tol + half + 1e-44)


def check_all(r, w, names=("vals", "W_dec", "W_enc", "b_enc", "b_dec", "X")):
    for name in names:
        check(getattr(r, name), *w[name])


CASES = [  # B, d, F, k, hot: few codes (one CTA sorts) and many, odd widths, long lists, one token
    (1, 8, 1, 1, 0), (1, 64, 100, 5, 0), (3, 7, 50, 4, 0), (32, 768, 4096, 32, 0), (1, 4096, 70000, 64, 0),
    (64, 33, 20, 128, 0), (128, 264, 3, 64, 0.5), (1000, 40, 513, 8, 0.3), (1001, 1032, 3000, 33, 0.05),
    (2048, 256, 2047, 16, 0.2), (4100, 96, 5, 3, 0), (700, 130, 300000, 20, 0), (5000, 16, 2500, 40, 0.6),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,d,F,k,hot", CASES)
def test_matches_formulas(B, d, F, k, hot, dtype):
    import streamtopk_sae as stk
    t = make(B, d, F, k, dtype, seed=B + d, hot=hot, invalid=B > 2)
    X, W_enc, W_dec, vals, idxs, g = t
    r = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    assert r.X.dtype == dtype and r.W_enc.dtype == dtype and r.W_dec.dtype == dtype
    check_all(r, want(*t))
    again = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    for a, b in zip(r, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B,d,F,k,hot", [(32, 64, 300, 16, 0), (900, 72, 1000, 20, 0.3), (900, 71, 1000, 20, 0.3)])
def test_halves_and_given_gradient(B, d, F, k, hot):
    import streamtopk_sae as stk
    t = make(B, d, F, k, torch.bfloat16, seed=5, hot=hot, invalid=True)
    X, W_enc, W_dec, vals, idxs, g = t
    gv = torch.randn(B, k, generator=gen(6), device="cuda")
    r = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, grad_vals=gv, need_dx=True)
    check_all(r, want(*t, gv=gv))
    w = want(*t)
    dv, dW, db = stk.topk_sae_decode_backward(g, vals, idxs, W_dec)
    for got, name in ((dv, "vals"), (dW, "W_dec"), (db, "b_dec")):
        check(got, *w[name])
    # the encoder alone: dvals is what is given
    w = want(X, W_enc, W_dec, vals, idxs, torch.zeros_like(g), gv=gv)
    for need in (True, False):
        dX, dW, db = stk.topk_sae_encode_backward(gv, idxs, X, W_enc, need_dx=need)
        check(dW, *w["W_enc"])
        check(db, *w["b_enc"])
        if need:
            check(dX, *w["X"])
        else:
            assert dX is None


def test_no_rows_and_views():
    import streamtopk_sae as stk
    t = make(40, 64, 200, 8, torch.bfloat16, seed=9)
    X, W_enc, W_dec, vals, idxs, g = t
    r = stk.topk_sae_backward(g[:0], X[:0], W_enc, W_dec, vals[:0], idxs[:0], need_dx=True)
    assert not r.W_enc.any() and not r.W_dec.any() and not r.b_enc.any() and not r.b_dec.any()
    assert r.vals.shape == (0, 8) and r.X.shape == (0, 64)
    # gradients that are broadcast, strided or in 16 bits, codes as int64, weights that start off 16 bytes
    ones = torch.ones((), device="cuda").expand(40, 64)
    check_all(stk.topk_sae_backward(ones, X, W_enc, W_dec, vals, idxs.long(), need_dx=True),
              want(X, W_enc, W_dec, vals, idxs, ones))
    store = torch.empty(200 * 64 + 3, dtype=torch.bfloat16, device="cuda")
    off = store[3:].view(200, 64).copy_(W_dec)
    gt = g.T.contiguous().T
    a = stk.topk_sae_backward(gt, X, W_enc, off, vals, idxs)
    check_all(a, want(*t), ("vals", "W_dec", "W_enc", "b_enc", "b_dec"))
    check_all(stk.topk_sae_backward(g.to(torch.bfloat16), X, W_enc, W_dec, vals, idxs),
              want(X, W_enc, W_dec, vals, idxs, g.to(torch.bfloat16)), ("vals", "W_dec", "W_enc", "b_enc", "b_dec"))


def test_infinities_stay_with_their_features():
    """A row with NaN reaches only the features that it chose, and an index given twice counts twice."""
    import streamtopk_sae as stk
    t = make(50, 64, 400, 8, torch.float32, seed=10)
    X, W_enc, W_dec, vals, idxs, g = t
    idxs[3, 1] = idxs[3, 0]
    check_all(stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True), want(*t))
    g2 = g.clone()
    g2[7] = math.nan
    a, b = (stk.topk_sae_backward(x, X, W_enc, W_dec, vals, idxs) for x in (g, g2))
    touched = torch.zeros(400, dtype=torch.bool, device="cuda")
    touched[idxs[7].long()] = True
    for name in ("W_dec", "W_enc", "b_enc"):
        x, y = getattr(a, name), getattr(b, name)
        assert torch.equal(x[~touched], y[~touched]) and y[touched].isnan().all()
    # rows behind the last sequence: codes -1, anything in X and g
    idxs[40:] = -1
    X[40:] = math.nan
    c = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    assert c.W_enc.isfinite().all() and c.W_dec.isfinite().all() and not c.X[40:].any() and not c.vals[40:].any()


def test_matches_differences():
    """Central differences of the loss in 64 bits at fixed codes."""
    import streamtopk_sae as stk
    B, d, F, k = 4, 16, 12, 3
    X, W_enc, W_dec, _, _, _ = make(B, d, F, k, torch.float32, seed=11)
    b_enc, b_dec = torch.randn(F, generator=gen(12), device="cuda"), torch.randn(d, generator=gen(13), device="cuda")
    x_hat, vals, idxs = stk.topk_sae_forward(X, W_enc, b_enc, W_dec, b_dec, 2)
    r = stk.topk_sae_backward(2 * (x_hat - X), X, W_enc, W_dec, vals, idxs, need_dx=True)
    at = idxs.long()

    def loss(X, We, be, Wd, bd, target):
        v = (X[:, None, :] * We[at]).sum(2) + be[at]
        return ((bd + (v[:, :, None] * Wd[at]).sum(1) - target) ** 2).sum()

    p = [t.double() for t in (X, W_enc, b_enc, W_dec, b_dec)]
    target = X.double()
    for which, got in enumerate((r.X, r.W_enc, r.b_enc, r.W_dec, r.b_dec)):
        for n in range(0, p[which].numel(), 5):
            h, ends = 1e-4, []
            for sign in (1, -1):
                q = [t.clone() for t in p]
                q[which].view(-1)[n] += sign * h
                ends.append(loss(*q, target))
            diff = (ends[0] - ends[1]) / (2 * h)
            # the loss is quartic at most: differences are good to h^2; sums of some 100 terms below 50 in fp32
            assert abs(float(got.reshape(-1)[n]) - float(diff)) < 1e-5 * 50


@pytest.mark.parametrize("B", [16, 600])
def test_captured_replayed_and_other_stream(B):
    import streamtopk_sae as stk
    t = make(B, 128, 900, 32, torch.bfloat16, seed=14, hot=0.1)
    X, W_enc, W_dec, vals, idxs, g = t
    first = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = stk.topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=True)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, r):
        assert torch.equal(a, b) and torch.equal(a, c)
    n = make(B, 128, 900, 32, torch.bfloat16, seed=15, hot=0.4)
    for a, b in zip(t, n):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(r, stk.topk_sae_backward(n[5], *n[:3], *n[3:5], need_dx=True)):
        assert torch.equal(a, b)


def test_autograd_matches_explicit_calls():
    import streamtopk_sae as stk
    from streamtopk_sae import autograd as ag
    B, d, F, k = 30, 64, 500, 8
    X, W_enc, W_dec, _, _, g = make(B, d, F, k, torch.bfloat16, seed=16)
    b_enc, b_dec = torch.zeros(F, device="cuda"), torch.zeros(d, device="cuda", dtype=torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (X, W_enc, b_enc, W_dec, b_dec)]
    x_hat, vals, idxs = ag.topk_sae_forward(*leaves, k)
    (x_hat * g).sum().backward(retain_graph=True)
    r = stk.topk_sae_backward(g, X, W_enc, W_dec, vals.detach(), idxs, need_dx=True)
    for t, name in zip(leaves, ("X", "W_enc", "b_enc", "W_dec", "b_dec")):
        assert torch.equal(t.grad, getattr(r, name).to(t.dtype)), name
    # the halves, joined by what a program does in between, and vals alone
    for t in leaves:
        t.grad = None
    v, i = ag.topk_sae_encode(*leaves[:3], k)
    (ag.topk_sae_decode(v.relu(), i, *leaves[3:]) * g).sum().backward()
    dv, dWd, dbd = stk.topk_sae_decode_backward(g, v.detach().relu(), i, W_dec)
    dX, dWe, dbe = stk.topk_sae_encode_backward(dv * (v > 0), i, X, W_enc)
    for t, want_ in zip(leaves, (dX, dWe, dbe, dWd, dbd)):
        assert torch.equal(t.grad, want_.to(t.dtype))
    (gv,) = torch.autograd.grad(vals.square().sum(), leaves[2], retain_graph=True)
    w = stk.topk_sae_encode_backward(2 * vals.detach(), idxs, X, W_enc)[2]
    assert torch.allclose(gv, w, rtol=1e-6, atol=1e-6)
    logits = torch.randn(20, 12, generator=gen(17), device="cuda").requires_grad_()
    weights, experts = ag.route_experts(logits, 3, bias=torch.zeros(12, device="cuda"))
    gw = torch.randn(20, 3, generator=gen(18), device="cuda")
    (weights * gw).sum().backward()
    assert torch.equal(logits.grad, stk.route_experts_backward(gw, logits.detach(), experts))


def test_autograd_refuses_capture():
    from streamtopk_sae import autograd as ag
    X, W_enc, W_dec, _, _, _ = make(4, 64, 100, 2, torch.bfloat16, seed=19)
    b = torch.zeros(100, device="cuda")
    W = W_enc.clone().requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        with pytest.raises(RuntimeError, match="cannot be captured"):
            ag.topk_sae_forward(X, W, b, W_dec, None, 2)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            ag.route_experts(X.float(), 2)


def test_refusals():
    import streamtopk_sae as stk
    X, W_enc, W_dec, vals, idxs, g = make(6, 16, 30, 2, torch.bfloat16, seed=20)
    for args, msg in (((g, X.float(), W_enc, W_dec, vals, idxs), "one dtype"),
                      ((g, X, W_enc[:, :8], W_dec, vals, idxs), r"must be \(F, d\)"),
                      ((g[:3], X, W_enc, W_dec, vals, idxs), "grad_x_hat must be"),
                      ((g, X, W_enc, W_dec, vals[:, :1], idxs), r"must be \(B, k\)"),
                      ((g.cpu(), X, W_enc, W_dec, vals, idxs), "must be on CUDA")):
        with pytest.raises(RuntimeError, match=msg):
            stk.topk_sae_backward(*args)
    with pytest.raises(RuntimeError, match="k >= 1"):
        stk.topk_sae_backward(g, X, W_enc, W_dec, vals[:, :0], idxs[:, :0])


@pytest.mark.parametrize("state_bits,dtype", [(32, torch.float32), (8, torch.bfloat16)])
def test_training_steps_together(state_bits, dtype):
    """Whole steps: encode, decode, gradient, AdamW; eager and captured steps agree, and each step's update is AdamW's
    of the gradient in 64 bits of the codes that the encoder chose."""
    import streamtopk_sae as stk
    B, d, F, k = 64, 64, 600, 8
    r = gen(23)
    start = [torch.randn(F, d, generator=r, device="cuda") * d ** -0.5, torch.zeros(F, device="cuda"),
             torch.randn(F, d, generator=r, device="cuda") * d ** -0.5, torch.zeros(d, device="cuda")]
    batches = [torch.randn(B, d, generator=r, device="cuda").to(dtype) for _ in range(5)]
    ends, losses = [], []
    for capturable in (False, True):
        p = [t.clone() for t in start]
        tr = stk.TopkSAETrainer(*p, k, dtype=dtype, lr=1e-3, state_bits=state_bits, capturable=capturable)
        X = batches[0].clone()
        got, graph = [], None
        for x in batches:
            X.copy_(x)
            if not capturable:
                got.append(float(tr.step(X)))
                continue
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    loss = tr.step(X)
            graph.replay()
            got.append(float(loss))
        ends.append(p)
        losses.append(got)
    assert losses[0] == losses[1] and all(math.isfinite(v) for v in losses[0])
    for a, b in zip(*ends):
        assert torch.equal(a, b)
    # the first step by itself: every element moves by at most lr (1 + decay), towards less error
    p = [t.clone() for t in start]
    tr = stk.TopkSAETrainer(*p, k, dtype=dtype, lr=1e-3, weight_decay=0.0, state_bits=state_bits)
    tr.step(batches[0])
    low = [t.to(dtype) for t in (start[0], start[2])]
    x_hat, vals, idxs = stk.topk_sae_forward(batches[0], low[0], start[1], low[1], start[3], k)
    w = want(batches[0], low[0], low[1], vals, idxs, 2 / B * (x_hat - batches[0].float()))
    for t0, t1, name in zip(start, p, ("W_enc", "b_enc", "W_dec", "b_dec")):
        g, tol = w[name]
        sure = g.abs() > 1e-4 * g.abs().max() + 100 * tol
        # AdamW's first step is lr * g / (|g| + eps): lr times the sign
        assert torch.all(((t0 - t1)[sure].double() - 1e-3 * g[sure].sign()).abs() <= 1e-3 * 1e-2 + 2 * U * t0.abs().max())


def test_routed_sae_step():
    """Router, routed encode, decode, the gradients of all of them, AdamW, as a switch SAE trains."""
    import streamtopk_sae as stk
    E, Fe, d, B, k, m = 4, 300, 64, 80, 8, 2
    F = E * Fe
    r = gen(24)
    W_enc, W_dec = (torch.randn(F, d, generator=r, device="cuda") * d ** -0.5 for _ in range(2))
    W_r = torch.randn(E, d, generator=r, device="cuda") * d ** -0.5
    b_enc, b_dec = torch.zeros(F, device="cuda"), torch.zeros(d, device="cuda")
    X = torch.randn(B, d, generator=r, device="cuda")
    logits = X @ W_r.T
    vals, idxs, weights, experts = stk.topk_sae_routed_encode(X, logits, W_enc.view(E, Fe, d), b_enc.view(E, Fe), k, m)
    scaled = (vals.view(B, m, k) * weights[:, :, None]).view(B, m * k)
    x_hat = stk.topk_sae_decode(scaled, idxs, W_dec, b_dec)
    g = 2 / B * (x_hat - X)
    ds, dW_dec, db_dec = stk.topk_sae_decode_backward(g, scaled, idxs, W_dec)
    ds = ds.view(B, m, k)
    dweights = (ds * vals.view(B, m, k)).sum(2)
    dX, dW_enc, db_enc = stk.topk_sae_encode_backward((ds * weights[:, :, None]).reshape(B, m * k), idxs, X, W_enc)
    dlogits = stk.route_experts_backward(dweights, logits, experts)
    dW_r = dlogits.T @ X
    # the same in 64 bits, by differentiation at the same choices
    leaves = [t.double().requires_grad_() for t in (W_enc, b_enc, W_dec, b_dec, W_r)]
    We, be, Wd, bd, Wr = leaves
    x = X.double()
    s = torch.softmax(x @ Wr.T, 1).gather(1, experts.long())
    w = (s / s.sum(1, keepdim=True)).repeat_interleave(k, 1)
    at = idxs.long()
    v = ((x[:, None, :] * We[at]).sum(2) + be[at]) * w
    (((bd + (v[:, :, None] * Wd[at]).sum(1) - x) ** 2).sum() / B).backward()
    for got, leaf in zip((dW_enc, db_enc, dW_dec, db_dec, dW_r), leaves):
        # fp32 throughout (the encode is 3-pass TF32, within 1e-5 of a row's scale)
        scale = leaf.grad.abs().max()
        assert torch.all((got.double() - leaf.grad).abs() <= 1e-4 * scale)
    params = [W_enc, b_enc, W_dec, b_dec, W_r]
    before = [t.clone() for t in params]
    opt = stk.AdamW(params, lr=1e-3, state_bits=8)
    for t, gr in zip(params, (dW_enc, db_enc, dW_dec, db_dec, dW_r)):
        t.grad = gr
    opt.step()
    torch.cuda.synchronize()
    assert all(t.isfinite().all() and not torch.equal(t, b) for t, b in zip(params, before))

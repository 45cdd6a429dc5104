"""The training operators where element offsets pass 32 bits, and with two calls on the GPU at once: the same results as
smaller calls, or calls one after the other, give."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("B,k", [(16, 8), (300, 40)])
def test_sae_backward_of_a_dictionary_beyond_32_bits(B, k):
    """The last features of (1.1 million, 2048): as the same codes in a small dictionary."""
    import streamtopk_sae as stk
    F, d, few = 1_100_000, 2048, 500
    W = torch.zeros(F, d, dtype=torch.bfloat16, device="cuda")
    small = torch.randn(few, d, generator=gen(1), device="cuda").to(torch.bfloat16)
    W[F - few:] = small
    X = torch.randn(B, d, generator=gen(2), device="cuda").to(torch.bfloat16)
    g = torch.randn(B, d, generator=gen(3), device="cuda")
    vals = torch.randn(B, k, generator=gen(4), device="cuda")
    idxs = torch.randint(0, few, (B, k), generator=gen(5), device="cuda", dtype=torch.int32)
    a = stk.topk_sae_backward(g, X, W, W, vals, idxs + (F - few), need_dx=True)
    b = stk.topk_sae_backward(g, X, small, small, vals, idxs, need_dx=True)
    for name in ("W_enc", "b_enc", "W_dec"):
        x = getattr(a, name)
        assert torch.equal(x[F - few:], getattr(b, name))
        assert not x[: F - few].any()
    for name in ("b_dec", "vals", "X"):
        assert torch.equal(getattr(a, name), getattr(b, name))


def test_route_of_rows_beyond_32_bits():
    import streamtopk_sae as stk
    N, E, k = 2_200_000, 1024, 4
    logits = torch.zeros(N, E, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(300, E, generator=gen(6), device="cuda").to(torch.bfloat16)
    logits[N - 300:] = tail
    w, e, c = stk.route_experts(logits, k, return_counts=True)
    ww, ee = stk.route_experts(tail, k)
    assert torch.equal(w[N - 300:], ww) and torch.equal(e[N - 300:], ee)
    assert torch.equal(e[: N - 300], torch.arange(k, dtype=torch.int32, device="cuda").expand(N - 300, k))
    assert int(c.sum()) == N * k
    gw = torch.zeros(N, k, device="cuda")
    gw[N - 300:] = torch.randn(300, k, generator=gen(7), device="cuda")
    got = stk.route_experts_backward(gw, logits, e)
    assert torch.equal(got[N - 300:], stk.route_experts_backward(gw[N - 300:], tail, ee))
    assert not got[: N - 300].any()


def test_adamw_of_a_tensor_beyond_32_bits():
    import streamtopk_sae as stk
    n, tail = (1 << 31) + 12345, 1 << 20
    start = (n - tail) // 256 * 256                      # a block of its own begins here
    p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    ms, vs = (torch.ones(-(-n // 256), device="cuda") for _ in range(2))
    g[start:] = torch.randn(n - start, generator=gen(8), device="cuda").to(torch.bfloat16)
    q = [p[start:].clone(), g[start:].clone(), m[start:].clone(), v[start:].clone(), ms[start // 256:].clone(),
         vs[start // 256:].clone()]
    how = dict(step=1, lr=0.5, weight_decay=0.0)
    stk.adamw_step([p], [g], [m], [v], exp_avg_scales=[ms], exp_avg_sq_scales=[vs], **how)
    stk.adamw_step([q[0]], [q[1]], [q[2]], [q[3]], exp_avg_scales=[q[4]], exp_avg_sq_scales=[q[5]], **how)
    assert torch.equal(p[start:], q[0]) and torch.equal(ms[start // 256:], q[4]) and torch.equal(vs[start // 256:], q[5])
    assert torch.equal(m[start:].view(torch.uint8), q[2].view(torch.uint8))
    assert torch.equal(v[start:].view(torch.uint8), q[3].view(torch.uint8))
    assert bool((p[:start] == 1).all())


def test_two_calls_at_once():
    """Two host threads, each on a stream of its own, many times over."""
    import streamtopk_sae as stk

    def work(seed, stream, out):
        with torch.cuda.stream(stream):
            r = gen(seed)
            B, d, F, k = 200 + seed, 128, 900, 50
            X = torch.randn(B, d, generator=r, device="cuda").to(torch.bfloat16)
            W = torch.randn(F, d, generator=r, device="cuda").to(torch.bfloat16)
            g = torch.randn(B, d, generator=r, device="cuda")
            vals = torch.randn(B, k, generator=r, device="cuda")
            idxs = torch.randint(0, F, (B, k), generator=r, device="cuda", dtype=torch.int32)
            logits, bias = torch.randn(B, 64, generator=r, device="cuda"), torch.randn(64, generator=r, device="cuda") * 0.1
            p, m, v = W.float(), torch.zeros(F, d, device="cuda"), torch.zeros(F, d, device="cuda")
            for step in range(1, 21):
                s = stk.topk_sae_backward(g, X, W, W, vals, idxs)
                w, e, c = stk.route_experts(logits, 6, bias=bias, return_counts=True)
                stk.adamw_step([p], [s.W_enc], [m], [v], step=step, lr=1e-2)
            out[seed] = [*s[1:], w, e, c, p, m, v]
            stream.synchronize()

    alone, together = {}, {}
    for seed in (1, 2):
        work(seed, torch.cuda.Stream(), alone)
    threads = [threading.Thread(target=work, args=(seed, torch.cuda.Stream(), together)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for seed in (1, 2):
        for a, b in zip(alone[seed], together[seed]):
            assert torch.equal(a, b)

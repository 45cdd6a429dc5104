"""The AdamW step (stk_adamw_step) against its formula in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32).  m' = b1 m + (1 - b1) g is a
sum of two products of rounded scalars: each term carries at most four
roundings (gradient scale, scalar, product, sum), so |error| <= 4 u M with
M = |b1 m| + |(1 - b1) g|.  v' is a sum of positive terms with at most seven
roundings each (the gradient's scale twice, the square, scalar, product, sum).
The update: m' 4 u; the denominator 7 u (half of v's six, the root itself, the
two scalars, the product, the sum); the division, good to two units in the last
place, 4 u; the step size and its product 2 u; the subtraction u: 18 u U with
U = M / denominator * step size, 19 with the second order.
p's own term carries three roundings.  What is rounded to 16 bits adds
finfo.eps / 2 of the value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn
HYP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _blocks(t, scales):
    """Each element's scale."""
    return scales.double().repeat_interleave(256)[: t.numel()].view(t.shape)


def make(shapes, seed, pdt=torch.float32, gdt=torch.float32, bits=32, copy=None, offset=0):
    g = _gen(seed)

    def new(shape, dt):
        n = math.prod(shape)
        return torch.zeros(n + offset, dtype=dt, device="cuda")[offset:].view(shape)

    out = {"p": [], "g": [], "m": [], "v": [], "ms": [], "vs": [], "c": []}
    for shape in shapes:
        n = math.prod(shape)
        p, gr = new(shape, pdt), new(shape, gdt)
        p.copy_(torch.randn(shape, generator=g, device="cuda"))
        gr.copy_(torch.randn(shape, generator=g, device="cuda") * 1e-2)
        m32 = torch.randn(shape, generator=g, device="cuda") * 1e-2
        v32 = torch.randn(shape, generator=g, device="cuda").square() * 1e-4
        sdt = torch.float32 if bits == 32 else E4M3
        m, v = new(shape, sdt), new(shape, sdt)
        if bits == 32:
            m.copy_(m32)
            v.copy_(v32)
        else:
            m.copy_((m32 * 1e4).clamp(-448, 448))
            v.copy_((v32.sqrt() * 1e4).clamp(2.0 ** -9, 448))
            nb = -(-n // 256)
            out["ms"].append(torch.rand(nb, generator=g, device="cuda") * 1e-4 + 1e-5)
            out["vs"].append(torch.rand(nb, generator=g, device="cuda") * 1e-4 + 1e-5)
        for name, t in (("p", p), ("g", gr), ("m", m), ("v", v)):
            out[name].append(t)
        if copy is not None:
            out["c"].append(new(shape, copy))
    return out


def formula(t, i, step, scale=1.0, lr=HYP["lr"], betas=HYP["betas"], eps=HYP["eps"], weight_decay=HYP["weight_decay"]):
    """(p', m', v', M, U) in 64 bits."""
    b1, b2 = betas
    p, g = t["p"][i].double(), t["g"][i].double() * scale
    m, v = t["m"][i].double(), t["v"][i].double()
    if t["ms"]:
        m = m * _blocks(m, t["ms"][i])
        v = (v * _blocks(v, t["vs"][i])) ** 2
    M = (b1 * m).abs() + ((1 - b1) * g).abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    denom = (v / (1 - b2 ** step)).sqrt() + eps
    size = lr / (1 - b1 ** step)
    return p * (1 - lr * weight_decay) - size * m / denom, m, v, M, size * M / denom


def call(t, step, **kw):
    import streamtopk_sae as stk
    hyp = dict(HYP)
    hyp.update(kw)
    stk.adamw_step(t["p"], t["g"], t["m"], t["v"], step=step, exp_avg_scales=t["ms"] or None,
                   exp_avg_sq_scales=t["vs"] or None, copies=t["c"] or None, **hyp)


def half_step(dt):
    return 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2


def check(t, want, p_before):
    for i, (p, m, v, M, upd) in enumerate(want):
        tol = U * (19 * upd + 3 * p_before[i].double().abs())
        got = t["p"][i]
        assert torch.all((got.double() - p).abs() <= tol + half_step(got.dtype) * (p.abs() + tol)), i
        if t["c"]:
            c = t["c"][i]
            assert torch.all((c.double() - p).abs() <= tol + half_step(c.dtype) * (p.abs() + tol)), i
        if not t["ms"]:
            assert torch.all((t["m"][i].double() - m).abs() <= 4 * U * M + 1e-45), i
            assert torch.all((t["v"][i].double() - v).abs() <= 7 * U * v + 1e-45), i
            continue
        for codes, scales, x in ((t["m"][i], t["ms"][i], m), (t["v"][i], t["vs"][i], v.sqrt())):
            sc = _blocks(codes, scales)
            top, most = (torch.nn.functional.pad(y.abs().reshape(-1), (0, -x.numel() % 256)).view(-1, 256).amax(1)
                         for y in (x, M if x is m else x))
            assert torch.all((scales.double() * 448 - top).abs() <= 8 * U * most)
            # half a step of E4M3: 2^-4 of the value, 2^-10 of the scale below the normal range (the full 2^-9 where
            # a positive root is kept from 0); the fp32 value before it is within 8 u of its terms
            err = (codes.double() * sc - x).abs()
            least = 2.0 ** -9 if x is not m else 2.0 ** -10
            assert torch.all(err <= torch.maximum(x.abs() * 2.0 ** -4, sc * least) + 16 * U * (x.abs() + M)), i
            if x is not m:
                assert torch.all((codes.float() > 0) | (x == 0))


SHAPES = [(5,), (256,), (257,), (1,), (64, 40), (33, 1037), (8192,), (3, 8200)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdt,gdt,copy,offset", [
    (torch.float32, torch.float32, None, 0), (torch.float32, torch.bfloat16, torch.bfloat16, 0),
    (torch.float32, torch.float16, torch.float16, 1), (torch.bfloat16, torch.bfloat16, None, 0),
    (torch.float16, torch.float32, torch.float32, 3), (torch.bfloat16, torch.bfloat16, None, 1)])
def test_step_matches_formula(bits, pdt, gdt, copy, offset):
    t = make(SHAPES, 7, pdt, gdt, bits, copy, offset)
    before = [p.clone() for p in t["p"]]
    want = [formula(t, i, 3) for i in range(len(SHAPES))]
    call(t, 3)
    check(t, want, before)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_several_launches(bits):
    shapes = [(1 + (37 * i) % 900,) for i in range(131)]
    t = make(shapes, 1, bits=bits)
    before = [p.clone() for p in t["p"]]
    want = [formula(t, i, 1) for i in range(len(shapes))]
    call(t, 1)
    check(t, want, before)


def test_steps_in_a_row_and_empty_tensors():
    t = make([(300,), (0,), (7, 0), (50, 50)], 2, bits=32)
    for step in range(1, 6):
        before = [p.clone() for p in t["p"]]
        want = [formula(t, i, step) for i in range(4)]
        call(t, step)
        check(t, want, before)


@pytest.mark.parametrize("bits", [32, 8])
def test_same_bits_twice_and_any_layout(bits):
    """A block's result depends on its values alone, not on alignment or on the launch."""
    ref = make([(4096,), (700,)], 3, bits=bits)
    call(ref, 9)
    for offset in (0, 1, 5):
        t = make([(4096,), (700,)], 3, bits=bits, offset=offset)
        call(t, 9)
        for name in ("p", "m", "v", "ms", "vs"):
            for a, b in zip(ref[name], t[name]):
                assert torch.equal(a.view(torch.uint8) if a.dtype == E4M3 else a, b.view(torch.uint8) if b.dtype == E4M3 else b)


def test_device_step_lr_and_grad_scale():
    t = make(SHAPES, 4)
    before = [p.clone() for p in t["p"]]
    want = [formula(t, i, 12, scale=0.25, lr=float(torch.tensor(3e-3))) for i in range(len(SHAPES))]
    call(t, torch.tensor(12, device="cuda"), lr=torch.tensor(3e-3, device="cuda"),
         grad_scale=torch.tensor([0.25], device="cuda"))
    check(t, want, before)


def test_extreme_values_stay_in_their_block():
    """Zeros, tiny values, infinities and NaN in one block leave the other blocks alone; a zero gradient on zero state
    moves nothing but the decay."""
    t = make([(1024,)], 5, bits=8)
    clean = make([(1024,)], 5, bits=8)
    t["g"][0][256:260] = torch.tensor([math.inf, -math.inf, math.nan, 1e30], device="cuda")
    for x in (t, clean):
        x["g"][0][512:768] = 0
        x["m"][0][512:768] = 0
        x["v"][0][512:768] = 0
    p0 = t["p"][0].clone()
    call(t, 2)
    call(clean, 2)
    m, v = t["m"][0].float(), t["v"][0].float()
    assert m[256:259].isnan().all() and v[256:259].isnan().all()
    rest = torch.ones(1024, dtype=torch.bool, device="cuda")
    rest[256:512] = False
    for name in ("m", "v", "p"):
        assert torch.equal(t[name][0].float()[rest], clean[name][0].float()[rest])
    assert m[260:512].isfinite().all() and t["p"][0][260:512].isfinite().all()
    assert float(t["ms"][0][2]) == 1 and float(t["vs"][0][2]) == 1
    assert m[512:768].eq(0).all() and v[512:768].eq(0).all()
    decay = 1 - HYP["lr"] * HYP["weight_decay"]
    assert torch.all((t["p"][0][512:768].double() - p0[512:768].double() * decay).abs() <= 3 * U * p0[512:768].abs())


def test_optimizer_trains_and_captures():
    import streamtopk_sae as stk
    for bits in (32, 8):
        runs = []
        for capturable in (False, True):
            g = _gen(11)
            p = torch.randn(40, 30, generator=g, device="cuda")
            q = torch.randn(17, generator=g, device="cuda")
            low = torch.empty_like(p, dtype=torch.bfloat16)
            opt = stk.AdamW([p, q], lr=1e-2, state_bits=bits, copies={p: low}, capturable=capturable)
            p.grad, q.grad = torch.empty_like(p), torch.empty_like(q)
            grads = [(torch.randn(40, 30, generator=g, device="cuda"), torch.randn(17, generator=g, device="cuda"))
                     for _ in range(4)]
            graph = None
            for a, b in grads:
                p.grad.copy_(a)
                q.grad.copy_(b)
                if not capturable:
                    opt.step()
                    continue
                if graph is None:
                    torch.cuda.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        opt.step()
                graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(low, p.to(torch.bfloat16))
            runs.append((p, q))
        for a, b in zip(*runs):
            assert torch.equal(a, b)


def test_optimizer_state_dict_and_missing_grads():
    import streamtopk_sae as stk
    g = _gen(12)
    p = [torch.randn(300, generator=g, device="cuda") for _ in range(2)]
    a = stk.AdamW(p, state_bits=8)
    p[0].grad = torch.randn(300, generator=g, device="cuda")
    a.step()
    assert [s["step"] for s in a.state] == [1, 0]
    b = stk.AdamW([x.clone() for x in p], state_bits=8)
    b.load_state_dict(a.state_dict())
    for x, y in zip(p, b.params):
        x.grad = torch.randn(300, generator=g, device="cuda")
        y.grad = x.grad.clone()
    a.step()
    b.step()
    assert all(torch.equal(x, y) for x, y in zip(p, b.params))
    with pytest.raises(RuntimeError, match="other params"):
        stk.AdamW(p, state_bits=32).load_state_dict(a.state_dict())


def test_autograd_notices_a_step():
    """A backward pass over weights that a step has changed since is refused, as with torch's own optimizers."""
    import streamtopk_sae as stk
    w = torch.ones(300, device="cuda", requires_grad=True)
    opt = stk.AdamW([w])
    loss = (w * w).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_on_another_stream_and_expanded_gradient():
    t = make([(500, 64)], 6)
    t["g"][0] = torch.full((1,), 0.5, device="cuda").expand(500, 64)
    want = [formula(t, 0, 1)]
    before = [t["p"][0].clone()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call(t, 1)
    s.synchronize()
    check(t, want, before)


def test_refusals():
    import streamtopk_sae as stk
    t = make([(300,), (20,)], 8, bits=8)
    before = t["p"][0].clone()
    with pytest.raises(RuntimeError, match="given twice"):
        call({**t, "p": [t["p"][0], t["p"][0]], "g": [t["g"][0]] * 2, "m": [t["m"][0], t["m"][0].clone()],
              "v": [t["v"][0], t["v"][0].clone()], "ms": [t["ms"][0]] * 2, "vs": [t["vs"][0]] * 2}, 1)
    with pytest.raises(RuntimeError, match="one for every 256"):
        call({**t, "ms": [t["ms"][0][:1], t["ms"][1]]}, 1)
    with pytest.raises(RuntimeError, match="must be contiguous"):
        x = torch.zeros(20, 30, device="cuda").T
        stk.adamw_step([x], [x], [x], [x], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="step must be >= 1"):
        call(t, 0)
    with pytest.raises(RuntimeError, match="lr must be >= 0"):
        call(t, 1, lr=float("nan"))
    with pytest.raises(RuntimeError, match="betas"):
        call(t, 1, betas=(0.9, 1.0))
    with pytest.raises(RuntimeError, match="step must be one int64"):
        call(t, torch.ones(1, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(before, t["p"][0])

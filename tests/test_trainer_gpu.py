"""TopkSAETrainer's weights are the user's own: what a program does to them between steps is what the next step sees.

Both sides of a comparison run the same kernels on the same values, so results are compared bit for bit.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

B, D, F, K = 48, 64, 500, 8


def start(seed=31):
    r = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(F, D, generator=r, device="cuda") * D ** -0.5, torch.randn(F, generator=r, device="cuda") * 0.1,
            torch.randn(F, D, generator=r, device="cuda") * D ** -0.5, torch.randn(D, generator=r, device="cuda") * 0.1]


def batches(n, dtype, seed=32):
    r = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, D, generator=r, device="cuda").to(dtype) for _ in range(n)]


def in_place(W_enc, W_dec):
    W_dec.div_(W_dec.norm(dim=1, keepdim=True))
    W_enc[3:9] = W_dec[3:9] * 0.2


def by_data(W_enc, W_dec):
    W_dec.data /= W_dec.data.norm(dim=1, keepdim=True)
    W_enc.data[3:9] = W_dec.data[3:9] * 0.2


def fresh(trainer, **how):
    """A trainer of the same weights and states that has kept nothing else."""
    import streamtopk_sae as stk
    t = stk.TopkSAETrainer(*(p.clone() for p in trainer.params), K, dtype=trainer.dtype, **how)
    t.optimizer.load_state_dict(trainer.optimizer.state_dict())
    return t


def same(a, b):
    for x, y in zip(a.params, b.params):
        assert torch.equal(x, y)
    assert torch.equal(a.W_enc, b.W_enc) and torch.equal(a.W_dec, b.W_dec)
    for W, low in ((a.params[0], a.W_enc), (a.params[2], a.W_dec)):
        assert torch.equal(W.to(a.dtype), low)


@pytest.mark.parametrize("change", [in_place, by_data])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_step_sees_weights_that_were_changed(dtype, change):
    """Decoder rows brought back to length 1 and features given new weights, between eager steps."""
    import streamtopk_sae as stk
    how = dict(lr=1e-2, state_bits=32)
    t = stk.TopkSAETrainer(*start(), K, dtype=dtype, **how)
    for x in batches(3, dtype):
        change(t.params[0], t.params[2])
        other = fresh(t, **how)
        assert torch.equal(t.step(x), other.step(x))
        same(t, other)


@pytest.mark.parametrize("inside", [False, True])
def test_a_replayed_step_sees_weights_that_were_changed(inside):
    """The same between replays of a captured step, and where the change is captured along with the step."""
    import streamtopk_sae as stk
    how = dict(lr=1e-2, state_bits=8, capturable=True)
    xs = batches(4, torch.bfloat16)
    t = stk.TopkSAETrainer(*start(), K, **how)
    x = xs[0].clone()
    t.step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = t.step(x)
        if inside:
            in_place(t.params[0], t.params[2])
    for new in xs[1:]:
        if not inside:
            in_place(t.params[0], t.params[2])
        other = fresh(t, **how)
        x.copy_(new)
        graph.replay()
        assert torch.equal(loss, other.step(new))
        if inside:
            in_place(other.params[0], other.params[2])
        for a, b in zip(t.params, other.params):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("made,stepped", [(True, False), (False, True), (True, True)])
def test_made_or_stepped_in_inference_mode(made, stepped, dtype):
    """As outside of it: weights of inference mode stepped outside, others inside."""
    import streamtopk_sae as stk
    x = batches(1, dtype)[0]
    plain = stk.TopkSAETrainer(*start(), K, dtype=dtype, lr=1e-2)
    with torch.inference_mode(made):
        t = stk.TopkSAETrainer(*start(), K, dtype=dtype, lr=1e-2)
    for _ in range(2):
        want = plain.step(x)
        with torch.inference_mode(stepped):
            assert torch.equal(t.step(x), want)
    same(t, plain)


def test_weights_that_autograd_knows():
    import streamtopk_sae as stk
    x = batches(1, torch.bfloat16)[0]
    plain, t = (stk.TopkSAETrainer(*(p.requires_grad_(grad) for p in start()), K, lr=1e-2) for grad in (False, True))
    for _ in range(2):
        assert torch.equal(t.step(x), plain.step(x))
    same(t, plain)
    assert not t.W_enc.requires_grad

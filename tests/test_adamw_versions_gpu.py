"""What autograd learns of an AdamW step, which writes its tensors by their addresses."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_autograd_learns_of_a_step(bits):
    """A backward pass over weights that adamw_step has changed since, or over their copies, is refused, as after torch's
    own operations in place; the gradient, which is read, is as it was."""
    import streamtopk_sae as stk
    w = torch.ones(300, device="cuda", requires_grad=True)
    copy = torch.ones(300, device="cuda")
    dt = torch.float8_e4m3fn if bits == 8 else torch.float32
    m, v = (torch.zeros(300, dtype=dt, device="cuda") for _ in range(2))
    scales = [torch.ones(2, device="cuda") for _ in range(2)] if bits == 8 else []
    x = torch.ones(300, device="cuda", requires_grad=True)
    losses = [(w * w).sum(), (x * copy).sum()]
    grad = torch.ones(300, device="cuda")
    stk.adamw_step([w], [grad], [m], [v], step=1, lr=0.1, copies=[copy], exp_avg_scales=scales[:1] or None,
                   exp_avg_sq_scales=scales[1:] or None)
    assert w._version == copy._version == 1 and grad._version == 0
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("kind", [tuple, list, torch.nn.ParameterList])
def test_sequences_of_tensors_and_no_copies(kind):
    import streamtopk_sae as stk
    p, m, v = ([torch.zeros(40, device="cuda"), torch.zeros(3, device="cuda")] for _ in range(3))
    p = kind(p)
    versions = [t._version for t in p]
    stk.adamw_step(p, tuple(torch.ones_like(t) for t in p), m, v, step=1, lr=0.1)
    assert all(t._version > n and bool((t < 0).all()) for t, n in zip(p, versions))


def test_tensors_of_inference_mode():
    """They have no version, and are stepped like any other."""
    import streamtopk_sae as stk
    with torch.inference_mode():
        p, m, v = (torch.zeros(40, device="cuda") for _ in range(3))
    stk.adamw_step([p], [torch.ones(40, device="cuda")], [m], [v], step=1, lr=0.1)
    assert bool((p < 0).all())
    with torch.inference_mode():
        stk.adamw_step([p], [torch.ones(40, device="cuda")], [m], [v], step=2, lr=0.1)
        assert bool((p < -0.15).all())

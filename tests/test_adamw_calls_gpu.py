"""A step that AdamW refuses leaves params, states, step counts and copies as they were."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def state(o):
    return [x.clone() if isinstance(x, torch.Tensor) else x for s in o.state for x in s.values()]


def equal(a, b):
    raw = [(x.view(torch.uint8) if isinstance(x, torch.Tensor) and x.dtype == torch.float8_e4m3fn else x) for x in (a, b)]
    return torch.equal(*raw) if isinstance(a, torch.Tensor) else a == b


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("fault", ["shape", "scale", "copy", "betas", "lr", "missing"])
def test_a_refused_step_changes_nothing(fault, capturable, bits):
    """Params in two groups (fp32 and bf16), the second one's arguments, or all, refused."""
    import streamtopk_sae as stk
    p = [torch.randn(300, device="cuda"), torch.randn(70, device="cuda").to(torch.bfloat16)]
    low = torch.zeros(70, device="cuda")
    o = stk.AdamW(p, state_bits=bits, capturable=capturable, copies={p[1]: low})
    grads = [torch.randn(300, device="cuda"), torch.randn(70, device="cuda").to(torch.bfloat16)]
    o.step(grads)
    start, before = [t.clone() for t in p], state(o)
    bad, how = list(grads), {}
    good = (o.betas, o.lr)
    if fault == "shape":
        bad[1] = bad[1][:69]
    elif fault == "scale":
        how["grad_scale"] = torch.ones(2, device="cuda")
    elif fault == "copy":
        o.copies[1] = low[:69]
    elif fault == "betas":
        o.betas = (0.9, math.nan)
    elif fault == "lr":
        o.lr = -1.0
    elif not capturable:
        pytest.skip("a param without a gradient is passed over")
    else:
        bad[1] = None
    with pytest.raises(RuntimeError):
        o.step(bad, **how)
    assert all(torch.equal(a, b) for a, b in zip(p, start))
    assert all(equal(a, b) for a, b in zip(state(o), before))
    if capturable:
        assert int(o.step_dev) == 1
    # and the next one is as if it had not been
    o.copies[1], o.betas, o.lr = low, *good
    o.step(grads)
    q = [t.clone() for t in start]
    other = stk.AdamW(q, state_bits=bits, capturable=capturable, copies={q[1]: torch.zeros_like(low)})
    it = iter(before)
    for s in other.state:
        for name in s:
            s[name] = next(it)
    if capturable:
        other.step_dev.fill_(1)
    other.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(p, q))

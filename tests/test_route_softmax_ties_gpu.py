"""Choices of softmax scores with a bias that differ by less than fp32 can tell: those of 64 bits have to come out, at
every number of experts a lane holds.  (The sigmoid's are in test_route_gpu, with the tolerances.)"""
import pytest
import torch
from test_route_gpu import close, plain, randn, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spread", [0.0, 3e-7, 3e-6])
@pytest.mark.parametrize("E,N,groups", [(20, 300, (4, 2)), (64, 300, (8, 3)), (64, 4200, (4, 2)), (256, 4200, (8, 4)),
                                        (300, 300, (4, 2)), (1024, 300, (32, 5))])
def test_choice_is_that_of_64_bits(E, N, groups, spread):
    """s + bias equal to within 2^-25 or so, or spread over `spread`, in rows that are one row moved by a constant and
    rounded, which leaves the scores but for the rounding of the logits."""
    k = 8
    logits = randn(N, E, seed=E)
    s = torch.softmax(logits[0].double(), 0)
    noise = torch.rand(E, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    bias = (0.7 + spread * noise - s).float()
    logits[1:150] = logits[0] + randn(149, 1, seed=4)
    logits[150:200] = logits[0]
    logits[150:200, ::2] -= 1e-6
    logits[200:230, ::3] = logits[200:230, :1]            # equal logits, equal biases below
    flat = bias.clone()
    flat[::3] = flat[0]
    n_groups, topk_groups = groups
    for b in (bias, flat):
        for kw in ({}, {"n_groups": n_groups, "topk_groups": topk_groups}):
            w, e = run(logits, k, bias=b, **kw)
            at = torch.cat([torch.arange(230), torch.arange(230, N, 50)]).cuda()
            pw, pe = plain(logits[at], k, bias=b, **kw)
            assert torch.equal(e[at].cpu(), pe)
            close(w[at], pw, logits[at], "softmax")
            if spread == 0.0 and not kw and b is bias:  # so close that rounding the logits decides
                assert len({tuple(row) for row in e[:150].tolist()}) > 1

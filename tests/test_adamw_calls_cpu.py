"""What AdamW refuses leaves it as it was, without a GPU: params that are not on CUDA are refused by the step itself."""
import pytest
import torch

from streamtopk_sae import optim


def test_a_refused_step_is_not_counted():
    p = torch.ones(5)
    o = optim.AdamW([p], capturable=True)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        o.step([torch.ones(5)])
    assert int(o.step_dev) == 0


def test_capturable_takes_one_device():
    with pytest.raises(RuntimeError, match="on one device"):
        optim.AdamW([torch.ones(5), torch.ones(5, device="meta")], capturable=True)
    optim.AdamW([torch.ones(5), torch.ones(5, device="meta")])
    optim.AdamW([], capturable=True)

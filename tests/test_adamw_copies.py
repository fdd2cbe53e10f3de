"""Copies and pickles of optim.AdamW before its first step (no GPU needed)."""
import copy
import pickle

import pytest
import torch

from loquetier_amd.optim import AdamW


@pytest.mark.parametrize("again", [copy.deepcopy, copy.copy, lambda o: pickle.loads(pickle.dumps(o))])
def test_before_the_first_step(again):
    p = [torch.nn.Parameter(torch.zeros(4, 3)) for _ in range(2)]
    opt = AdamW([dict(params=p[:1], lr=0.5), dict(params=p[1:])], lr=0.25, state_bits=8, master=False)
    one = again(opt)
    assert (one.state_bits, one.master) == (8, False) and one.state_dict() == opt.state_dict()
    one.load_state_dict(opt.state_dict())
    one.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2))]))
    with pytest.raises(RuntimeError, match="No suitable kernel"):  # (nothing is on a GPU)
        one.step()

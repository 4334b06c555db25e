"""nmrf_amd.optim.AdamW's state before its first step, and moments that share storage (nmrf_amd/ops/adamw.py)."""
import pytest
import torch

from nmrf_amd import optim as O


def test_asking_for_moments_leaves_no_state_behind():
    p = torch.nn.Parameter(torch.zeros(4))
    o = O.AdamW([p], lr=0.1)
    with pytest.raises(KeyError, match="no step"):
        o.moments(p)
    assert o.state_dict()["state"] == {}
    o.state[p]                                                      # (a defaultdict: anyone's lookup leaves an empty entry)
    sd = o.state_dict()
    assert sd["state"] == {}
    c = O.AdamW([torch.nn.Parameter(torch.zeros(4))])
    c.load_state_dict(sd)
    assert c.param_groups[0]["lr"] == 0.1

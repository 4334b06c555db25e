"""nmrf_amd.optim.AdamW's state before its first step, and moments that share storage (nmrf_amd/ops/adamw.py)."""
import pytest
import torch

from nmrf_amd import _lib
from nmrf_amd import optim as O
from nmrf_amd.ops import AdamWPlan


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


@pytest.mark.gpu
def test_shared_storage_is_refused():
    z = lambda n, dt=torch.float32: torch.zeros(n, device="cuda", dtype=dt)  # noqa: E731
    flat = z(1000)
    m = z(300)
    for p, a, b in (([z(300)], [m], [m]), ([flat[:300], flat[299:599]], [z(300), z(300)], [z(300), z(300)]),
                    ([z(300), z(300)], [m, m], [z(300), z(300)]), ([flat[:300]], [flat[200:500]], [z(300)])):
        with pytest.raises(_lib.NmrfHipError, match="share storage"):
            AdamWPlan(p, a, b)
    c = z(600, torch.uint8)
    s = z(4)
    for a, b, sa, sb in ((c[:300], c[300:], s[:2], s[1:3]), (c[:300], c[299:599], s[:2], s[2:])):
        with pytest.raises(_lib.NmrfHipError, match="share storage"):
            AdamWPlan([z(300)], [a], [b], [sa], [sb])
    # neighbours in one buffer are the ordinary case, empty tensors anywhere
    plan = AdamWPlan([flat[:300], flat[300:300], flat[300:600]], [z(300), z(0), z(300)], [z(300), z(0), z(300)])
    plan.step([torch.ones(300, device="cuda"), z(0), torch.ones(300, device="cuda")], step=1, lr=0.5)
    # (m / bc1) / (sqrt(v / bc2) + eps) = 1 / (1 + 1e-8): -0.5 after a handful of roundings
    assert float((flat[:600] + 0.5).abs().max()) <= 8 * 0.5 * 2.0 ** -24 + 1e-8 and not bool(flat[600:].any())
    plan = AdamWPlan([z(300)], [c[:300]], [c[300:]], [s[:2]], [s[2:]])
    plan.step([torch.ones(300, device="cuda")], step=1, lr=0.5)

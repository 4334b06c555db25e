"""relu in the gated feed-forward block with every row at work: g is kept away from the jump of its slope by the gate's bias (2 in size, of random sign, against
x Wg^T of spread 0.25), so that half of the hidden values are open and no row or product of any size is empty.  Bounds as in test_gated_ffn."""
import pytest
import torch

from tests.test_gated_ffn import SHAPES, case, check, formula

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [s for i, s in enumerate(SHAPES) if i % 3 == 2] + [(4099, 520, 1600, 515)])
def test_relu_with_every_row(shape, dtype):
    t, d, f, do = shape
    v, dy = case(*shape, dtype, bias=True, seed=31, odd=True)
    gen = torch.Generator(device="cuda").manual_seed(32)
    v["x"].mul_(0.25)
    v["b_gate"].copy_(2 - 4 * (torch.rand(f, generator=gen, device="cuda") < 0.5).to(dtype))
    v["b_gate"][0] = 2.0
    g = v["x"].double() @ v["w_gate"].double().t() + v["b_gate"].double()
    assert float(g.abs().min()) > 0.1                               # (the products' errors are below 1e-2)
    want, _ = formula(v, dy, "relu")
    assert bool((want["y"][0] != 0).all()) and float((want["x"][0] != 0).double().mean()) > 0.99
    for k in ("w_gate", "w_up", "w_down"):                          # (a closed gate has no gradient; h of a closed gate none to give)
        on = v["b_gate"] > 0
        assert float((want[k][0][on] if k != "w_down" else want[k][0][:, on]).ne(0).double().mean()) > 0.99, k
    check(v, dy, "relu")
    check(v, dy, "relu", grad=False)

"""Dense products: forms that only outputs with aligned rows take, fp32 sums of long rows, small activations."""
import math

import pytest

from test_linear_dense import OWN, SLOPE, act64, check, half_step, sum_tol, untouched, wide


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 3000])
def test_gelu_of_negative_values(pkg, cuda, rows):
    """v (1 + erf(v / sqrt 2)) / 2 keeps its relative accuracy where 1 + erf is small.  With a^2 = v^2 / 2: exp(-a^2) by the fast exponential (2 + 1.2 a^2 units in
    the last place, an argument rounded to a^2 half steps: 4 + 3.4 a^2 half steps), its factor within 8, the products within 3."""
    import torch
    for dtype in (torch.bfloat16, torch.float16):
        v = torch.linspace(-9, 3, rows * 64, device=cuda).reshape(rows, 64).to(dtype)
        x, w = torch.zeros((rows, 64), dtype=dtype, device=cuda), torch.zeros((64, 64), dtype=dtype, device=cuda)
        w.fill_diagonal_(1)
        x.copy_(v)
        d = v.double()
        want, a2 = 0.5 * d * torch.special.erfc(-d / math.sqrt(2)), d * d / 2
        tol = want.abs() * (11 + 3 * (2 * a2 + 2)) * 2.0 ** -24 + 2.0 ** -140
        got = pkg.linear(x, w, act="gelu", out_dtype=torch.float32)
        both = pkg.gated_linear(x, w, w, bias_gate=None, bias_up=torch.ones(64, device=cuda), act="gelu", out_dtype=torch.float32)
        narrow = pkg.linear(x, w, act="gelu")
        torch.cuda.synchronize()
        assert ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() / tol).max())
        assert ((both.double() - want * (d + 1)).abs() <= tol * (d + 1).abs() + (want * (d + 1)).abs() * 2.0 ** -23).all()
        tiny = torch.finfo(dtype).smallest_normal
        assert ((narrow.double() - want).abs() <= tol + (want.abs() + tiny) * half_step(dtype) * (1 + 2.0 ** -10)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 40, 3000])
def test_gelu_of_the_largest_values(pkg, cuda, rows):
    """Infinities, NaN and values whose square is beyond the range: as the formula has it."""
    import torch
    special = torch.tensor([float("inf"), -float("inf"), float("nan"), 3e38, -3e38, 1e20, -1e20, 0.0, -0.0, -40.0, 40.0], device=cuda)
    x, w = torch.zeros((rows, 8), dtype=torch.bfloat16, device=cuda), torch.zeros((len(special), 8), dtype=torch.bfloat16, device=cuda)
    got = pkg.linear(x, w, bias=special, act="gelu", out_dtype=torch.float32)
    torch.cuda.synchronize()
    d = special.double()
    want = 0.5 * d * (1 + torch.erf(d / math.sqrt(2)))
    assert torch.equal(torch.isnan(got), torch.isnan(want).expand(rows, -1)) and int(torch.isnan(want).sum()) == 2
    fine = ~torch.isnan(want)
    assert torch.equal(got.double()[:, fine], want[fine].expand(rows, -1).float().double())

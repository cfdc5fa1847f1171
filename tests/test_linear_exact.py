"""Dense products: forms that only outputs with aligned rows take, fp32 sums of long rows, small activations."""
import math

import pytest

from test_linear_dense import OWN, SLOPE, act64, check, half_step, sum_tol, untouched, wide


def long_tol(x, w, passes=512):
    """How far a product with an fp32 output may be off.  Sums of at most 512 k: 32 groups of 16, for each at most two truncations by a step of 2^-23 of what has
    been added up in magnitude so far, the sum of |x w| over the sum's k; that is least tight where all of it comes first, 64 steps of the whole, and on
    rows whose magnitudes are spread evenly 2 * (1 + .. + 32) / 32 = 33.  Then an fp32 addition for each sum (half a step) and for each of at most 16 parts of K."""
    K = x.shape[1]
    groups = math.ceil(min(K, passes) / 16)
    # evenly spread rows: the first j of n groups hold at most (j + 2) / n of the whole
    first = 2 * sum(min(1.0, (j + 2) / groups) for j in range(1, groups + 1))
    return (first + 0.5 * (math.ceil(K / passes) + 16)) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t())


def aligned(rows, N, dtype, cuda, more):
    import torch
    buf = torch.full((rows + 2, N + more), -7.0, dtype=dtype, device=cuda)
    return buf, buf[:rows, :N]


def plain(pkg, cuda, rows, K, N, dtype, bias_t, act, res_t, out_t, seed, res_more=0, inplace=False):
    """Output rows 16-byte aligned (8 elements of room behind each), residual rows aligned or not."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(seed)
    x, w = wide(gen, rows, K, -K % 8 + 8, dtype), wide(gen, N, K, -K % 8, dtype, K ** -0.5)
    bias = None if bias_t is None else torch.randn(N, generator=gen, device=cuda).to(bias_t)
    buf, out = aligned(rows, N, out_t, cuda, 8)
    residual = None
    if res_t is not None:
        residual = torch.randn((rows, N + res_more), generator=gen, device=cuda).to(res_t)[:, :N]
        if inplace:
            out.copy_(residual)
            residual = out.clone()
    v = x.double() @ w.double().t()
    if bias is not None:
        v = v + bias.double()
    tol = sum_tol(x, w, bias) * SLOPE + OWN * v.abs()
    want = act64(v, act)
    if residual is not None:
        want = want + residual.double()
        tol = tol + want.abs() * 2.0 ** -24
    pkg.linear(x, w, out=out, bias=bias, act=act, residual=out if inplace else residual)
    torch.cuda.synchronize()
    check(out, want, tol, out_t)
    assert untouched(buf, rows, N)


def gated(pkg, cuda, rows, K, N, dtype, bias_t, act, limit, out_t, seed):
    import torch
    gen = torch.Generator(device=cuda).manual_seed(seed)
    x = wide(gen, rows, K, -K % 8, dtype)
    wg, wu = wide(gen, N, K, -K % 8, dtype, 2 * K ** -0.5), wide(gen, N, K, -K % 8 + 8, dtype, 2 * K ** -0.5)
    bg, bu = (None, None) if bias_t is None else (torch.randn(N, generator=gen, device=cuda).to(bias_t) for _ in range(2))
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    if bg is not None:
        g, u = g + bg.double(), u + bu.double()
    dg, du = sum_tol(x, wg, bg), sum_tol(x, wu, bu)
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    a = act64(g, act)
    tol = (dg * SLOPE + OWN * g.abs()) * (u.abs() + du) + a.abs() * du + (a * u).abs() * 2.0 ** -24
    buf, out = aligned(rows, N, out_t, cuda, 8)
    pkg.gated_linear(x, wg, wu, out=out, bias_gate=bg, bias_up=bu, act=act, limit=limit)
    torch.cuda.synchronize()
    check(out, a * u, tol, out_t)
    assert untouched(buf, rows, N)


# Few outputs against the rows, so that rows lie along M: remainders of rows and outputs, one and several rounds of tiles, short and long K
FEW = [(3000, 1024, 304), (4096, 4096, 288), (8191, 2048, 64), (8192, 2048, 72), (5001, 584, 88), (3001, 1000, 304), (2500, 2048, 296)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", FEW)
def test_few_outputs(pkg, cuda, rows, K, N):
    import torch
    b, h, f = torch.bfloat16, torch.float16, torch.float32
    for i, (dtype, bias_t, act, res_t, out_t, res_more, inplace) in enumerate([
            (b, f, "silu", None, b, 0, False), (h, h, "none", h, h, 0, True), (b, b, "gelu_tanh", f, f, 0, True), (h, f, "relu", f, h, 3, False),
            (b, None, "none", b, f, 1, False), (h, f, "gelu", None, f, 0, False), (b, None, "none", b, b, 8, False)]):
        plain(pkg, cuda, rows, K, N, dtype, bias_t, act, res_t, out_t, rows + K + i, res_more, inplace)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", FEW + [(8192, 4096, 384)])
def test_few_gated_outputs(pkg, cuda, rows, K, N):
    import torch
    b, h, f = torch.bfloat16, torch.float16, torch.float32
    for i, (dtype, bias_t, act, limit, out_t) in enumerate([(b, f, "silu", 10.0, b), (h, None, "gelu_tanh", 0.0, h), (b, b, "silu", 2.0, f), (h, h, "gelu", 0.0, f)]):
        gated(pkg, cuda, rows, K, N, dtype, bias_t, act, limit, out_t, rows + K + i)


# The down projection of a prompt's dense shared expert: fp32 sums of several passes, added to what is there
@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(4096, 1536, 2048), (2000, 776, 1500), (3001, 1100, 1001), (1000, 4096, 4096), (300, 2048, 2048), (60, 1536, 2048)])
def test_long_rows_onto_their_residual(pkg, cuda, rows, K, N):
    import torch
    b, h, f = torch.bfloat16, torch.float16, torch.float32
    plain(pkg, cuda, rows, K, N, b, None, "none", f, f, rows, 0, True)
    plain(pkg, cuda, rows, K, N, h, f, "silu", h, f, rows + 1, 5, False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(1, 4096, 512), (16, 2048, 512), (16, 16384, 520), (40, 16384, 520), (200, 16384, 1000), (2048, 16384, 2048), (4096, 16384, 288), (8192, 8192, 64)])
def test_fp32_sums_of_long_rows(pkg, cuda, rows, K, N):
    """fp32 outputs are as far off as sums of 512 k: one sum over all of K, truncated at each step, would lose K / 64 half steps on rows of one sign."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(rows + K)
    for dtype in (torch.bfloat16, torch.float16):
        x = (1 + torch.rand((rows, K), generator=gen, device=cuda)).to(dtype)
        w = (1 + torch.rand((N, K), generator=gen, device=cuda)).to(dtype)
        want = x.double() @ w.double().t()
        out, tol = torch.zeros((rows, N), device=cuda), long_tol(x, w)
        pkg.linear(x, w, out=out)
        torch.cuda.synchronize()
        assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())
        up = (torch.rand((N, K), generator=gen, device=cuda) / K).to(dtype)
        pkg.gated_linear(x, w, up, out=out, act="none")
        torch.cuda.synchronize()
        u = x.double() @ up.double().t()
        both = tol * u + long_tol(x, up) * want + 2 * want * u * 2.0 ** -24
        assert ((out - want * u).abs() <= both * (1 + 2.0 ** -15)).all(), float(((out - want * u).abs() / both).max())
        # signs as they come
        x, w = (torch.randn((n, K), generator=gen, device=cuda).to(dtype) for n in (rows, N))
        pkg.linear(x, w, out=out)
        torch.cuda.synchronize()
        assert ((out - x.double() @ w.double().t()).abs() <= long_tol(x, w)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 3000])
def test_gelu_of_negative_values(pkg, cuda, rows):
    """v (1 + erf(v / sqrt 2)) / 2 keeps its relative accuracy where 1 + erf is small.  a = -v / sqrt 2 is off by three half steps, which erfc(a) multiplies by
    2 a exp(-a^2) / (sqrt(pi) erfc(a)) < 2 a^2 + 2; erfc itself by eight, the products by three."""
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
def test_arguments_that_are_no_numbers(pkg, cuda):
    import torch
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16, device=cuda), torch.zeros((32, 64), dtype=torch.bfloat16, device=cuda)
    for kw in (dict(limit=1e39), dict(limit=None), dict(limit="1"), dict(act=[]), dict(act=None)):
        with pytest.raises(pkg.GlmFlashError):
            pkg.gated_linear(x, w, w, **kw)

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


def product64(x, w):
    """x . w^T in 64 bits, 8192 k at a time."""
    return sum(x[:, k:k + 8192].double() @ w[:, k:k + 8192].double().t() for k in range(0, x.shape[1], 8192))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(2048, 65536, 512), (4096, 32768, 256), (512, 131072, 256), (30, 262144, 64), (3, 262144, 64)])
def test_16_bit_outputs_of_very_long_rows(pkg, cuda, rows, K, N):
    """Rows of one sign: sums of at most 8192 k, evenly spread, lose at most 2 * (1 + .. + 512) / 512 steps of 2^-23; the additions of sums and of parts of
    K half a step each; then one rounding.  One sum over all of K would lose K / 16 half steps, more than the rounding."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(rows)
    x = (1 + torch.rand((rows, K), generator=gen, device=cuda)).half()
    w, up = ((0.25 + torch.rand((N, K), generator=gen, device=cuda) / 4).mul_(4096 / K).half() for _ in range(2))
    tol = (2 * 515 + 0.5 * (K / 8192 + 16)) * 2.0 ** -23
    want, u = product64(x, w) / 4096, product64(x, up) / 4096
    x *= 2.0 ** -12                                           # (exact: x is 1 at least)
    got, both = pkg.linear(x, w), pkg.gated_linear(x, w, up, act="none")
    torch.cuda.synchronize()
    r = half_step(torch.float16)
    assert ((got.double() - want).abs() <= want * (r + tol)).all(), float(((got.double() - want) / want).mean())
    assert ((both.double() - want * u).abs() <= want * u * (r + 2 * tol + tol * tol)).all(), float(((both.double() - want * u) / (want * u)).mean())


# 16-bit outputs in more than one pass: gated pairs that keep act(gate) beside their sums, remainders of rows, outputs and K
@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(3001, 8264, 1000), (8192, 8320, 64), (8190, 8320, 72), (3000, 16500, 304), (2000, 8968, 1500), (200, 8968, 500), (17, 9000, 40)])
def test_16_bit_outputs_in_passes(pkg, cuda, rows, K, N):
    import torch
    b, h, f = torch.bfloat16, torch.float16, torch.float32
    gated(pkg, cuda, rows, K, N, b, f, "silu", 2.0, b, rows + K)
    gated(pkg, cuda, rows, K, N, h, None, "gelu", 0.0, h, rows + K + 1)
    plain(pkg, cuda, rows, K, N, b, f, "none", b, b, rows + K + 2, 0, True)
    plain(pkg, cuda, rows, K, N, h, None, "gelu_tanh", f, h, rows + K + 3, 3, False)


# Few outputs against the rows, so that rows lie along M: remainders of rows and outputs, one and several rounds of tiles, short and long K
FEW = [(20001, 1024, 288), (3000, 1024, 304), (4096, 4096, 288), (8191, 2048, 64), (8192, 2048, 72), (5001, 584, 88), (3001, 1000, 304), (2500, 2048, 296)]

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


def long_tol(x, w, passes=512):
    """How far a product with an fp32 output may be off.  Sums of at most 512 k: 32 groups of 16, for each at most two truncations by a step of 2^-23 of what has
    been added up in magnitude so far, the sum of |x w| over the sum's k; that is least tight where all of it comes first, 64 steps of the whole, and on
    rows whose magnitudes are spread evenly 2 * (1 + .. + 32) / 32 = 33.  Then an fp32 addition for each sum (half a step) and for each of at most 16 parts of K."""
    K = x.shape[1]
    groups = math.ceil(min(K, passes) / 16)
    # evenly spread rows: the first j of n groups hold at most (j + 2) / n of the whole
    first = 2 * sum(min(1.0, (j + 2) / groups) for j in range(1, groups + 1))
    return (first + 0.5 * (math.ceil(K / passes) + 16)) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t())


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
@pytest.mark.parametrize("rows", [9, 40, 2000])
def test_offsets_beyond_32_bits(pkg, cuda, rows):
    """Rows far apart: offsets of elements past 2^31 and strides past what 32 bits hold for a block of rows."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(rows)
    K, N, far = 72, 48, (1 << 32) // rows + 8 & -8
    x = torch.randn((rows, K), generator=gen, device=cuda).to(torch.bfloat16)
    w, w2 = ((torch.randn((N, K), generator=gen, device=cuda) / 8).to(torch.bfloat16) for _ in range(2))
    room = torch.empty(rows * far, dtype=torch.bfloat16, device=cuda)
    fx = room.as_strided((rows, K), (far, 1))
    fx.copy_(x)
    fres, out = (room.as_strided((rows, N), (far, 1), room.storage_offset() + 128 + 64 * i) for i in range(2))
    res = torch.randn((rows, N), generator=gen, device=cuda).to(torch.bfloat16)
    fres.copy_(res)
    want, want2 = pkg.linear(x, w, residual=res, act="gelu"), pkg.gated_linear(x, w, w2)
    pkg.linear(fx, w, residual=fres, act="gelu", out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(fx, x) and torch.equal(fres, res)
    pkg.linear(fx, w, residual=fres, act="gelu", out=fres)
    pkg.gated_linear(fx, w, w2, out=out)
    torch.cuda.synchronize()
    assert torch.equal(fres, want) and torch.equal(out, want2) and torch.equal(fx, x)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(300000, 64, 8), (300001, 72, 3), (70000, 8, 1)])
def test_many_rows(pkg, cuda, rows, K, N):
    import torch
    plain(pkg, cuda, rows, K, N, torch.bfloat16, torch.float32, "silu", torch.float32, torch.float32, rows, 0, True)
    gated(pkg, cuda, rows, K, N, torch.float16, None, "silu", 2.0, torch.float16, rows + 1)

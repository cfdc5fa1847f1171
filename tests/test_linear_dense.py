"""Dense products with their epilogue (linear, gated_linear) against the formula in 64 bits, and their refusals."""
import ctypes as C
import math
import struct

import numpy as np
import pytest

ARGS = struct.Struct("=12q8if3i")
FIELDS = ("x w w_up bias bias_up residual out x_stride w_stride w_up_stride residual_stride out_stride rows inner outer type bias_type residual_type "
          "out_type act limit pdl r0 r1").split()


def act64(v, act):
    import torch
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return torch.where(v < 0, torch.zeros_like(v), v) if act == "relu" else v


def wide(gen, rows, cols, pitch, dtype, scale=1.0):
    """rows x cols inside a buffer with `pitch` more elements a row, NaN there."""
    import torch
    buf = torch.full((rows, cols + pitch), float("nan"), dtype=dtype, device=gen.device)
    buf[:, :cols] = (torch.randn((rows, cols), generator=gen, device=gen.device) * scale).to(dtype)
    return buf[:, :cols]


def sum_tol(x, w, bias):
    """How far an fp32 sum of the products may be off, whatever its order: products of 16-bit values are exact in 32 bits; a tensor core adds 16 of
    them at a time with truncated alignment, at most one step of 2^-23 of the largest partial sum for each addition of such a group (2 per group), the sums
    of parts of K and the bias add 18 more."""
    K = x.shape[1]
    big = x.double().abs() @ w.double().abs().t()
    if bias is not None:
        big = big + bias.double().abs()
    return (2 * math.ceil(K / 16) + 18) * 2.0 ** -23 * big


SLOPE = 1.13                                            # no activation is steeper
# exp, erf, tanh and quotient: 8 half steps of a value of at most |v|
OWN = 8 * 2.0 ** -24


def half_step(t):
    import torch
    return torch.finfo(t).eps / 2


def check(got, want, tol, dtype):
    import torch
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    assert torch.equal(got.double()[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    # (below the smallest normal value of the output's type a step is that value's eps)
    tol = tol * (1 + half_step(dtype)) + want.abs() * half_step(dtype) + torch.finfo(dtype).smallest_normal * half_step(dtype)
    bad = ((got.double() - want).abs() > tol) & fine
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol)[fine].max()))


def guarded(rows, N, dtype, cuda, more=5):
    """An output inside a larger buffer, to see that nothing beside it is written."""
    import torch
    buf = torch.full((rows + 2, N + more), -7.0, dtype=dtype, device=cuda)
    return buf, buf[:rows, :N]


def untouched(buf, rows, N):
    return bool((buf[rows:] == -7).all()) and bool((buf[:, N:] == -7).all())


ROWS = [1, 2, 8, 9, 16, 17, 40, 64, 65, 129, 300]
SHAPES = [(1, 1), (7, 3), (8, 16), (40, 17), (64, 64), (72, 128), (100, 129), (513, 255), (1000, 257), (2048, 96)]


def plain_case(pkg, cuda, rows, K, N, dtype, bias_t, act, res_t, out_t, pitch, seed, inplace=False):
    import torch
    gen = torch.Generator(device=cuda).manual_seed(seed)
    x, w = wide(gen, rows, K, pitch, dtype), wide(gen, N, K, pitch, dtype, K ** -0.5)
    bias = None if bias_t is None else torch.randn(N, generator=gen, device=cuda).to(bias_t)
    buf, out = guarded(rows, N, out_t, cuda)
    residual = None
    if res_t is not None:
        residual = torch.randn((rows, N + 3), generator=gen, device=cuda).to(res_t)[:, :N]
        if inplace:
            out.copy_(residual)
    v = x.double() @ w.double().t()
    if bias is not None:
        v = v + bias.double()
    tol = sum_tol(x, w, bias) * SLOPE + OWN * v.abs()
    want = act64(v, act)
    if residual is not None:
        want = want + residual.double()
        tol = tol + want.abs() * 2.0 ** -24
    pkg.linear(x, w, out=out, bias=bias, act=act, residual=out if inplace and residual is not None else residual)
    torch.cuda.synchronize()
    check(out, want, tol, out_t)
    assert untouched(buf, rows, N)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_linear_sizes(pkg, cuda, rows):
    import torch
    for i, (K, N) in enumerate(SHAPES):
        for dtype in (torch.bfloat16, torch.float16):
            plain_case(pkg, cuda, rows, K, N, dtype, None, "none", None, torch.float32 if i % 2 else dtype, -K % 8 + 8 * (i % 2), 1000 * rows + i)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 13, 50, 200])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "relu"])
def test_linear_epilogues(pkg, cuda, rows, act):
    import torch
    b, h, f = torch.bfloat16, torch.float16, torch.float32
    for i, (dtype, bias_t, res_t, out_t) in enumerate([(b, f, None, b), (b, b, f, f), (h, h, h, h), (h, f, f, h), (b, None, b, b), (h, f, h, f), (b, f, f, b)]):
        plain_case(pkg, cuda, rows, 203, 333, dtype, bias_t, act, res_t, out_t, 5, 50 * rows + i)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 33, 260])
def test_linear_onto_its_residual(pkg, cuda, rows):
    import torch
    plain_case(pkg, cuda, rows, 512, 300, torch.bfloat16, torch.float32, "none", torch.float32, torch.float32, 0, rows, inplace=True)
    plain_case(pkg, cuda, rows, 512, 300, torch.float16, None, "gelu", torch.float16, torch.float16, 0, rows, inplace=True)


# many tiles, long K, more rows than a tile; the last ones in several rounds of a persistent grid
@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(1, 4096, 4096), (16, 8192, 1000), (16, 512, 20000), (30, 4096, 2000), (128, 8200, 520), (500, 2048, 1536), (1000, 1536, 2048),
                                      (2049, 776, 1537), (4096, 520, 4000), (8192, 256, 2304)])
def test_linear_large(pkg, cuda, rows, K, N):
    import torch
    plain_case(pkg, cuda, rows, K, N, torch.bfloat16, torch.float32, "none", torch.float32, torch.float32, 0, rows + K)
    plain_case(pkg, cuda, rows, K, N, torch.float16, None, "silu", torch.float16, torch.float16, 8, rows + K + 1)


# the residual under the output in pairs' first and later tiles, tiles of few rows without a cut of K, few outputs against the rows
@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(700, 1024, 2040), (6000, 520, 1030), (3000, 1024, 304), (1500, 1000, 300), (300, 512, 8192), (4096, 264, 97), (5000, 128, 1)])
def test_linear_tilings(pkg, cuda, rows, K, N):
    import torch
    plain_case(pkg, cuda, rows, K, N, torch.bfloat16, torch.bfloat16, "gelu_tanh", torch.bfloat16, torch.bfloat16, 0, rows + K, inplace=True)
    plain_case(pkg, cuda, rows, K, N, torch.float16, None, "none", torch.float32, torch.float16, 8, rows + K + 1)
    gated_case(pkg, cuda, rows, K, N, torch.bfloat16, torch.float32, "silu", 2.0, torch.bfloat16, 0, rows + K + 2)


def gated_case(pkg, cuda, rows, K, N, dtype, bias_t, act, limit, out_t, pitch, seed, only_up=False):
    import torch
    gen = torch.Generator(device=cuda).manual_seed(seed)
    x = wide(gen, rows, K, pitch, dtype)
    wg, wu = wide(gen, N, K, pitch, dtype, 2 * K ** -0.5), wide(gen, N, K, pitch + 8, dtype, 2 * K ** -0.5)
    bg = None if bias_t is None or only_up else torch.randn(N, generator=gen, device=cuda).to(bias_t)
    bu = None if bias_t is None else torch.randn(N, generator=gen, device=cuda).to(bias_t)
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    g = g if bg is None else g + bg.double()
    u = u if bu is None else u + bu.double()
    dg, du = sum_tol(x, wg, bg), sum_tol(x, wu, bu)
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    a = act64(g, act)
    tol = (dg * SLOPE + OWN * g.abs()) * (u.abs() + du) + a.abs() * du + (a * u).abs() * 2.0 ** -24
    buf, out = guarded(rows, N, out_t, cuda)
    pkg.gated_linear(x, wg, wu, out=out, bias_gate=bg, bias_up=bu, act=act, limit=limit)
    torch.cuda.synchronize()
    check(out, a * u, tol, out_t)
    assert untouched(buf, rows, N)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_gated_sizes(pkg, cuda, rows):
    import torch
    for i, (K, N) in enumerate(SHAPES):
        gated_case(pkg, cuda, rows, K, N, (torch.bfloat16, torch.float16)[i % 2], None if i % 3 else torch.float32, "silu", 1.5, torch.float32 if i % 4 == 3 else (torch.bfloat16, torch.float16)[i % 2],
                   -K % 8, 2000 * rows + i)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "relu"])
def test_gated_epilogues(pkg, cuda, rows, act):
    import torch
    b, h, f = torch.bfloat16, torch.float16, torch.float32
    for i, (dtype, bias_t, limit, out_t, only_up) in enumerate([(b, f, 0.0, b, False), (b, b, 10.0, f, False), (h, h, 0.5, h, True), (h, None, 2.0, h, False)]):
        gated_case(pkg, cuda, rows, 300, 200, dtype, bias_t, act, limit, out_t, 4, 70 * rows + i, only_up)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(1, 2048, 1536), (16, 4096, 512), (200, 4096, 512), (1000, 2048, 1536), (3000, 520, 1100), (8192, 256, 1000)])
def test_gated_large(pkg, cuda, rows, K, N):
    import torch
    gated_case(pkg, cuda, rows, K, N, torch.bfloat16, torch.float32, "silu", 10.0, torch.bfloat16, 0, rows + K)
    gated_case(pkg, cuda, rows, K, N, torch.float16, None, "gelu", 0.0, torch.float32, 8, rows + K + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 60, 400])
def test_infinities_and_nan_go_through(pkg, cuda, rows):
    """A row with an infinity or a NaN has what the formula gives; other rows are as without it, bit for bit; clamps do not hide a NaN."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(rows)
    x = torch.randn((rows, 96), generator=gen, device=cuda).to(torch.bfloat16)
    w, w2 = (torch.randn((70, 96), generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))
    bad = x.clone()
    bad[1, 5], bad[3, 95] = float("nan"), float("inf")
    for act in ("none", "relu"):
        clean, dirty = pkg.linear(x, w, act=act, out_dtype=torch.float32), pkg.linear(bad, w, act=act, out_dtype=torch.float32)
        torch.cuda.synchronize()
        want = act64(bad.double() @ w.double().t(), act)
        assert torch.isnan(dirty[1]).all()
        assert torch.equal(dirty[3].double(), want[3])                        # infinities (zeros behind relu)
        keep = [r for r in range(rows) if r not in (1, 3)]
        assert torch.equal(clean[keep], dirty[keep])
    y = pkg.gated_linear(bad, w, w2, limit=3.0, act="silu", out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert torch.isnan(y[1]).all()
    g, u = (bad[3].double() @ m.double().t() for m in (w, w2))
    want = act64(g.clamp(max=3.0).clamp(min=-1e30), "silu") * u.clamp(-3, 3)
    up = g > 0
    assert (y[3][up].double() - want[up]).abs().max() <= 1e-5
    # overflow of the output's type gives infinities
    big = pkg.linear(torch.full((rows, 64), 100.0, device=cuda, dtype=torch.float16), torch.full((8, 64), 100.0, device=cuda, dtype=torch.float16))
    torch.cuda.synchronize()
    assert torch.isinf(big).all()


@pytest.mark.gpu
def test_the_weights_may_come_from_the_kernel_in_front(pkg, cuda):
    """Launches that overlap their predecessor's end read nothing of it too early: weights, bias, residual and x are written right in front."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(1)
    for rows in (1, 16, 40, 300):
        x0, w0 = torch.randn((rows, 512), generator=gen, device=cuda), torch.randn((640, 512), generator=gen, device=cuda) / 20
        x, w = torch.zeros_like(x0, dtype=torch.bfloat16), torch.zeros_like(w0, dtype=torch.bfloat16)
        w2 = torch.zeros((512, 640), dtype=torch.bfloat16, device=cuda)
        outs = []
        for k in range(4):
            w.copy_(w0 * (k + 1))
            x.copy_(x0)
            y = pkg.linear(x, w)
            w2.copy_(w0.t() * (k + 1))
            outs.append((y, pkg.linear(y, w2, out_dtype=torch.float32), pkg.linear(y, w2, residual=y[:, :512], out_dtype=torch.float32)))
        torch.cuda.synchronize()
        for k, (y, z, zr) in enumerate(outs):
            wk, w2k = (w0 * (k + 1)).to(torch.bfloat16), (w0.t() * (k + 1)).to(torch.bfloat16)
            y2 = pkg.linear(x, wk.clone(), pdl=0)
            torch.cuda.synchronize()
            z2 = pkg.linear(y2, w2k.contiguous(), out_dtype=torch.float32, pdl=0)
            torch.cuda.synchronize()
            assert torch.equal(y, y2) and torch.equal(z, z2) and torch.equal(zr, z2 + y2[:, :512].float())


@pytest.mark.gpu
def test_two_streams_and_replays(pkg, cuda):
    """Calls share nothing: two streams at once, a captured graph replayed beside them."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(2)
    for rows in (4, 48, 260):
        x = [torch.randn((rows, 1024), generator=gen, device=cuda).to(torch.bfloat16) for _ in range(3)]
        w = [(torch.randn((1500, 1024), generator=gen, device=cuda) / 32).to(torch.bfloat16) for _ in range(3)]
        want = [pkg.linear(a, b) for a, b in zip(x, w)]
        torch.cuda.synchronize()
        st = [torch.cuda.Stream() for _ in range(3)]
        out = [torch.zeros_like(want[0]) for _ in range(3)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st[2]):
            for _ in range(3):
                pkg.linear(x[2], w[2], out=out[2])
        torch.cuda.synchronize()
        out[2].zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for i in range(2):
                pkg.linear(x[i], w[i], out=out[i], stream=st[i])
            with torch.cuda.stream(st[2]):
                graph.replay()
        made = pkg.linear(x[0], w[0], stream=st[0])
        torch.cuda.synchronize()
        for i in range(3):
            assert torch.equal(out[i], want[i])
        assert torch.equal(made, want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 12, 100, 700])
def test_dense_shared_expert_layer(pkg, synth, cuda, rows):
    """A layer of a real checkpoint: router with bias and scale, the routed experts, the dense shared expert added to their sum in place."""
    import torch
    H, I, E, S = 512, 256, 16, 5
    gen = torch.Generator(device=cuda).manual_seed(rows)
    bank = synth.device_bank(31, H, I, E, cuda)
    x = torch.randn((rows, H), generator=gen, device=cuda).to(torch.bfloat16)
    wr = (torch.randn((E, H), generator=gen, device=cuda) / H ** 0.5).to(torch.bfloat16)
    bias = torch.randn(E, generator=gen, device=cuda) * 0.1
    wg, wu = ((torch.randn((I, H), generator=gen, device=cuda) / H ** 0.5).to(torch.bfloat16) for _ in range(2))
    wd = (torch.randn((H, I), generator=gen, device=cuda) / I ** 0.5).to(torch.bfloat16)
    moe = pkg.Moe(pkg.make_config(H, I, E, S, max_rows=rows, shared_exl3=0))
    logits = torch.empty((rows, E), device=cuda)
    picks, weights = torch.empty((rows, S), dtype=torch.int32, device=cuda), torch.empty((rows, S), device=cuda)

    def layer(shared):
        pkg.route_by(x, wr, logits, picks, weights, bias=bias, scale=2.5)
        moe.run(bank, x, picks, weights, rows)
        if shared:
            mid = pkg.gated_linear(x, wg, wu, limit=10.0)
            pkg.linear(mid, wd, residual=moe.output[:rows], out=moe.output[:rows])
            return mid

    layer(False)
    torch.cuda.synchronize()
    routed = moe.output[:rows].clone()
    for _ in range(3):
        mid = layer(True)
    torch.cuda.synchronize()
    got = moe.output[:rows].clone()
    down = mid.double() @ wd.double().t()
    tol = sum_tol(mid, wd, None) + (down + routed.double()).abs() * 2.0 ** -23
    # (the routed experts' sum is the same bytes in every call)
    assert ((got.double() - (routed.double() + down)).abs() <= tol).all()
    assert int(moe.status.item()) == 0


def base_args(**kw):
    a = dict.fromkeys(FIELDS, 0)
    a.update(x=4096, w=8192, out=16384, x_stride=64, w_stride=64, out_stride=32, rows=4, inner=64, outer=32, type=2, out_type=2, limit=0.0)
    a.update(kw)
    return ARGS.pack(*(a[f] for f in FIELDS))


def test_refusals(pkg):
    """Bad arguments end in a message, in front of any launch (no GPU needed)."""
    L = pkg.lib()
    assert L.glmflash_linear_args_bytes() == ARGS.size
    for kw, word in [(dict(x=0), b"null"), (dict(w=0), b"null"), (dict(out=0), b"null"), (dict(rows=0), b"rows"), (dict(rows=-1), b"rows"), (dict(inner=0), b"inner"),
                     (dict(outer=0), b"outer"), (dict(rows=(1 << 30) + 1), b"2^30"), (dict(type=0, out_type=0), b"fp16 or bf16"), (dict(type=3), b"fp16 or bf16"),
                     (dict(bias=64, bias_type=1), b"bias"), (dict(residual=64, residual_stride=32, residual_type=1), b"residual"), (dict(out_type=1), b"output"),
                     (dict(act=5), b"activation"), (dict(act=-1), b"activation"), (dict(limit=1.0), b"limit"), (dict(bias_up=64), b"bias_up"),
                     (dict(w_up=64, w_up_stride=64, limit=-1.0), b"limit"), (dict(w_up=64, w_up_stride=64, limit=float("nan")), b"limit"),
                     (dict(w_up=64, w_up_stride=64, limit=float("inf")), b"limit"),
                     (dict(w_up=64, w_up_stride=64, residual=64, residual_stride=32, residual_type=2), b"residual"),
                     (dict(w_up=64, w_up_stride=56), b"inner"), (dict(w_up=64, w_up_stride=68), b"multiples of 8"), (dict(x_stride=56), b"inner"), (dict(w_stride=56), b"inner"),
                     (dict(x_stride=68), b"multiples of 8"), (dict(w_stride=65), b"multiples of 8"), (dict(out_stride=31), b"outer"),
                     (dict(residual=64, residual_stride=31, residual_type=2), b"outer"), (dict(x=4104), b"aligned"), (dict(w=8194), b"aligned"),
                     (dict(w_up=72, w_up_stride=64), b"aligned"), (dict(out=16385), b"aligned"), (dict(bias=66), b"aligned"),
                     (dict(residual=66, residual_stride=32), b"aligned"), (dict(r0=1), b"reserved"), (dict(r1=1), b"reserved"), (dict(x_stride=1 << 39), b"large")]:
        assert L.glmflash_linear(None, base_args(**kw), ARGS.size) == -1, kw
        assert word in L.glmflash_error(), (kw, L.glmflash_error())
    assert L.glmflash_linear(None, base_args(), ARGS.size - 8) == -1 and b"size" in L.glmflash_error()
    assert L.glmflash_linear(None, None, ARGS.size) == -1 and b"null" in L.glmflash_error()


@pytest.mark.gpu
def test_refusals_of_the_binding(pkg, cuda):
    import torch
    b = torch.bfloat16
    x, w = torch.zeros((4, 64), dtype=b, device=cuda), torch.zeros((32, 64), dtype=b, device=cuda)
    r = torch.zeros((4, 32), dtype=b, device=cuda)
    for args, kw in [((x.cpu(), w), {}), ((x, w.cpu()), {}), ((x, w.half()), {}), ((x.float(), w.float()), {}), ((x, w[:, :56]), {}), ((x[0], w), {}), ((x[:0], w), {}),
                     ((x[:, :0], w[:, :0]), {}), ((x, torch.zeros((64, 32), dtype=b, device=cuda).t()), {}), ((x[:, 1:], w[:, 1:]), {}),
                     ((x[:, :61].contiguous(), w[:, :61].contiguous()), {}), ((x, w), dict(out=r[:3])), ((x, w), dict(out=r.half())),
                     ((x, w), dict(out=r, out_dtype=torch.float32)), ((x, w), dict(out=r.t().contiguous().t())), ((x, w), dict(out=r[:1].expand(4, 32))),
                     ((x, w), dict(bias=torch.zeros(31, device=cuda))), ((x, w), dict(bias=torch.zeros(32, device=cuda, dtype=torch.float16))),
                     ((x, w), dict(residual=r[:3])), ((x, w), dict(residual=r.half())), ((x, w), dict(act="swish")), ((x, w), dict(out_dtype=torch.float16))]:
        with pytest.raises(pkg.GlmFlashError):
            pkg.linear(*args, **kw)
    for args, kw in [((x, w, w[:16]), {}), ((x, w, w.half()), {}), ((x, w, None), {}), ((x, w, w), dict(limit=-1.0)),
                     ((x, w, w), dict(bias_gate=torch.zeros(32, device=cuda), bias_up=torch.zeros(32, device=cuda, dtype=b)))]:
        with pytest.raises(pkg.GlmFlashError):
            pkg.gated_linear(*args, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N", [(300, 4096, 2000), (40, 4096, 1000)])
def test_status_word(pkg, cuda, rows, K, N):
    """A status word that is set makes long waits give up; the call returns, the context stays usable, and after a reset results are right."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(7)
    x, w = torch.randn((rows, K), generator=gen, device=cuda).to(torch.bfloat16), (torch.randn((N, K), generator=gen, device=cuda) / 64).to(torch.bfloat16)
    want = pkg.linear(x, w)
    torch.cuda.synchronize()
    status = pkg.linear_status()
    assert int(status.item()) == 0
    status.fill_(3)
    pkg.linear(x, w)
    torch.cuda.synchronize()
    assert int(status.item()) == 3
    pkg.linear_clear_status()
    got = pkg.linear(x, w)
    torch.cuda.synchronize()
    assert int(status.item()) == 0 and torch.equal(got, want)


@pytest.mark.gpu
def test_the_first_calls_may_be_captured(pkg, cuda):
    """In a process that has not called anything yet."""
    import os
    import subprocess
    import sys
    from conftest import ROOT
    code = f"""
import sys
sys.path.insert(0, {ROOT!r})
import torch
import __graft_entry__ as entry
pkg = entry.load_package()
x = torch.randn(300, 512, device='cuda').to(torch.bfloat16)
w = torch.randn(256, 512, device='cuda').to(torch.bfloat16)
bias = torch.randn(256, device='cuda')
outs = [torch.zeros(r, 256, dtype=torch.bfloat16, device='cuda') for r in (1, 40, 300)]
gated = torch.zeros(300, 256, dtype=torch.bfloat16, device='cuda')
logits = torch.zeros(300, 256, device='cuda')
picks, weights = torch.zeros(300, 5, dtype=torch.int32, device='cuda'), torch.zeros(300, 5, device='cuda')
def calls():
    for o in outs:
        pkg.linear(x[:o.shape[0]], w, out=o)
    pkg.gated_linear(x, w, w, out=gated)
    pkg.route_by(x, w, logits, picks, weights, bias=bias)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
graph.replay()
torch.cuda.synchronize()
kept = [t.clone() for t in outs + [gated, logits, picks, weights]]
calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(kept, outs + [gated, logits, picks, weights]))
assert float(outs[2].float().abs().sum()) > 0
print('captured')
"""
    env = dict(os.environ)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_arguments_that_are_no_numbers(pkg, cuda):
    import torch
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16, device=cuda), torch.zeros((32, 64), dtype=torch.bfloat16, device=cuda)
    for kw in (dict(limit=1e39), dict(limit=None), dict(limit="1"), dict(act=[]), dict(act=None)):
        with pytest.raises(pkg.GlmFlashError):
            pkg.gated_linear(x, w, w, **kw)

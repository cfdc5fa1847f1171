"""Selection of experts by a rule (topk_by, route_by) against the definition in 64 bits, and its refusals."""
import ctypes as C
import struct

import numpy as np
import pytest

RULE = struct.Struct("=5if2i")
# Weights: scores by a 32-bit exponential (2 units in the last place, 4 half steps), quotient and scale (3 half steps), a softmax's sum (37 terms one
# after another at most, each with its exponential's error) and the sum of the chosen (31 terms): 4 + 3 + 37 + 4 + 31 half steps of 2^-24.
WTOL = 80 * 2.0 ** -24


def table(logits, bias, k, scores="sigmoid", groups=1, keep=None, group_score="max", renorm=True, scale=1.0):
    """The definition, in 64 bits."""
    rows, E = logits.shape
    keep = groups if keep is None else keep
    l = logits.astype(np.float64)
    l[np.isnan(l)] = -np.inf
    with np.errstate(all="ignore"):
        if scores == "sigmoid":
            s = 1 / (1 + np.exp(-l))
        else:
            top = l.max(1, keepdims=True)
            e = np.where(l == top, 1.0, np.exp(l - top))
            e[np.isneginf(l)] = 0
            s = np.where(e.sum(1, keepdims=True) > 0, e / e.sum(1, keepdims=True), 0)
    c = l.copy()
    if bias is not None:
        b = bias.astype(np.float64)
        c = np.where(np.isnan(b), -np.inf, s + b)
    n = E // groups
    open_ = np.ones((rows, E), bool)
    if keep < groups:
        v = (c if bias is not None or group_score == "max" else s).reshape(rows, groups, n)
        v = -np.sort(-v, 2)
        v = v[:, :, 0] if group_score == "max" or n == 1 else v[:, :, 0] + v[:, :, 1]
        order = np.argsort(-v, 1, kind="stable")[:, :keep]
        open_[:] = False
        for r in range(rows):
            for g in order[r]:
                open_[r, g * n:(g + 1) * n] = True
    picks = np.empty((rows, k + 1), np.int32)
    w = np.ones((rows, k + 1))
    for r in range(rows):
        ids = np.flatnonzero(open_[r])
        picks[r, :k] = ids[np.argsort(-c[r, ids], kind="stable")][:k]
        sc = s[r, picks[r, :k]]
        if renorm:
            sc = sc / sc.sum() if sc.sum() > 0 else 0 * sc
        w[r, :k] = sc * scale
    picks[:, k] = E
    return picks, w


def make_logits(rows, E, seed):
    g = np.random.default_rng(seed)
    logits = g.standard_normal((rows, E)).astype(np.float32)
    bias = (g.standard_normal(E) * 0.1).astype(np.float32)
    special = [lambda r: r.fill(0.25),                                       # all tied
               lambda r: r.fill(-np.inf),                                    # nothing left
               lambda r: r.fill(np.nan),
               lambda r: r.__setitem__(slice(0, None, 2), np.nan),
               lambda r: r.__setitem__(slice(0, None, 3), np.inf),
               lambda r: r.__setitem__(slice(1, None), -np.inf),             # one left
               lambda r: r.fill(-80.0),                                      # scores near the end of the range
               lambda r: r.__setitem__(0, np.finfo(np.float32).min),
               lambda r: r.__iadd__(np.float32(-30)),
               lambda r: np.copyto(r, np.nextafter(np.float32(0.5), np.float32(1)) + np.float32(2.0 ** -24) * (np.arange(E) % 5).astype(np.float32)),   # last places
               lambda r: r.__setitem__(0, np.finfo(np.float32).max)]
    for i, f in enumerate(special):
        if 2 * i + 1 < rows:
            f(logits[2 * i + 1])
    return logits, bias


def run(pkg, cuda, logits, bias, k, pad=0, **rule):
    import torch
    rows, E = logits.shape
    buf = torch.full((rows, E + pad), float("nan"), device=cuda)
    buf[:, :E] = torch.from_numpy(logits).to(cuda)
    picks = torch.full((rows + 1, k + 1), -7, dtype=torch.int32, device=cuda)
    weights = torch.full((rows + 1, k + 1), -7.0, device=cuda)
    b = None if bias is None else torch.from_numpy(bias).to(cuda)
    pkg.topk_by(buf[:, :E], picks[:rows], weights[:rows], bias=b, **rule)
    torch.cuda.synchronize()
    assert (picks[rows] == -7).all() and (weights[rows] == -7).all()        # rows behind the last: as they were
    return picks[:rows].cpu().numpy(), weights[:rows].cpu().numpy()


CASES = [
    # rows, experts, k, rule
    (1, 1, 1, {}),
    (1, 64, 4, {}),
    (3, 5, 5, dict(scores="softmax")),
    (40, 64, 4, dict(scores="softmax", renorm=False)),
    (40, 288, 8, dict(scale=2.5)),
    (33, 288, 8, dict(groups=8, keep_groups=4, group_score="top2", scale=2.5)),
    (33, 256, 8, dict(groups=8, keep_groups=4, group_score="top2")),
    (33, 160, 6, dict(groups=8, keep_groups=3, scores="softmax", renorm=False, scale=16.0)),
    (29, 32, 3, dict(groups=32, keep_groups=3, group_score="top2")),         # groups of one
    (29, 60, 5, dict(groups=20, keep_groups=2, group_score="max")),
    (25, 1024, 31, {}),
    (25, 1024, 31, dict(groups=32, keep_groups=1, scores="softmax")),
    (25, 1000, 16, dict(scores="softmax", groups=4, keep_groups=2, group_score="top2")),
    (27, 31, 31, {}),
    (27, 33, 8, dict(groups=3, keep_groups=2)),
    (25, 96, 8, dict(groups=3, keep_groups=1, group_score="top2", renorm=False)),
    (700, 65, 4, dict(scores="softmax")),
]


@pytest.mark.gpu
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("rows,E,k,rule", CASES)
def test_topk_by_equals_the_definition(pkg, cuda, rows, E, k, rule, biased):
    logits, bias = make_logits(rows, E, 100 * rows + E)
    r = dict(rule)
    keep = r.pop("keep_groups", None)
    want_p, want_w = table(logits, bias if biased else None, k, keep=keep, **r)
    got_p, got_w = run(pkg, cuda, logits, bias if biased else None, k, **rule)
    assert np.array_equal(got_p, want_p)
    assert np.isfinite(got_w).all()
    # (scores below the smallest normal value of 32 bits have fewer bits)
    assert (np.abs(got_w - want_w) <= WTOL * np.abs(want_w) + rule.get("scale", 1.0) * 2.0 ** -126).all()


@pytest.mark.gpu
def test_bias_closes_experts(pkg, cuda):
    """A bias of -inf (or the lowest value, or NaN) closes an expert while others are open; where it leaves too few, the lowest ids follow."""
    logits, _ = make_logits(30, 64, 5)
    for shut in (-np.inf, np.finfo(np.float32).min, np.nan):
        for left in (10, 3, 0):
            bias = np.full(64, shut, np.float32)
            bias[5:5 + left] = 0.01
            want_p, want_w = table(logits, bias, 4, scores="softmax")
            got_p, got_w = run(pkg, cuda, logits, bias, 4, scores="softmax")
            assert np.array_equal(got_p, want_p)
            assert (np.abs(got_w - want_w) <= WTOL * np.abs(want_w) + 2.0 ** -126).all()
    # an open expert by +inf comes first
    bias = np.zeros(64, np.float32)
    bias[[7, 9]] = np.inf
    want_p, want_w = table(logits, bias, 4)
    got_p, _ = run(pkg, cuda, logits, bias, 4)
    assert np.array_equal(got_p, want_p) and (got_p[:, :2] == [7, 9]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_order_of_neighbouring_values(pkg, cuda, scores, group_score):
    """Scores and sums that differ in bits which 32 bits do not hold are ordered by them, ties by the id."""
    g = np.random.default_rng(9)
    rows, E = 200, 96
    base = g.standard_normal((rows, 1)).astype(np.float32)
    logits = (base + g.integers(0, 4, (rows, E)).astype(np.float32) * np.float32(2.0 ** -22)).astype(np.float32)
    bias = (np.float32(0.125) + g.integers(-2, 3, E).astype(np.float32) * np.float32(2.0 ** -27)).astype(np.float32)
    for b in (None, bias):
        want_p, _ = table(logits, b, 8, scores, 6, 3, group_score)
        got_p, _ = run(pkg, cuda, logits, b, 8, scores=scores, groups=6, keep_groups=3, group_score=group_score)
        assert np.array_equal(got_p, want_p)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("biased", [False, True])
def test_small_scores_keep_their_weight(pkg, cuda, scores, biased):
    """Chosen scores many orders of magnitude apart, down to what 32 bits do not hold: renormalised weights as in 64 bits."""
    logits = np.full((6, 40), -400.0, np.float32)
    for r, (a, step) in enumerate([(-30.0, 20.0), (5.0, 40.0), (-87.0, 1.0), (-100.0, 3.0), (-300.0, 5.0), (-60.0, 14.0)]):
        logits[r, 3:9] = a - step * np.arange(6, dtype=np.float32)
    bias = np.full(40, -1.0, np.float32)
    bias[3:9] = [0.5, 0.4, 0.3, 0.2, 0.1, 0.0]                                # (the order of the logits, whatever the scores)
    b = bias if biased else None
    want_p, want_w = table(logits, b, 6, scores, scale=2.5)
    got_p, got_w = run(pkg, cuda, logits, b, 6, scores=scores, scale=2.5)
    assert np.array_equal(got_p, want_p)
    assert (np.abs(got_w - want_w) <= WTOL * np.abs(want_w) + 2.5 * 2.0 ** -126).all()


@pytest.mark.gpu
def test_many_ties_and_closed_experts(pkg, cuda):
    """More candidates than lanes: ties in every row, with and without a bias, experts left open on one lane only, groups with few experts left."""
    g = np.random.default_rng(3)
    logits = g.integers(0, 2, (64, 288)).astype(np.float32)
    closed = np.full(288, -np.inf, np.float32)
    closed[0::32] = g.standard_normal(9).astype(np.float32) * np.float32(0.1)
    for b in (None, np.zeros(288, np.float32), np.full(288, 0.125, np.float32), closed):
        for rule in (dict(), dict(groups=8, keep_groups=1), dict(groups=32, keep_groups=2, group_score="top2"), dict(scores="softmax", groups=4, keep_groups=3, group_score="top2")):
            r = dict(rule)
            want_p, _ = table(logits, b, 8, keep=r.pop("keep_groups", None), **r)
            got_p, got_w = run(pkg, cuda, logits, b, 8, **rule)
            assert np.array_equal(got_p, want_p), (b is None, rule)
            assert np.isfinite(got_w).all()


@pytest.mark.gpu
def test_plain_rule_is_topk(pkg, cuda):
    """Sigmoid scores without bias and groups: the table of `topk`."""
    import torch
    logits = torch.randn((500, 64), generator=torch.Generator(device=cuda).manual_seed(4), device=cuda)
    picks, weights = torch.empty((500, 5), dtype=torch.int32, device=cuda), torch.empty((500, 5), device=cuda)
    p2, w2 = torch.empty_like(picks), torch.empty_like(weights)
    pkg.topk(logits, picks, weights)
    pkg.topk_by(logits, p2, w2)
    torch.cuda.synchronize()
    assert torch.equal(picks, p2)
    assert (weights - w2).abs().max() <= 2 * WTOL


@pytest.mark.gpu
def test_strided_logits_a_stream_and_replay(pkg, cuda):
    import torch
    logits, bias = make_logits(50, 288, 77)
    rule = dict(groups=8, keep_groups=4, group_score="top2", scale=2.5)
    a = run(pkg, cuda, logits, bias, 8, **rule)
    b = run(pkg, cuda, logits, bias, 8, pad=13, **rule)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    ld, bd = torch.from_numpy(logits).to(cuda), torch.from_numpy(bias).to(cuda)
    picks, weights = torch.zeros((50, 9), dtype=torch.int32, device=cuda), torch.zeros((50, 9), device=cuda)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    pkg.topk_by(ld, picks, weights, bias=bd, stream=st, **rule)
    st.synchronize()
    assert np.array_equal(picks.cpu().numpy(), a[0])
    with torch.cuda.graph(graph, stream=st):
        pkg.topk_by(ld, picks, weights, bias=bd, **rule)
    other, _ = make_logits(50, 288, 78)
    ld.copy_(torch.from_numpy(other))
    graph.replay()
    torch.cuda.synchronize()
    want_p, _ = table(other, bias, 8, "sigmoid", 8, 4, "top2", True, 2.5)
    assert np.array_equal(picks.cpu().numpy(), want_p)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,H,E,k,rule", [
    (1, 2048, 64, 4, dict(scale=2.5)), (16, 4096, 288, 8, dict(groups=8, keep_groups=4, group_score="top2")), (300, 256, 65, 3, dict(scores="softmax")),
    (2500, 512, 128, 8, dict(scores="softmax", renorm=False)), (5, 264, 1024, 31, {}), (17, 8, 1, 1, {}), (4000, 128, 32, 4, dict(groups=4, keep_groups=2))])
def test_route_by_is_logits_and_selection(pkg, cuda, rows, H, E, k, rule):
    """The bytes of the dense product in fp32 followed by topk_by on the same rows."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(rows)
    x = torch.randn((rows, H + 8), generator=gen, device=cuda).to(torch.bfloat16)[:, :H]
    wr = (torch.randn((E, H), generator=gen, device=cuda) / H ** 0.5).to(torch.bfloat16)
    bias = torch.randn(E, generator=gen, device=cuda) * 0.1
    if rows > 3:
        x[1], x[2, 0], x[3, 3] = 0, float("nan"), float("inf")
    out = [torch.full((rows, E), 9.0, device=cuda), torch.full((rows, k + 1), -7, dtype=torch.int32, device=cuda), torch.zeros((rows, k + 1), device=cuda)]
    pkg.route_by(x, wr, *out, bias=bias, **rule)
    l2 = pkg.linear(x, wr, out_dtype=torch.float32)
    p2, w2 = torch.empty_like(out[1]), torch.empty_like(out[2])
    pkg.topk_by(l2, p2, w2, bias=bias, **rule)
    torch.cuda.synchronize()
    assert torch.equal(l2.view(torch.int32), out[0].view(torch.int32))
    assert torch.equal(p2, out[1]) and torch.equal(w2.view(torch.int32), out[2].view(torch.int32))
    r = dict(rule)
    want_p, want_w = table(l2.cpu().numpy(), bias.cpu().numpy(), k, keep=r.pop("keep_groups", None), **r)
    assert np.array_equal(p2.cpu().numpy(), want_p)
    assert (np.abs(w2.cpu().numpy() - want_w) <= WTOL * np.abs(want_w) + 4 * 2.0 ** -126).all()

@pytest.mark.gpu
@pytest.mark.parametrize("pdl", [0, 1])
@pytest.mark.parametrize("rows,H,E,k,biased,rule", [
    (1, 2048, 64, 4, True, {}), (3, 8, 1, 1, True, {}), (8, 40, 16, 3, False, dict(scores="softmax", scale=1.5)), (9, 264, 17, 8, True, dict(renorm=False)),
    (16, 2048, 64, 8, True, dict(groups=8, keep_groups=3, group_score="top2")), (7, 4096, 128, 31, True, dict(scores="softmax")),
    (13, 1000, 100, 5, False, dict(groups=4, keep_groups=2, group_score="top2")), (8, 512, 33, 8, True, dict(groups=3, keep_groups=2)),
    (16, 136, 129, 4, True, {}), (5, 2048, 127, 6, True, dict(scores="softmax", groups=1))])
def test_route_by_of_few_rows(pkg, cuda, rows, H, E, k, biased, rule, pdl):
    """The same for few rows, whose experts share a cluster: bias and activations written by the kernels just in front, ties, rows of NaN and infinities."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(rows + E)
    x = torch.randn((rows, H + 8), generator=gen, device=cuda).to(torch.bfloat16)[:, :H]
    wr = (torch.randn((E, H), generator=gen, device=cuda) / H ** 0.5).to(torch.bfloat16)
    source = torch.randn(E, generator=gen, device=cuda) * 0.1
    bias = torch.full((E,), 5.0, device=cuda) if biased else None
    if E > 5:
        wr[E - 1], wr[2] = wr[0], wr[0]                      # three logits alike
        source[E - 1], source[2] = source[0], source[0]
    wide = [torch.full((rows, E), 9.0, device=cuda), torch.full((rows + 1, k + 1), -7, dtype=torch.int32, device=cuda), torch.full((rows + 1, k + 1), -7.0, device=cuda)]
    out = [wide[0], wide[1][:rows], wide[2][:rows]]
    fresh = x.clone()
    if rows > 3:
        fresh[1], fresh[2, 0], fresh[3, 3] = 0, float("nan"), float("inf")
    torch.cuda.synchronize()
    for _ in range(3):
        x.copy_(fresh)
        if biased:
            bias.copy_(source)
        pkg.route_by(x, wr, *out, bias=bias, pdl=pdl, **rule)
        if biased:
            bias.fill_(7.0)
        x.zero_()
    x.copy_(fresh)
    l2 = pkg.linear(x, wr, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert torch.equal(l2.view(torch.int32), out[0].view(torch.int32))
    r = dict(rule)
    want_p, want_w = table(l2.cpu().numpy(), source.cpu().numpy() if biased else None, k, keep=r.pop("keep_groups", None), **r)
    assert np.array_equal(out[1].cpu().numpy(), want_p)
    assert (np.abs(out[2].cpu().numpy() - want_w) <= WTOL * np.abs(want_w) + 4 * 2.0 ** -126).all()
    assert (wide[1][rows] == -7).all() and (wide[2][rows] == -7.0).all()          # rows behind the last, left as they were



def test_refusals(pkg):
    """Bad arguments end in a message, in front of any launch (no GPU needed)."""
    L = pkg.lib()
    p = C.c_void_p(4096)

    def call(E=64, k=4, rows=3, stride=None, scores=0, groups=1, keep=1, group_score=0, scale=1.0, res=0, size=RULE.size, null=None, logits=p):
        rule = RULE.pack(scores, groups, keep, group_score, 1, scale, res, 0)
        args = [logits, E if stride is None else stride, None, rows, E, k, rule, size, p, p, 0]
        if null is not None:
            args[null] = None
        return L.glmflash_topk_by(None, *args), L.glmflash_error()

    for kw, word in [(dict(E=0), b"experts"), (dict(E=1025), b"experts"), (dict(k=0), b"topk"), (dict(k=32), b"topk"), (dict(E=8, k=9), b"topk"),
                     (dict(rows=0), b"rows"), (dict(rows=-1), b"rows"), (dict(stride=63), b"logits_stride"), (dict(scores=2), b"scores"),
                     (dict(groups=0), b"groups"), (dict(groups=33, E=66), b"groups"), (dict(groups=3), b"groups"), (dict(groups=4, keep=5), b"keep_groups"),
                     (dict(groups=4, keep=0), b"keep_groups"), (dict(groups=32, keep=1, k=3), b"topk"), (dict(group_score=2), b"group_score"),
                     (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(res=1), b"reserved"), (dict(size=28), b"size"),
                     (dict(logits=C.c_void_p(4098)), b"aligned"), (dict(null=0), b"null"), (dict(null=6), b"null"), (dict(null=8), b"null"), (dict(null=9), b"null")]:
        rc, msg = call(**kw)
        assert rc == -1 and word in msg, (kw, msg)
    rule = RULE.pack(0, 1, 1, 0, 1, 1.0, 0, 0)

    def route(x=p, hidden=64, stride=64, rows=2):
        return L.glmflash_route_by(None, x, stride, p, None, rows, hidden, 64, 4, rule, RULE.size, p, p, p, 0), L.glmflash_error()
    for kw, word in [(dict(x=None), b"null"), (dict(hidden=60), b"hidden"), (dict(stride=56), b"x_stride"), (dict(stride=68), b"x_stride"),
                     (dict(x=C.c_void_p(4104)), b"aligned"), (dict(rows=0), b"rows")]:
        rc, msg = route(**kw)
        assert rc == -1 and word in msg, (kw, msg)
    assert L.glmflash_topk_rule_bytes() == RULE.size


@pytest.mark.gpu
def test_refusals_of_the_binding(pkg, cuda):
    import torch
    l, p, w = torch.zeros((4, 64), device=cuda), torch.zeros((4, 5), dtype=torch.int32, device=cuda), torch.zeros((4, 5), device=cuda)
    b = torch.zeros(64, device=cuda)
    for args, kw in [((l.cpu(), p, w), {}), ((l.half(), p, w), {}), ((l, p.long(), w), {}), ((l, p, w[:3]), {}), ((l, p[:, :4], w[:, :4]), {}),
                     ((l.t(), p, w), {}), ((l[0], p, w), {}), ((l, p, w), dict(bias=b[:63])), ((l, p, w), dict(bias=b.double())),
                     ((l, p, w), dict(scores="tanh")), ((l, p, w), dict(group_score="mean")), ((l, p, w), dict(bias=torch.zeros(128, device=cuda)[::2])),
                     ((l[:1].expand(4, 64), p, w), {})]:
        with pytest.raises(pkg.GlmFlashError):
            pkg.topk_by(*args, **kw)
    x, wr = torch.zeros((4, 64), dtype=torch.bfloat16, device=cuda), torch.zeros((64, 64), dtype=torch.bfloat16, device=cuda)
    for xx, ww in [(x.float(), wr), (x, wr[:63]), (x[:3], wr), (x[:, :56], wr), (x.cpu(), wr), (x, wr[:, ::2])]:
        with pytest.raises(pkg.GlmFlashError):
            pkg.route_by(xx, ww, l, p, w)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,per,keep", [(2, 2, 1), (8, 2, 3), (3, 5, 1), (8, 8, 4), (8, 36, 4), (32, 32, 5)])
def test_sums_of_two_that_cancel(pkg, cuda, scores, groups, per, keep):
    """Biases that open one expert of a group and close the others by finite values: a group's two largest c cancel, and what decides between the
    sums is far below the last place of their terms in 32 bits."""
    g = np.random.default_rng(groups * per)
    E, k = groups * per, min(4, keep * per)
    opener = g.integers(0, per, groups) + per * np.arange(groups)
    logits = g.standard_normal((1500, E)).astype(np.float32)
    if (groups, per) == (2, 2):
        opener = np.array([0, 2])
        logits[0] = [0.6270455, -1.6190524, -0.58814746, -0.1600341]
    for size in (30.0, 1e2, 1e3, 1e4, 1e5, 1e6, 3e38):
        bias = np.full(E, -size, np.float32)
        bias[opener] = size
        for b in (bias, np.where(np.arange(E) // per % 2 == 0, bias, -bias)):        # (and groups that all but one are open in)
            want_p, want_w = table(logits, b, k, scores, groups, keep, "top2")
            got_p, got_w = run(pkg, cuda, logits, b, k, scores=scores, groups=groups, keep_groups=keep, group_score="top2")
            assert np.array_equal(got_p, want_p), (size, int((got_p != want_p).any(1).sum()))
            assert (np.abs(got_w - want_w) <= WTOL * np.abs(want_w) + 2.0 ** -126).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shut", [-np.inf, np.nan])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_bias_closes_experts_of_groups(pkg, cuda, group_score, shut):
    """As the formula has it: a group that stays may hold closed experts, which are chosen where it has too few open ones; as a sum of two a group with one
    open expert counts like a closed one."""
    logits, _ = make_logits(30, 24, 6)
    g = np.random.default_rng(8)
    for open_ in ([0, 1, 2, 12, 13, 14], [5, 6, 18], [7], [1, 8, 15, 22], [], list(range(18))):
        bias = np.full(24, shut, np.float32)
        bias[open_] = g.standard_normal(len(open_)).astype(np.float32) * np.float32(0.1)
        for groups, keep, k in ((2, 1, 4), (4, 1, 2), (4, 2, 8), (4, 3, 3), (12, 5, 6)):
            for scores in ("sigmoid", "softmax"):
                want_p, want_w = table(logits, bias, k, scores, groups, keep, group_score)
                got_p, got_w = run(pkg, cuda, logits, bias, k, scores=scores, groups=groups, keep_groups=keep, group_score=group_score)
                assert np.array_equal(got_p, want_p), (open_, groups, keep, scores)
                assert (np.abs(got_w - want_w) <= WTOL * np.abs(want_w) + 2.0 ** -126).all()


@pytest.mark.gpu
def test_rules_are_read_at_each_call(pkg, cuda):
    """A rule's numbers may be any objects that stand for one: what they hold at the call counts, not which object it is.  Others end in the
    library's error."""
    import torch
    logits, bias = make_logits(20, 64, 12)
    ld, bd = torch.from_numpy(logits).to(cuda), torch.from_numpy(bias).to(cuda)
    picks, weights = torch.empty((20, 5), dtype=torch.int32, device=cuda), torch.empty((20, 5), device=cuda)
    scale, keep = torch.tensor(2.5), torch.tensor(2)
    for s, n in ((2.5, 2), (1.25, 3)):
        scale.fill_(s)
        keep.fill_(n)
        pkg.topk_by(ld, picks, weights, bias=bd, groups=np.int64(4), keep_groups=keep, scale=scale)
        want_p, want_w = table(logits, bias, 4, groups=4, keep=n, scale=s)
        assert np.array_equal(picks.cpu().numpy(), want_p)
        assert (np.abs(weights.cpu().numpy() - want_w) <= WTOL * np.abs(want_w) + 4 * 2.0 ** -126).all()
    pkg.topk_by(ld, picks, weights, groups=2)
    for kw in (dict(scale=1e39), dict(scale=None), dict(scale="2"), dict(groups=2.0), dict(groups=1 << 40), dict(keep_groups="1"), dict(scores=[]), dict(scores=None),
               dict(group_score={})):
        with pytest.raises(pkg.GlmFlashError):
            pkg.topk_by(ld, picks, weights, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,H,E", [(1, 2048, 64), (16, 4096, 128), (9, 4096, 288), (40, 4096, 64), (600, 4096, 288), (4096, 4096, 288), (4096, 8192, 64)])
def test_logits_of_the_router_in_64_bits(pkg, cuda, rows, H, E):
    """Ordinary bf16 rows: the logits against the product in 64 bits, by the error of fp32 sums of at most 512 k (test_linear_exact.py has the bound)."""
    import torch
    from test_linear_exact import long_tol
    gen = torch.Generator(device=cuda).manual_seed(rows + H)
    x = torch.randn((rows, H), generator=gen, device=cuda).to(torch.bfloat16)
    wr = (torch.randn((E, H), generator=gen, device=cuda) / H ** 0.5).to(torch.bfloat16)
    logits, picks, weights = torch.empty((rows, E), device=cuda), torch.empty((rows, 5), dtype=torch.int32, device=cuda), torch.empty((rows, 5), device=cuda)
    pkg.route_by(x, wr, logits, picks, weights)
    torch.cuda.synchronize()
    assert ((logits.double() - x.double() @ wr.double().t()).abs() <= long_tol(x, wr)).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(pkg, cuda):
    """Logits of rows that are far apart, rows of the router product too."""
    import torch
    rows, E, far = 20, 96, (1 << 32) // 20
    logits, bias = make_logits(rows, E, 3)
    room = torch.empty(rows * far, device=cuda)
    fl = room.as_strided((rows, E), (far, 1))
    fl.copy_(torch.from_numpy(logits))
    picks, weights, b = torch.empty((rows, 5), dtype=torch.int32, device=cuda), torch.empty((rows, 5), device=cuda), torch.from_numpy(bias).to(cuda)
    pkg.topk_by(fl, picks, weights, bias=b)
    torch.cuda.synchronize()
    assert np.array_equal(picks.cpu().numpy(), table(logits, bias, 4)[0])
    gen = torch.Generator(device=cuda).manual_seed(3)
    x, wr = torch.randn((rows, 256), generator=gen, device=cuda).to(torch.bfloat16), (torch.randn((E, 256), generator=gen, device=cuda) / 16).to(torch.bfloat16)
    step = far * 2 // 8 * 8
    for n in (rows, 7):
        fx = room.view(torch.bfloat16).as_strided((n, 256), (step, 1))
        fx.copy_(x[:n])
        out, want = (([torch.empty((n, E), device=cuda), torch.empty((n, 5), dtype=torch.int32, device=cuda), torch.empty((n, 5), device=cuda)]) for _ in range(2))
        pkg.route_by(fx, wr, *out, bias=b)
        pkg.route_by(x[:n], wr, *want, bias=b)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))

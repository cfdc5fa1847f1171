"""Operators next to the expert path, measured: selection of experts from router logits by a rule (topk_by), the router product and the
selection in one call (route_by), the dense product with bias, activation and residual (linear), and its gated form (gated_linear).

A case is a dict of plain values:
  kind    "select"  router logits in hand -> routing table (topk_by)
          "route"   rows in hand -> logits and routing table (route_by)
          "linear"  out = act(x . w^T + bias) + residual
          "gated"   out = act(min(x . wg^T + bg, limit)) * clamp(x . wu^T + bu, -limit, limit)
  rows    tokens of the call
  select, route: experts, topk, scores ("sigmoid" or "softmax"), bias (added to the scores for the choice alone), groups, keep (groups
          that stay), group_score ("max" or "top2"), renorm, scale; route: hidden
  linear, gated: inner, outer (sizes of the product), dtype of x and the weights, bias, act, pitch (elements that a row of x and of the
          weights takes beyond `inner`), linear: residual and out ("none", "same" type as x, or "float32"), gated: limit (0: none)
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
ACTS = ("none", "silu", "gelu", "gelu_tanh", "relu")
MOST_FLOPS = 2 * 8192 * 4096 * 4096                              # the largest listed case
MOST_BYTES = 2 * (3 * 8192 * 4096 + 4096 * 4096)


def _select(name, rows, experts, topk, **kw):
    c = dict(name=name, kind="select", rows=rows, experts=experts, topk=topk, scores="sigmoid", bias=True, groups=1, keep=1, group_score="max",
             renorm=True, scale=1.0)
    c.update(kw)
    return c


def _linear(name, rows, inner, outer, **kw):
    c = dict(name=name, kind="linear", rows=rows, inner=inner, outer=outer, dtype="bfloat16", bias=False, act="none", residual="none", out="same",
             pitch=0)
    c.update(kw)
    return c


def _gated(name, rows, inner, outer, **kw):
    c = dict(name=name, kind="gated", rows=rows, inner=inner, outer=outer, dtype="bfloat16", bias=False, act="silu", limit=10.0, pitch=0)
    c.update(kw)
    return c


def listed():
    return [
        # one token of the larger model: 288 experts, top-8, scores with a balance bias, weights scaled
        _select("select-1", 1, 288, 8, scale=2.5),
        # a prompt of the benchmark's bank, softmax scores
        _select("select-4096-softmax", 4096, 64, 4, scores="softmax", bias=False),
        # the largest chunk with experts in groups, of which half stay
        _select("select-8192-groups", 8192, 288, 8, groups=8, keep=4, group_score="top2", scale=2.5),
        # one token of the benchmark's bank from its row, the smallest call that a decode loop makes
        _select("route-1", 1, 64, 4, kind="route", hidden=2048),
        # a prompt of the larger model from its rows
        _select("route-4096", 4096, 288, 8, kind="route", hidden=4096, scale=2.5),
        # the down projection of a dense shared expert for one token, added to the routed experts' sum in 32 bits
        _linear("linear-1", 1, 1536, 2048, residual="float32", out="float32"),
        # the scores of a vocabulary for a verify window
        _linear("linear-16-vocabulary", 16, 2048, 32768, out="float32"),
        # odd sizes, rows that are wider than what is used, a projection with bias and activation for a short chunk
        _linear("linear-45-odd", 45, 1999, 1001, dtype="float16", bias=True, act="gelu", pitch=9),
        # the projection of a long chunk with the residual stream added
        _linear("linear-8192", 8192, 4096, 4096, residual="same"),
        # gate and up projection of a dense shared expert for one token
        _gated("gated-1", 1, 2048, 1536),
        # the same for a chunk on one of four tensor-parallel shards of the larger model
        _gated("gated-200", 200, 4096, 512, dtype="float16"),
        # and for a prompt of the benchmark's sizes
        _gated("gated-4096", 4096, 2048, 1536),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("select", "route", "linear", "gated"))
    rows = _log_int(rng, 1, 8192)
    if kind in ("select", "route"):
        groups = rng.choice((1, 1, 2, 4, 8))
        per = _log_int(rng, max(2, 8 // groups), 512 // groups)
        keep = rng.randint(1, groups)
        c = _select("", rows, groups * per, rng.randint(1, min(16, keep * per)), kind=kind, scores=rng.choice(("sigmoid", "softmax")),
                    bias=rng.random() < 0.6, groups=groups, keep=keep, group_score=rng.choice(("max", "top2")), renorm=rng.random() < 0.7,
                    scale=rng.choice((1.0, 2.5)))
        if kind == "route":
            c["hidden"] = 8 * _log_int(rng, 32, 512)
    else:
        while True:
            inner, outer = _log_int(rng, 64, 8192), _log_int(rng, 16, 32768)
            pitch = -inner % 8 + rng.choice((0, 0, 8))
            c = dict(kind=kind, rows=rows, inner=inner, outer=outer, dtype=rng.choice(("bfloat16", "float16")), bias=rng.random() < 0.5, pitch=pitch)
            if kind == "linear":
                c = _linear("", act=rng.choice(ACTS), residual=rng.choice(("none", "same", "float32")), out=rng.choice(("same", "float32")), **c)
            else:
                c = _gated("", act=rng.choice(("silu", "silu", "gelu", "gelu_tanh")), limit=rng.choice((0.0, 2.0, 10.0)), **c)
            w = work(c)
            if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
                break
    del c["name"]
    return c


def work(case):
    r = case["rows"]
    if case["kind"] in ("select", "route"):
        e, k = case["experts"], case["topk"] + 1
        table = r * k * 8 + (4 * e if case["bias"] else 0)
        if case["kind"] == "select":
            return {"bytes": 4 * r * e + table, "flops": 4 * r * e}
        h = case["hidden"]
        return {"bytes": 2 * h * (r + e) + 4 * r * e + table, "flops": 2 * r * e * h + 4 * r * e}
    k, n, mats = case["inner"], case["outer"], 2 if case["kind"] == "gated" else 1
    size = {"none": 0, "same": 2, "float32": 4}
    out = size[case.get("out", "same")] + size[case.get("residual", "none")]
    return {"bytes": 2 * k * (r + mats * n) + out * r * n + (4 * mats * n if case["bias"] else 0), "flops": 2 * r * k * n * mats}


def _grid(gen, shape, spread, step):
    """bf16 values on a grid of 8 bits, as rows and weights have that were held in 8 bits: their products add up without rounding in 32 bits,
    in any order, so that experts whose logits are alike are so for everybody."""
    v = torch.randn(shape, generator=gen, device="cuda") * (spread / step)
    return (v.round().clamp(-127, 127) * step).to(torch.bfloat16)


def _wide(gen, rows, cols, pitch, spread, dtype):
    """[rows][cols] of a buffer whose rows are `pitch` longer."""
    return (torch.randn((rows, cols + pitch), generator=gen, device="cuda") * spread).to(dtype)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, s = case["rows"], {"case": case}
    if case["kind"] in ("select", "route"):
        e, k = case["experts"], case["topk"]
        # balance biases as training leaves them: a fraction of the scores' spread
        s["bias"] = torch.randn(e, generator=gen, device="cuda") * 0.1 if case["bias"] else None
        s["picks"] = torch.zeros((rows, k + 1), dtype=torch.int32, device="cuda")
        s["weights"] = torch.zeros((rows, k + 1), device="cuda")
        if case["kind"] == "select":
            s["logits"] = torch.randn((rows, e), generator=gen, device="cuda")
        else:
            h = case["hidden"]
            s["x"] = _grid(gen, (rows, h), 1.0, 2.0 ** -4)
            s["wr"] = _grid(gen, (e, h), h ** -0.5, 2.0 ** -(5 + round(math.log2(h) / 2)))
            s["logits"] = torch.zeros((rows, e), device="cuda")
        return s
    k, n, t = case["inner"], case["outer"], TYPES[case["dtype"]]
    names = ("w_gate", "w_up") if case["kind"] == "gated" else ("w",)
    s["x"] = _wide(gen, rows, k, case["pitch"], 1.0, t)
    for name in names:
        s[name] = _wide(gen, n, k, case["pitch"], k ** -0.5, t)
        s[name.replace("w", "bias", 1)] = torch.randn(n, generator=gen, device="cuda") * 0.3 if case["bias"] else None
    kinds = {"same": t, "float32": torch.float32}
    if case.get("residual", "none") != "none":
        s["residual"] = torch.randn((rows, n), generator=gen, device="cuda").to(kinds[case["residual"]])
    s["out"] = torch.zeros((rows, n), dtype=kinds[case.get("out", "same")], device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------

def _choose(logits, bias, c):
    """Routing table of fp32 logits.  In 64 bits: which of two scores is larger decides."""
    rows, e = logits.shape
    v = logits.double()
    if c["scores"] == "sigmoid":
        s = 1 / (1 + torch.exp(-v))
    else:
        s = torch.exp(v - v.amax(1, keepdim=True))
        s = s / s.sum(1, keepdim=True)
    full = s if bias is None else s + bias.double()
    key = v if bias is None else full                     # without a bias the logits have the scores' order
    if c["groups"] > 1:
        if c["group_score"] == "max":
            g = key.view(rows, c["groups"], -1).amax(2)
        else:
            g = full.view(rows, c["groups"], -1).sort(2, descending=True)[0][:, :, :2].sum(2)
        first = torch.sort(g, dim=1, descending=True, stable=True)[1][:, : c["keep"]]
        stay = torch.zeros_like(g, dtype=torch.bool).scatter_(1, first, True)
        key = key.masked_fill(~stay.repeat_interleave(e // c["groups"], 1), -math.inf)
    picks = torch.sort(key, dim=1, descending=True, stable=True)[1][:, : c["topk"]]
    w = s.gather(1, picks)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = w * c["scale"]
    # the shared expert closes each row
    return torch.cat([picks, torch.full_like(picks[:, :1], e)], 1).int(), torch.cat([w, torch.ones_like(w[:, :1])], 1).float()


def _act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    return v.clamp(min=0) if act == "relu" else v


def _product(x, w, bias):
    y = x.float() @ w.float().t()
    return y if bias is None else y + bias


def _plain(s):
    c = s["case"]
    if c["kind"] == "select":
        return _choose(s["logits"], s["bias"], c)
    if c["kind"] == "route":
        logits = s["x"].float() @ s["wr"].float().t()
        return (logits,) + _choose(logits, s["bias"], c)
    if c["kind"] == "linear":
        y = _act(_product(s["x"], s["w"], s["bias"]), c["act"])
        if "residual" in s:
            y = y + s["residual"].float()
        return y.to(s["out"].dtype)
    g, u = _product(s["x"], s["w_gate"], s["bias_gate"]), _product(s["x"], s["w_up"], s["bias_up"])
    if c["limit"] > 0:
        g, u = g.clamp(max=c["limit"]), u.clamp(-c["limit"], c["limit"])
    return (_act(g, c["act"]) * u).to(s["out"].dtype)


# ---- the framework's calls ---------------------------------------------------------------------------------------------------------

_pkg = None


def _package():
    global _pkg
    if _pkg is None:
        import __graft_entry__ as entry
        _pkg = entry.load_package()
    return _pkg


def _own(s):
    pkg, c = _package(), s["case"]
    if c["kind"] == "linear":
        return pkg.linear(s["x"], s["w"], out=s["out"], bias=s["bias"], act=c["act"], residual=s.get("residual"))
    if c["kind"] == "gated":
        return pkg.gated_linear(s["x"], s["w_gate"], s["w_up"], out=s["out"], bias_gate=s["bias_gate"], bias_up=s["bias_up"], act=c["act"],
                                limit=c["limit"])
    rule = dict(bias=s["bias"], scores=c["scores"], groups=c["groups"], keep_groups=c["keep"], group_score=c["group_score"], renorm=c["renorm"],
                scale=c["scale"])
    if c["kind"] == "select":
        return pkg.topk_by(s["logits"], s["picks"], s["weights"], **rule)
    pkg.route_by(s["x"], s["wr"], s["logits"], s["picks"], s["weights"], **rule)
    return s["logits"], s["picks"], s["weights"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------

def _table(logits, bias, c):
    """numpy, a row's experts ordered by (score descending, id ascending)."""
    rows, e = logits.shape
    with np.errstate(over="ignore"):
        if c["scores"] == "sigmoid":
            score = np.where(logits >= 0, 1 / (1 + np.exp(-np.abs(logits))), 1 - 1 / (1 + np.exp(-np.abs(logits))))
            score = np.where(logits < -1, np.exp(-np.logaddexp(0, -logits)), score)
        else:
            score = np.exp(logits - np.logaddexp.reduce(logits, 1)[:, None])
    chosen_by = logits if bias is None else score + bias
    if c["groups"] > 1:
        n = e // c["groups"]
        if c["group_score"] == "max":
            value = chosen_by.reshape(rows, -1, n).max(2)
        else:
            value = np.sort((score if bias is None else chosen_by).reshape(rows, -1, n), 2)[:, :, -2:].sum(2)
        place = np.argsort(np.argsort(-value, 1, kind="stable"), 1)
        chosen_by = np.where(np.repeat(place < c["keep"], n, 1), chosen_by, -np.inf)
    picks = np.argsort(-chosen_by, 1, kind="stable")[:, : c["topk"]]
    w = np.take_along_axis(score, picks, 1)
    w = c["scale"] * (w / w.sum(1, keepdims=True) if c["renorm"] else w)
    return np.concatenate([w, np.ones((rows, 1))], 1)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] in ("select", "route"):
        bias = None if s["bias"] is None else s["bias"].cpu().numpy().astype(np.float64)
        if c["kind"] == "select":
            return None, _table(s["logits"].cpu().numpy().astype(np.float64), bias, c)
        logits = torch.einsum("rh,eh->re", s["x"].double(), s["wr"].double()).cpu().numpy()
        return logits, None, _table(logits, bias, c)
    x = s["x"].double()

    def product(w, bias):
        y = torch.einsum("rk,nk->rn", x, w.double())
        return y if bias is None else y + bias.double()

    def activation(v):
        if c["act"] == "silu":
            return v * torch.special.expit(v)
        if c["act"] == "gelu":
            return v * torch.special.ndtr(v)
        if c["act"] == "gelu_tanh":                       # (1 + tanh(z)) / 2 is the logistic function of 2 z
            return v * torch.special.expit(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))
        return torch.maximum(v, torch.zeros_like(v)) if c["act"] == "relu" else v

    if c["kind"] == "linear":
        y = activation(product(s["w"], s["bias"]))
        return y + s["residual"].double() if "residual" in s else y
    g, u = product(s["w_gate"], s["bias_gate"]), product(s["w_up"], s["bias_up"])
    if c["limit"] > 0:
        g, u = torch.clamp(g, max=c["limit"]), torch.clamp(u, -c["limit"], c["limit"])
    return activation(g) * u

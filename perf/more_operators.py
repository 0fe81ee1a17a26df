"""Measured calls of what a mixture-of-experts block needs around its products: the norm before it, the
routing of its tokens, and the rows' way to the experts and back, each with its gradients.

    layer_norm, rms_norm   s = x + residual, y = norm(s) * weight + bias; or the norm of x alone
    route_experts          scores of the router's logits, each token's top_k experts, their weights, and the
                           picks' order by expert
    dispatch_rows          the tokens' rows, once per pick, in the experts' order
    combine_rows           the weighted sum of each token's rows, plus a residual

A case is a dict of plain values:

    op        "layer_norm", "rms_norm", "route", "dispatch" or "combine"
    rows      rows of x, or tokens; of the tokens the last `pad` are padding, which no expert takes
    cols      columns of x
    experts, top_k, groups, top_groups, scoring, bias, renormalize, scale       of the routing
    residual  x is added to a residual first (norms), or the sum is added to one (combine)
    dtype     of x or the logits; wtype: of the norm's weight and bias
    train     forward and backward

`run` computes the plain form in 32 bits, or with `own` set calls the framework; `exact` is the same from
the definition in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_INF = math.inf


def _norm(name, op, rows, cols, dtype, wtype=None, residual=False, train=False):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype, "wtype": wtype or dtype,
            "residual": residual, "train": train}


def _route(name, rows, experts, top_k, dtype, scoring="softmax", groups=1, top_groups=1, bias=False,
           renormalize=True, scale=1.0, pad=0, train=False):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "top_k": top_k, "dtype": dtype,
            "scoring": scoring, "groups": groups, "top_groups": top_groups, "bias": bias,
            "renormalize": renormalize, "scale": scale, "pad": pad, "train": train}


def _move(name, op, rows, top_k, experts, cols, dtype, residual=False, pad=0, train=False):
    return {"name": name, "op": op, "rows": rows, "top_k": top_k, "experts": experts, "cols": cols,
            "dtype": dtype, "residual": residual, "pad": pad, "train": train}


def listed():
    return [
        # the norm before a DeepSeek-V2-Lite block, one token
        _norm("rms_1_token", "rms_norm", 1, 2048, "bf16", residual=True),
        # a layer norm in a verify step
        _norm("layer_verify", "layer_norm", 32, 4096, "fp16", residual=True),
        # the norm before a Mixtral block in training, 16384 tokens, weights kept in 32 bits
        _norm("rms_train", "rms_norm", 16384, 4096, "bf16", wtype="fp32", residual=True, train=True),
        # a layer norm over a ragged fp32 batch of odd rows: no row is aligned
        _norm("layer_train_odd", "layer_norm", 2999, 1001, "fp32", train=True),
        # the norm of the query heads of 4096 tokens: many short rows
        _norm("rms_train_heads", "rms_norm", 131072, 128, "bf16", train=True),
        # one token of DeepSeek-V2-Lite: 6 of 64 experts
        _route("route_1_token", 1, 64, 6, "bf16", renormalize=False),
        # a prompt of 8191 tokens over 256 experts in groups, with a bias for balance
        _route("route_prefill", 8191, 256, 8, "fp32", scoring="sigmoid", groups=8, top_groups=4, bias=True,
               scale=2.5),
        # training DeepSeek-V2-Lite's router on 16384 tokens, the batch padded
        _route("route_train", 16384, 64, 6, "bf16", renormalize=False, pad=500, train=True),
        # the rows of a verify step of 32 tokens to DeepSeek-V2-Lite's experts
        _move("dispatch_verify", "dispatch", 32, 6, 64, 2048, "bf16"),
        # the rows of 8192 tokens to Mixtral's experts in training
        _move("dispatch_train", "dispatch", 8192, 2, 8, 4096, "bf16", pad=100, train=True),
        # one token back from Mixtral's experts to the residual stream
        _move("combine_1_token", "combine", 1, 2, 8, 4096, "fp16", residual=True),
        # 8191 tokens back from DeepSeek-V2-Lite's experts in training
        _move("combine_train", "combine", 8191, 6, 64, 2048, "bf16", residual=True, train=True),
    ]


def _size(rng, low, high):
    """A size of [low, high], even over its logarithm: half of them multiples of 64, a quarter
    multiples of 8, the rest whatever comes."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    step = rng.choice((64, 64, 8, 1))
    return max(low, min(high, round(v / step) * step))


def _count(rng, high):
    return round(math.exp(rng.uniform(0.0, math.log(high))))


def draw(rng):
    while True:
        op = rng.choice(("layer_norm", "rms_norm", "route", "dispatch", "combine"))
        dtype, train = rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.5
        size = 4 if dtype == "fp32" else 2
        if op.endswith("norm"):
            case = _norm(None, op, _count(rng, 131072), _size(rng, 64, 16384), dtype,
                         rng.choice((dtype, dtype, "fp32")), rng.random() < 0.5, train)
            volume = case["rows"] * case["cols"]
        elif op == "route":
            groups = rng.choice((1, 1, 2, 4, 8))
            experts = max(2, round(math.exp(rng.uniform(math.log(4), math.log(512))) / groups)) * groups
            top_groups = rng.randint(1, groups)
            case = _route(None, _count(rng, 65536), experts, rng.randint(1, min(8, experts // groups * top_groups)),
                          dtype, rng.choice(("softmax", "sigmoid")), groups, top_groups, rng.random() < 0.5,
                          rng.random() < 0.5, rng.choice((1.0, 2.5)), train=train)
            # (the one weight of a renormalised top-1 is constant: no gradient to speak of)
            case["renormalize"] = case["renormalize"] and (case["top_k"] > 1 or not train)
            volume = case["rows"] * case["experts"] * 4
        else:
            top_k = rng.randint(1, 8)
            case = _move(None, op, _count(rng, 32768), top_k, max(top_k, _count(rng, 256)), _size(rng, 64, 8192),
                         dtype, op == "combine" and rng.random() < 0.5, train=train)
            volume = case["rows"] * case["cols"] * top_k
        if not op.endswith("norm") and rng.random() < 0.25:
            case["pad"] = rng.randrange(case["rows"]) // 8
        del case["name"]
        if volume * size <= 16384 * 4096 * 2:
            return case


def _picks(case, gen, dev):
    """The picks' places in the experts' order, and the pick at each place; complements (~) for those of
    padding, which come last."""
    rows, k, experts = case["rows"], case["top_k"], case["experts"]
    load = 0.5 * torch.randn(experts, generator=gen, device=dev)
    noise = torch.rand((rows, experts), generator=gen, device=dev).clamp_min_(1e-20)
    ids = (load - torch.log(-torch.log(noise))).topk(k, dim=1).indices  # distinct, by uneven loads
    ids[rows - case["pad"]:] = experts
    order = torch.sort(ids.flatten(), stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(rows * k, device=dev)
    idle = ids.flatten() == experts
    places = torch.where(idle, ~places, places).view(rows, k)
    return places.int(), torch.where(idle[order], ~order, order).int()


def prepare(case, seed):
    dev, dt, op = torch.device("cuda"), _TYPES[case["dtype"]], case["op"]
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, train = case["rows"], case["train"]

    def normal(shape, scale=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, dtype=torch.float32, device=dev).normal_(mean, scale, generator=gen).to(dtype)

    s = {"case": case, "leaves": []}

    def leaf(name, t):
        s[name] = t
        if train:
            s["leaves"].append(t.requires_grad_())

    if op.endswith("norm"):
        wt, cols = _TYPES[case["wtype"]], case["cols"]
        leaf("x", normal((rows, cols), 1.5, 0.25))
        if case["residual"]:
            leaf("residual", normal((rows, cols), 2.0))
        leaf("weight", normal((cols,), 0.2, 1.0, wt))
        if op == "layer_norm":
            leaf("bias", normal((cols,), 0.1, 0.0, wt))
        if train:
            s["dy"] = normal((rows, cols))
            if case["residual"]:
                s["ds"] = normal((rows, cols))
    elif op == "route":
        logits = normal((rows, case["experts"]), 1.5)
        logits[rows - case["pad"]:] = -_INF
        leaf("logits", logits)
        s["bias"] = normal((case["experts"],), 0.1, 0.0, torch.float32) if case["bias"] else None
        if train:
            s["dw"] = normal((rows, case["top_k"]), dtype=torch.float32)
    else:
        s["places"], s["order"] = _picks(case, gen, dev)
        picks, cols = rows * case["top_k"], case["cols"]
        if op == "dispatch":
            leaf("x", normal((rows, cols)))
        else:
            leaf("rows", normal((picks, cols)))
            leaf("weights", torch.rand((rows, case["top_k"]), generator=gen, device=dev))
            if case["residual"]:
                leaf("residual", normal((rows, cols)))
        if train:
            s["dy"] = normal((picks if op == "dispatch" else rows, cols))
    return s


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"layer_norm": _plain_norm, "rms_norm": _plain_norm, "route": _plain_route,
                "dispatch": _plain_dispatch, "combine": _plain_combine}[state["case"]["op"]](state)


def _run_own(s):
    from ae_amd.layers import combine_rows, dispatch_rows, layer_norm, rms_norm, route_experts

    case, op = s["case"], s["case"]["op"]
    if op.endswith("norm"):
        residual = s.get("residual")
        if op == "rms_norm":
            outs = rms_norm(s["x"], s["weight"], _EPS, residual=residual)
        else:
            outs = layer_norm(s["x"], s["weight"], s["bias"], _EPS, residual=residual)
        outs = list(outs) if case["residual"] else [outs]
        given = [s.get("dy"), s.get("ds")][:len(outs)]
    elif op == "route":
        r = route_experts(s["logits"], case["top_k"], scoring=case["scoring"], bias=s["bias"],
                          num_groups=case["groups"], top_groups=case["top_groups"],
                          renormalize=case["renormalize"], scale=case["scale"])
        outs, given = [r.weights], [s.get("dw")]
    elif op == "dispatch":
        outs, given = [dispatch_rows(s["x"], s["places"])], [s.get("dy")]
    else:
        outs = [combine_rows(s["rows"], s["places"], s["weights"], residual=s.get("residual"))]
        given = [s.get("dy")]
    grads = torch.autograd.grad(outs, s["leaves"], given) if case["train"] else ()
    whole = [r.ids, r.places, r.order, r.offsets] if op == "route" else []
    return [*outs, *whole, *grads]


def _plain_norm(s):
    case = s["case"]
    dt = _TYPES[case["dtype"]]
    n, rms = case["cols"], case["op"] == "rms_norm"
    outs = []
    h = s["x"].float()
    if case["residual"]:
        total = (h + s["residual"].float()).to(dt)  # the sum is an output, and what is normalised
        outs = [total]
        h = total.float()
    mean = 0.0 if rms else h.sum(1, keepdim=True) / n
    c = h - mean
    rstd = 1.0 / torch.sqrt((c * c).sum(1, keepdim=True) / n + _EPS)
    xh = c * rstd
    w = s["weight"].float()
    y = xh * w
    if not rms:
        y = y + s["bias"].float()
    outs = [y.to(dt), *outs]
    if case["train"]:
        wt = _TYPES[case["wtype"]]
        dy = s["dy"].float()
        g = dy * w
        dx = g - xh * ((g * xh).sum(1, keepdim=True) / n)
        if not rms:
            dx = dx - g.sum(1, keepdim=True) / n
        dx = dx * rstd
        if case["residual"]:
            dx = dx + s["ds"].float()
        dx = dx.to(dt)
        outs += [dx, dx] if case["residual"] else [dx]
        outs.append((dy * xh).sum(0).to(wt))
        if not rms:
            outs.append(dy.sum(0).to(wt))
    return outs


def _scores(scoring, logits):
    """Scores of the rows, zero throughout in rows without any."""
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - torch.where(top == -_INF, 0.0, top))
    return e / e.sum(1, keepdim=True).clamp_min(1e-30)


def _plain_route(s):
    case = s["case"]
    rows, experts, k, groups = case["rows"], case["experts"], case["top_k"], case["groups"]
    logits = s["logits"].float()
    # what picks are compared by: the logits themselves, or with a bias sums that may lie close, in 64 bits
    choice = logits
    if case["bias"]:
        choice = _scores(case["scoring"], logits.double()) + s["bias"].double()
        choice = torch.where(logits == -_INF, -_INF, choice)
    if case["top_groups"] < groups:
        best = torch.sort(choice.view(rows, groups, -1), dim=2, descending=True).values
        rank = best[:, :, 0]
        if case["bias"]:
            rank = rank + torch.where(best[:, :, 1] == -_INF, 0.0, best[:, :, 1])
        kept = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        out = torch.ones((rows, groups), dtype=torch.bool, device=logits.device).scatter_(1, kept, False)
        choice = choice.masked_fill(out.repeat_interleave(experts // groups, 1), -_INF)
    value, ids = torch.sort(choice, dim=1, descending=True, stable=True)
    idle, ids = value[:, :k] == -_INF, ids[:, :k]
    score = _scores(case["scoring"], logits)
    p = score.gather(1, ids).masked_fill(idle, 0.0)
    total = p.sum(1, keepdim=True).clamp_min(1e-30)
    weights = case["scale"] * (p / total if case["renormalize"] else p)
    # the picks in the experts' order, those of nobody last
    flat = ids.masked_fill(idle, experts).flatten()
    order = torch.sort(flat, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(rows * k, device=order.device)
    idle = idle.flatten()
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    offsets = counts.scatter_add_(0, flat, torch.ones_like(flat))[:experts]
    offsets = torch.cat([offsets.new_zeros(1), offsets.cumsum(0)])
    outs = [weights, ids.masked_fill(idle.view(rows, k), -1).int(),
            torch.where(idle, ~places, places).view(rows, k).int(),
            torch.where(idle[order], ~order, order).int(), offsets]
    if case["train"]:
        dw = case["scale"] * s["dw"].masked_fill(idle.view(rows, k), 0.0)
        if case["renormalize"]:
            q = p / total
            dp = (dw - (dw * q).sum(1, keepdim=True)) / total
        else:
            dp = dw
        if case["scoring"] == "sigmoid":
            d = torch.zeros_like(score).scatter_add_(1, ids, dp * p * (1.0 - p))
        else:
            d = torch.zeros_like(score).scatter_add_(1, ids, dp * p) - score * (dp * p).sum(1, keepdim=True)
        outs.append(d.to(s["logits"].dtype))
    return outs


def _gathered(rows, places):
    """[tokens, top_k, cols] in 32 bits, zero at picks of nobody."""
    return torch.where((places < 0)[:, :, None], 0.0, rows[places.clamp_min(0).long()].float())


def _plain_dispatch(s):
    case, order, x = s["case"], s["order"].long(), s["x"]
    rows = torch.where((order < 0)[:, None], 0.0, x[order.clamp_min(0) // case["top_k"]].float()).to(x.dtype)
    return [rows, _gathered(s["dy"], s["places"]).sum(1).to(x.dtype)] if case["train"] else [rows]


def _plain_combine(s):
    case, order, rows = s["case"], s["order"].long(), s["rows"]
    dt, w = rows.dtype, s["weights"]
    got = _gathered(rows, s["places"])
    y = (got * w[:, :, None]).sum(1)
    if case["residual"]:
        y = y + s["residual"].float()
    outs = [y.to(dt)]
    if case["train"]:
        dy, pick = s["dy"].float(), order.clamp_min(0)
        at = torch.where(order < 0, 0.0, w.flatten()[pick])
        outs += [(dy[pick // case["top_k"]] * at[:, None]).to(dt), (got * dy[:, None, :]).sum(2)]
        if case["residual"]:
            outs.append(s["dy"])
    return outs


def exact(case, seed):
    """The definition in 64 bits; the gradients are torch's own differentiation of it."""
    s = prepare(case, seed)
    op, train = case["op"], case["train"]
    leaves = [t.detach().double().requires_grad_(train) for t in s["leaves"]]
    names = [n for n in ("x", "residual", "weight", "bias") if n in s] if op.endswith("norm") else \
        {"route": ["logits"], "dispatch": ["x"],
         "combine": [n for n in ("rows", "weights", "residual") if n in s]}[op]
    if not train:
        leaves = [s[n].detach().double() for n in names]
    v = dict(zip(names, leaves))
    whole = []
    if op.endswith("norm"):
        h = v["x"]
        if case["residual"]:
            h = h + v["residual"]
            total = h
            # the sum as it is kept, with the gradient of the sum
            h = h + (h.detach().to(_TYPES[case["dtype"]]).double() - h.detach())
        if op == "layer_norm":
            var, mean = torch.var_mean(h, dim=1, keepdim=True, unbiased=False)
            y = (h - mean) * torch.rsqrt(var + _EPS) * v["weight"] + v["bias"]
        else:
            y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + _EPS) * v["weight"]
        outs = [y, total] if case["residual"] else [y]
        given = [s.get("dy"), s.get("ds")][:len(outs)]
    elif op == "route":
        outs, given = [_exact_weights(case, v["logits"], s["bias"])], [s.get("dw")]
        whole = [None] * 4  # whole numbers: the plain form's are right or wrong
    elif op == "dispatch":
        order = s["order"].long()
        taken = torch.cat([v["x"], v["x"].new_zeros((1, case["cols"]))])
        outs = [taken[torch.where(order < 0, case["rows"], order // case["top_k"])]]
        given = [s.get("dy")]
    else:
        places = s["places"].long()
        at = torch.where(places < 0, case["rows"] * case["top_k"], places)
        taken = torch.cat([v["rows"], v["rows"].new_zeros((1, case["cols"]))])
        y = sum(taken[at[:, j]] * v["weights"][:, j:j + 1] for j in range(case["top_k"]))
        outs = [y + v["residual"] if case["residual"] else y]
        given = [s.get("dy")]
    grads = torch.autograd.grad(outs, leaves, [g.double() for g in given]) if train else ()
    return [*(t.detach() for t in outs), *whole, *grads]


def _exact_weights(case, logits, bias):
    experts, groups = case["experts"], case["groups"]
    live = logits.detach() > -_INF
    some = live.any(1, keepdim=True)
    x = torch.where(live, logits, torch.where(some, -_INF, 0.0))
    score = torch.sigmoid(x) if case["scoring"] == "sigmoid" else torch.softmax(x, 1)
    with torch.no_grad():
        choice = score + bias.double() if case["bias"] else logits.detach()
        choice = choice.masked_fill(~live, -_INF)
        if case["top_groups"] < groups:
            each = choice.view(-1, groups, experts // groups)
            rank = each.amax(2)
            if case["bias"]:
                two = each.topk(2, dim=2).values
                rank = rank + two[:, :, 1].masked_fill(two[:, :, 1] == -_INF, 0.0)
            # a group is kept if fewer than top_groups others come before it
            before = (rank[:, None, :] > rank[:, :, None]) | (
                (rank[:, None, :] == rank[:, :, None]) &
                torch.ones((groups, groups), dtype=torch.bool, device=rank.device).tril(-1))
            kept = before.sum(2) < case["top_groups"]
            choice = choice.masked_fill(~kept.repeat_interleave(experts // groups, 1), -_INF)
        value, ids = torch.sort(choice, dim=1, descending=True, stable=True)
        value, ids = value[:, :case["top_k"]], ids[:, :case["top_k"]]
    p = torch.where(value == -_INF, 0.0, score.gather(1, ids))
    if case["renormalize"]:
        p = p / torch.where(some, p.sum(1, keepdim=True), 1.0)
    return case["scale"] * p


def work(case):
    op, rows, train = case["op"], case["rows"], case["train"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op.endswith("norm"):
        elems, vectors = rows * case["cols"], 1 + (op == "layer_norm")
        parts = 2 + 2 * case["residual"] + train * (2 + case["residual"])
        wsize = 4 if case["wtype"] == "fp32" else 2
        return {"bytes": elems * size * parts + case["cols"] * vectors * wsize * (1 + train),
                "flops": elems * (24 if train else 8)}
    picks = rows * case["top_k"]
    if op == "route":
        elems = rows * case["experts"]
        return {"bytes": elems * size * (1 + train) + picks * (16 + 4 * train) + 8 * (case["experts"] + 1) +
                4 * case["experts"] * case["bias"], "flops": elems * (10 if train else 6)}
    used = picks - case["pad"] * case["top_k"]
    cols = case["cols"]
    if op == "dispatch":  # rows in and out, and the gradients out and in
        return {"bytes": ((rows + picks) + train * (used + rows)) * cols * size + 4 * picks,
                "flops": used * cols * train + rows * cols}
    elems = used + rows * (1 + case["residual"]) + train * (rows + picks)
    return {"bytes": elems * cols * size + picks * (8 + 4 * train), "flops": used * cols * (2 + 3 * train)}

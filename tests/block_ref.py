"""Norms, routing, dispatch and combine in 64 bits, with a bound on how far the kernels' outputs may be off.

u = finfo.eps / 2 of the output's type (a rounding is off by at most half a step), e = 2^-24. A sum over a row runs in a chain
of at most D = 48 fp32 additions per term (16 elements of a thread, 6 steps of a wave, 16 waves, and a few
more): off by D e of the sum of the magnitudes. A sum over R rows: (R + 24) e. exp and rsqrt are good to
2^-22; exp of an argument that was rounded, to e of the argument's magnitude more. Half of a type's smallest number
is added wherever something is rounded to it.
"""
import torch

F64 = torch.float64
E32 = 2.0 ** -24
D = 48
INF = float("inf")


def rounded(v, err, dtype):
    """err, and one rounding to dtype (a result behind the type's largest number may be infinite)."""
    f = torch.finfo(dtype)
    return v, err + f.eps / 2 * (v.abs() + err) + f.smallest_normal * f.eps / 2


def norm(s, weight, bias, eps, rms, dtype, params=None, dy=None, ds=None):
    """{"y": (value, bound), and with dy "dx", "dw", "db"} for the rows s (as they are kept)."""
    s = s.to(F64)
    w = torch.ones(s.shape[1], dtype=F64, device=s.device) if weight is None else weight.to(F64)
    b = torch.zeros_like(w) if bias is None else bias.to(F64)
    mean = torch.zeros_like(s[:, :1]) if rms else s.mean(1, keepdim=True)
    c = s - mean
    ec = torch.zeros_like(c) if rms else D * E32 * s.abs().mean(1, keepdim=True) + 2 * E32 * c.abs()
    var = c.square().mean(1, keepdim=True) + eps
    # the variance: its terms' errors (at most 2 |c| ec, whose mean is at most 2 sqrt(var mean(ec^2)); and ec^2) and its sum
    rv = 2 * (ec.square().mean(1, keepdim=True) / var).sqrt() + ec.square().mean(1, keepdim=True) / var + (D + 4) * E32
    rr = rv / 2 + rv * rv + 2.0 ** -22
    rstd = var.rsqrt()
    n = c * rstd
    en = rstd * ec * (1 + rr) + n.abs() * (rr + 2 * E32)
    y = n * w + b
    out = {"y": rounded(y, w.abs() * en + 3 * E32 * ((n * w).abs() + b.abs()), dtype)}
    if dy is None:
        return out
    dy = dy.to(F64)
    params = dtype if params is None else params
    g = dy * w
    h = s.shape[1]
    c1 = torch.zeros_like(mean) if rms else g.mean(1, keepdim=True)
    e1 = (D + 2) * E32 * g.abs().mean(1, keepdim=True) if not rms else torch.zeros_like(mean)
    c2 = (g * n).mean(1, keepdim=True)
    e2 = (g.abs() * en).mean(1, keepdim=True) + (D + 4) * E32 * (g * n).abs().mean(1, keepdim=True)
    v = rstd * (g - c1 - n * c2)
    top = g.abs() + c1.abs() + (n * c2).abs()
    ev = rstd * (1 + rr) * (e1 + en * (c2.abs() + e2) + n.abs() * e2 + 4 * E32 * top) + rr * v.abs() + 3 * E32 * rstd * top
    if ds is not None:
        v = v + ds.to(F64)
        ev = ev + 2 * E32 * (v.abs() + ds.to(F64).abs())
    out["dx"] = rounded(v, ev, dtype)
    rows = s.shape[0]
    out["dw"] = rounded((dy * n).sum(0), (dy.abs() * en).sum(0) + (rows + 24) * E32 * (dy * n).abs().sum(0), params)
    out["db"] = rounded(dy.sum(0), (rows + 24) * E32 * dy.abs().sum(0), params)
    assert h == w.shape[0]
    return out


def scores(logits, scoring):
    live = logits > -INF
    if scoring == "sigmoid":
        return torch.where(live, torch.sigmoid(logits), 0.0) + torch.where(logits.isnan(), logits, 0.0)
    return torch.nan_to_num(torch.softmax(torch.where(live.any(1, keepdim=True), logits, 0.0), 1), nan=float("nan")) \
        * live.any(1, keepdim=True)


def choose(logits, k, scoring, bias, groups, top_groups):
    """ids [T, k] (-1: nobody) in 64 bits, one token at a time as the definition says it."""
    x = logits.to(F64)
    c = x.clone() if bias is None else scores(x, scoring) + bias.to(F64)
    c[x == -INF] = -INF
    c = torch.where(c.isnan(), INF, c) if bias is None else torch.where(c.isnan(), torch.finfo(F64).max, c)
    t, e = c.shape
    if top_groups < groups:
        two, at = torch.sort(c.view(t, groups, -1), dim=2, descending=True)
        rank = two[:, :, 0].clone()
        if bias is not None and two.shape[2] > 1:
            # (scores and biases each on their own: s + (b + 1/2) and (s + 1/2) + b are one number, but round differently)
            s, b = ((v.expand_as(c).reshape(t, groups, -1).gather(2, at[:, :, :2]) for v in (scores(x, scoring), bias.to(F64))))
            both = s.sum(2) + b.sum(2)
            rank = torch.where(two[:, :, 1] == -INF, rank, torch.where(both.isnan(), torch.finfo(F64).max, both))
        keep = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :top_groups]
        mask = torch.zeros((t, groups), dtype=torch.bool, device=c.device).scatter_(1, keep, True)
        c = torch.where(mask.repeat_interleave(e // groups, 1), c, -INF)
    value, ids = torch.sort(c, dim=1, descending=True, stable=True)
    return torch.where(value[:, :k] == -INF, -1, ids[:, :k])


def route(logits, ids, scoring, renormalize, scale, dw=None):
    """{"weights": (value, bound), and with dw "dlogits"} of the picks ids."""
    dtype = logits.dtype
    x = logits.to(F64)
    idle = ids < 0
    at = ids.clamp_min(0).long()
    sel = x.gather(1, at)
    live = torch.where(idle, 0.0, 1.0).to(F64)
    s = scores(x, scoring)
    p = s.gather(1, at) * live
    # the arguments of exp: distances from the largest logit, or the logits
    top = torch.where(x == -INF, -1e30, x).amax(1, keepdim=True)
    if renormalize:
        if scoring == "softmax":
            q = torch.softmax(torch.where(idle, -INF, sel), 1)
        else:
            ls = torch.where(idle, -INF, torch.nn.functional.logsigmoid(sel))
            q = torch.softmax(ls, 1)
        q = torch.where(idle, 0.0, q)
    else:
        q = p
    arg = torch.where(idle, 0.0, (sel - top) if scoring == "softmax" else sel).abs().amax(1, keepdim=True)
    rel = 4 * 2.0 ** -22 + 2 * arg * E32 + (D + 8) * E32
    tiny = 2.0 ** -125
    out = {"weights": (scale * q, abs(scale) * (q * (rel + 2 * E32) + tiny))}
    if dw is None:
        return out
    g = torch.where(idle, 0.0, scale * dw.to(F64))
    d = torch.zeros_like(x)
    err = torch.zeros_like(x)
    one = 1 - torch.sigmoid(sel) if scoring == "sigmoid" else torch.ones_like(sel)
    if scoring == "sigmoid":
        one = torch.sigmoid(-sel)
    if renormalize or scoring == "softmax":
        dot = (q * g).sum(1, keepdim=True)
        edot = (q.abs() * g.abs()).sum(1, keepdim=True) * (rel + 20 * E32)
    else:
        dot = edot = torch.zeros_like(x[:, :1])
    if renormalize:
        v = q * one * (g - dot)
        ev = q * one * ((g.abs() + dot.abs()) * (2 * rel + 8 * E32) + edot)
        d.scatter_add_(1, at, torch.where(idle, 0.0, v))
        err.scatter_add_(1, at, torch.where(idle, 0.0, ev))
    elif scoring == "sigmoid":
        v = p * one * g
        d.scatter_add_(1, at, torch.where(idle, 0.0, v))
        err.scatter_add_(1, at, torch.where(idle, 0.0, v.abs() * (2 * rel + 8 * E32)))
    else:
        reach = torch.where(x == -INF, 0.0, x - top).abs()
        rels = 4 * 2.0 ** -22 + 2 * reach * E32 + (D + 8) * E32
        d = -s * dot
        err = s * (dot.abs() * (rels + 4 * E32) + edot * (1 + rels))
        d = d.scatter_add(1, at, torch.where(idle, 0.0, p * g))
        err = err.scatter_add(1, at, torch.where(idle, 0.0, (p * g).abs() * (rel + 8 * E32)))
        err = err + 2 * E32 * d.abs()
    out["dlogits"] = rounded(d, err + tiny * (1 + g.abs().amax(1, keepdim=True)), dtype)
    return out


def order_of(ids, experts):
    """(places, order, offsets) of the stable sort of the picks by expert, picks of nobody last."""
    flat = torch.where(ids < 0, experts, ids.long()).flatten()
    order = torch.sort(flat, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(flat.numel(), device=ids.device)
    idle = flat == experts
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0)
    return (torch.where(idle, ~places, places).view(ids.shape).int(), torch.where(idle[order], ~order, order).int(),
            offsets)


def combine(rows, places, weights, residual, dtype, dy=None):
    """{"y": (value, bound), and with dy "drows", "dw"}."""
    t, k = places.shape
    live = (places >= 0) & (places < t * k)
    got = torch.where(live[:, :, None], rows.to(F64)[torch.where(live, places, 0).long()], 0.0)
    w = torch.where(live, 1.0 if weights is None else weights.to(F64), 0.0)
    terms = got * w[:, :, None]
    y, mag = terms.sum(1), terms.abs().sum(1)
    if residual is not None:
        y, mag = y + residual.to(F64), mag + residual.to(F64).abs()
    out = {"y": rounded(y, (k + 2) * E32 * mag, dtype)}
    if dy is None:
        return out
    dy = dy.to(F64)
    drows = torch.zeros(rows.shape, dtype=F64, device=rows.device)
    drows[torch.where(live, places, 0).long()[live]] = (dy[:, None, :] * w[:, :, None])[live]
    out["drows"] = rounded(drows, E32 * drows.abs(), dtype)
    h = rows.shape[1]
    out["dw"] = rounded((got * dy[:, None, :]).sum(2), (h + 24) * E32 * (got * dy[:, None, :]).abs().sum(2), torch.float32)
    return out

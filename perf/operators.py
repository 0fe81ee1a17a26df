"""Measured calls of the matrix products: `fused_linear` and `grouped_linear`, with gradients.

    y = residual + act(x W^T + b)              fused_linear, one weight
    the same with W[g], b[g] for the rows offsets[g] .. offsets[g + 1]       grouped_linear

act is the identity, relu, gelu, gelu_tanh, silu, or swiglu: silu(z[:, :N]) * z[:, N:] of a weight
of 2 N rows (gate rows, then up rows). A case is a dict of plain values:

    op        "linear" or "grouped"
    rows      rows of x; of these the last `spare` belong to no group (grouped)
    k, n      columns of x and of y
    groups    weights (grouped)
    pages     the weights are the gate and up parts of [gate | up | down] pages in a pool of twice as
              many slots, found through a slot map (grouped, act "swiglu")
    act, bias, residual, dtype
    train     forward and backward: y and the gradients of x, weight, bias and residual

`run` computes the plain form in 32 bits, or with `own` set calls the framework; `exact` is the same
from the definition in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "swiglu")


def _case(name, op, rows, k, n, dtype, act="none", bias=False, residual=False, train=False,
          groups=1, spare=0, pages=False):
    return {"name": name, "op": op, "rows": rows, "k": k, "n": n, "groups": groups, "spare": spare,
            "pages": pages, "act": act, "bias": bias, "residual": residual, "dtype": dtype,
            "train": train}


def listed():
    return [
        # the shared experts' gate and up projections of a DeepSeek-V2-Lite block, one token
        _case("linear_1_row", "linear", 1, 2048, 2816, "bf16", act="swiglu"),
        # a projection back to the residual stream in a verify step
        _case("linear_verify", "linear", 20, 4096, 4096, "fp16", bias=True, residual=True),
        # a small head of odd sizes: no row is aligned
        _case("linear_odd", "linear", 333, 1001, 515, "fp32", act="gelu", bias=True),
        # the first projection of a dense MLP over a prompt
        _case("linear_prefill", "linear", 8192, 4096, 14336, "bf16", act="gelu_tanh", bias=True),
        # the same in training, 4096 tokens, at Qwen1.5-MoE's shared-expert width
        _case("linear_train", "linear", 4096, 2048, 5632, "bf16", act="gelu", bias=True, train=True),
        # a ragged batch through a small fp32 block with a residual
        _case("linear_train_fp32", "linear", 777, 1024, 2816, "fp32", act="silu", bias=True,
              residual=True, train=True),
        # DeepSeek-V2-Lite experts of one token: 6 of 64, weights in the page pool
        _case("grouped_1_token", "grouped", 6, 2048, 1408, "bf16", act="swiglu", groups=64,
              pages=True),
        # Mixtral experts in a verify step of 32 tokens, weights in the page pool
        _case("grouped_verify", "grouped", 64, 4096, 14336, "fp16", act="swiglu", groups=8,
              pages=True),
        # Mixtral experts over a prompt of 8192 tokens
        _case("grouped_prefill", "grouped", 16384, 4096, 14336, "bf16", act="swiglu", groups=8),
        # training DeepSeek-V2-Lite's experts, 2047 tokens
        _case("grouped_train", "grouped", 12282, 2048, 1408, "bf16", act="swiglu", groups=64,
              train=True),
        # odd sizes with biases, a padded batch, more groups than some have rows for
        _case("grouped_train_odd", "grouped", 1000, 1021, 333, "fp16", act="gelu", bias=True,
              groups=60, spare=37, train=True),
        # an fp32 block of 8 experts, hidden 1024, whose outputs return to the residual stream
        _case("grouped_train_fp32", "grouped", 512, 1024, 2816, "fp32", act="gelu_tanh", bias=True,
              residual=True, groups=8, train=True),
    ]


def _weight_rows(case):
    return case["n"] * (2 if case["act"] == "swiglu" else 1)


def _size(rng, low, high):
    """A size of [low, high], even over its logarithm: half of them multiples of 64, a quarter
    multiples of 8, the rest whatever comes."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    step = rng.choice((64, 64, 8, 1))
    return max(low, min(high, round(v / step) * step))


def draw(rng):
    while True:
        op = rng.choice(("linear", "grouped"))
        train = rng.random() < 0.5
        # (relu's gradient jumps at 0, where the last bit of a sum decides: forward only)
        act = rng.choice([a for a in _ACTS if not (train and a == "relu")])
        grouped = op == "grouped"
        pages = grouped and act == "swiglu" and not train and rng.random() < 0.5
        rows = round(math.exp(rng.uniform(0.0, math.log(16384 if grouped else 8192))))
        spare = rng.randrange(rows) // 8 if grouped and rng.random() < 0.25 else 0
        case = _case(None, op, rows, _size(rng, 64, 8192), _size(rng, 64, 14336),
                     rng.choice(("bf16", "bf16", "fp16", "fp32")), act=act,
                     bias=not pages and rng.random() < 0.5, residual=rng.random() < 0.3,
                     train=train, groups=round(math.exp(rng.uniform(0.0, math.log(128)))) if grouped else 1,
                     spare=spare, pages=pages)
        del case["name"]
        weights = case["groups"] * _weight_rows(case) * case["k"]
        if weights > 4e8 or rows * case["k"] * _weight_rows(case) * (3 if train else 1) > 16384 * 4096 * 28672:
            continue
        if case["dtype"] == "fp32" and rows * case["k"] * _weight_rows(case) > 2e11:
            continue  # fp32 blocks are small ones
        return case


def _bounds(case, gen):
    """Row bounds of the groups: a token's picks are distinct experts; a batch's expert loads
    are uneven."""
    rows, groups = case["rows"] - case["spare"], case["groups"]
    if rows <= groups:
        counts = torch.zeros(groups, dtype=torch.int64)
        counts[torch.randperm(groups, generator=gen)[:rows]] = 1
    else:
        load = torch.softmax(0.5 * torch.randn(groups, generator=gen), 0)
        picks = torch.multinomial(load, rows, replacement=True, generator=gen)
        counts = torch.bincount(picks, minlength=groups)
    return [0] + torch.cumsum(counts, 0).tolist()


def prepare(case, seed):
    dev, dt = torch.device("cuda"), _TYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    rows, k, n, wr, groups = case["rows"], case["k"], case["n"], _weight_rows(case), case["groups"]

    def normal(shape, scale=1.0):
        return torch.empty(shape, dtype=dt, device=dev).normal_(0.0, scale, generator=gen)

    s = {"case": case, "x": normal((rows, k)), "bias": None, "residual": None, "slots": None}
    lead = () if case["op"] == "linear" else (groups,)
    if case["pages"]:
        pool = normal((2 * groups, 3 * n * k), k ** -0.5)
        s["weight"] = pool[:, :wr * k].unflatten(1, (wr, k))
        s["host_slots"] = torch.randperm(2 * groups, generator=host)[:groups].tolist()
        s["slots"] = torch.tensor(s["host_slots"], device=dev)
    else:
        s["weight"] = normal(lead + (wr, k), k ** -0.5)
    if case["bias"]:
        s["bias"] = normal(lead + (wr,), 0.1)
    if case["residual"]:
        s["residual"] = normal((rows, n))
    if case["op"] == "grouped":
        s["bounds"] = _bounds(case, host)  # what a loop over the groups needs on the host
        s["offsets"] = torch.tensor(s["bounds"], device=dev)
    if case["train"]:
        s["dy"] = normal((rows, n))
        for name in ("x", "weight", "bias", "residual"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def _run_own(s):
    from ae_amd.layers import fused_linear, grouped_linear

    case = s["case"]
    act = None if case["act"] == "none" else case["act"]
    if case["op"] == "linear":
        y = fused_linear(s["x"], s["weight"], s["bias"], act, s["residual"])
    else:
        y = grouped_linear(s["x"], s["weight"], s["offsets"], s["bias"], act, s["residual"],
                           weight_slots=s["slots"])
    if not case["train"]:
        return [y]
    leaves = [s[name] for name in ("x", "weight", "bias", "residual") if s[name] is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def _gelu_cdf(z):
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _gelu_tanh_t(z):
    return torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))


def _act(act, z, n):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return z * _gelu_cdf(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + _gelu_tanh_t(z))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z[:, :n] / (1.0 + torch.exp(-z[:, :n])) * z[:, n:]


def _act_grad(act, z, dy, n):
    if act == "none":
        return dy
    if act == "relu":
        return torch.where(z > 0, dy, torch.zeros_like(dy))
    if act == "gelu":
        return dy * (_gelu_cdf(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        t = _gelu_tanh_t(z)
        inner = math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * z * z)
        return dy * (0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * inner)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return dy * (s * (1.0 + z * (1.0 - s)))
    g, u = z[:, :n], z[:, n:]
    s = 1.0 / (1.0 + torch.exp(-g))
    return torch.cat([dy * u * (s * (1.0 + g * (1.0 - s))), dy * (g * s)], 1)


def _run_plain(s):
    case = s["case"]
    act, n, dt = case["act"], case["n"], _TYPES[case["dtype"]]
    x, w, res = s["x"], s["weight"], s["residual"]
    grouped = case["op"] == "grouped"
    bounds = s["bounds"] if grouped else [0, case["rows"]]
    y = torch.zeros((case["rows"], n), dtype=torch.float32, device=x.device)
    dx = torch.zeros(x.shape, dtype=dt, device=x.device) if case["train"] else None
    dw = torch.zeros(w.shape, dtype=dt, device=x.device) if case["train"] else None
    db = torch.zeros_like(s["bias"]) if case["train"] and case["bias"] else None
    for g in range(len(bounds) - 1):
        a, b = bounds[g], bounds[g + 1]
        if a == b:
            continue
        wg = (w[s["host_slots"][g]] if case["pages"] else w[g] if grouped else w).float()
        xg = x[a:b].float()
        z = xg @ wg.t()
        if case["bias"]:
            z = z + (s["bias"][g] if grouped else s["bias"]).float()
        y[a:b] = _act(act, z, n)
        if case["train"]:
            dz = _act_grad(act, z, s["dy"][a:b].float(), n)
            dx[a:b] = (dz @ wg).to(dt)
            (dw[g] if grouped else dw).copy_((dz.t() @ xg).to(dt))
            if case["bias"]:
                (db[g] if grouped else db).copy_(dz.sum(0).to(dt))
    if res is not None:
        y = y + res.float()
    outs = [y.to(dt)]
    if case["train"]:
        outs += [t for t in (dx, dw, db) if t is not None]
        if res is not None:
            outs.append(s["dy"])
    return outs


def exact(case, seed):
    """The definition in 64 bits; the gradients are torch's own differentiation of it, group by
    group."""
    s = prepare(case, seed)
    f64 = torch.float64

    def wide(t):
        return None if t is None else t.detach().to(f64)

    act, n, train = case["act"], case["n"], case["train"]
    x, res = wide(s["x"]), wide(s["residual"])
    grouped = case["op"] == "grouped"
    bounds = s["bounds"] if grouped else [0, case["rows"]]
    y = torch.zeros((case["rows"], n), dtype=f64, device=x.device) if res is None else res.clone()
    if train:
        dx = torch.zeros_like(x)
        dw = torch.zeros(s["weight"].shape, dtype=f64, device=x.device)
        db = torch.zeros(s["bias"].shape, dtype=f64, device=x.device) if case["bias"] else None
    functions = {
        "none": lambda z: z,
        "relu": torch.relu,
        "gelu": lambda z: z * torch.special.ndtr(z),
        "gelu_tanh": lambda z: z * torch.sigmoid(math.sqrt(8.0 / math.pi) * (z + 0.044715 * z ** 3)),
        "silu": lambda z: z * torch.sigmoid(z),
        "swiglu": lambda z: z[:, :n] * torch.sigmoid(z[:, :n]) * z[:, n:],
    }
    for g, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if a == b:
            continue
        at = s["host_slots"][g] if case["pages"] else g
        leaves = [x[a:b].clone(), wide(s["weight"][at] if grouped else s["weight"])]
        if case["bias"]:
            leaves.append(wide(s["bias"][at] if grouped else s["bias"]))
        if train:
            for t in leaves:
                t.requires_grad_()
        z = torch.matmul(leaves[0], leaves[1].t())
        if case["bias"]:
            z = z + leaves[2]
        out = functions[act](z)
        y[a:b] += out.detach()
        if train:
            grads = torch.autograd.grad(out, leaves, wide(s["dy"][a:b]))
            dx[a:b] = grads[0]
            (dw[g] if grouped else dw).copy_(grads[1])
            if case["bias"]:
                (db[g] if grouped else db).copy_(grads[2])
    outs = [y]
    if train:
        outs += [t for t in (dx, dw, db) if t is not None]
        if res is not None:
            outs.append(wide(s["dy"]))
    return outs


def work(case):
    rows, k, n, wr = case["rows"], case["k"], case["n"], _weight_rows(case)
    used = rows - case["spare"]
    groups = case["groups"]
    active = used if used <= groups else groups * (1.0 - (1.0 - 1.0 / groups) ** used) if groups > 1 else 1
    size = 4 if case["dtype"] == "fp32" else 2
    weights = active * wr * (k + case["bias"])
    elems = used * k + weights + rows * n * (1 + case["residual"])
    flops = 2.0 * used * k * wr
    if case["train"]:
        # dy in, the gradients out (those of weights without rows too); the residual's is dy
        elems += rows * n + rows * k + groups * wr * (k + case["bias"])
        flops *= 3
    return {"bytes": int(elems * size), "flops": int(flops)}

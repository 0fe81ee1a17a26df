"""dispatch_rows and combine_rows against the 64-bit reference, and a whole block of the operators together."""
import threading

import pytest
import torch
import torch.utils.checkpoint

from ae_amd._lib import SmxError
from ae_amd.layers import (combine_rows, dispatch_rows, fused_linear, grouped_linear, layer_norm, rms_norm, route_experts,
                           stack_fused_moe)
from tests.block_ref import F64, combine, order_of
from tests.helpers import make_pool
from tests.product_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _places(tokens, k, experts=8, idle=0.0, seed=1):
    g = _gen(seed + tokens)
    ids = torch.randint(0, experts, (tokens, k), generator=g, device=DEV)
    ids[torch.rand((tokens, k), generator=g, device=DEV) < idle] = -1
    return order_of(ids, experts)[:2]


def _check_dispatch(x, places, order, dy=None):
    k = places.shape[1]
    leaf = x.detach().requires_grad_(dy is not None)
    rows = dispatch_rows(leaf, places)
    want = torch.where((order < 0)[:, None], 0.0, x[order.clamp_min(0).long() // k]).to(x.dtype)
    assert rows.dtype == x.dtype and torch.equal(rows.detach(), want)
    if dy is not None:
        (dx,) = torch.autograd.grad([rows], [leaf], [dy])
        check(dx, *combine(dy, places, None, None, x.dtype)["y"], what="dx")
        return [rows.detach(), dx]
    return [rows]


def _check_combine(rows, places, weights, residual, dy=None):
    named = {"rows": rows, "w": weights, "r": residual}
    leaves = {n: t.detach().requires_grad_(dy is not None) for n, t in named.items() if t is not None}
    y = combine_rows(leaves["rows"], places, leaves.get("w"), leaves.get("r"))
    ref = combine(rows, places, weights, residual, rows.dtype, dy)
    assert y.dtype == rows.dtype
    check(y.detach(), *ref["y"], what="y")
    if dy is None:
        return [y]
    got = dict(zip(leaves, torch.autograd.grad([y], list(leaves.values()), [dy])))
    check(got["rows"], *ref["drows"], what="drows")
    if weights is not None:
        check(got["w"], *ref["dw"], what="dw")
    if residual is not None:
        assert torch.equal(got["r"], dy)
    return [y.detach(), *got.values()]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 64, 100, 128, 333, 1024, 2048, 2056, 4097, 8192])
def test_widths(cols, dtype):
    tokens, k = 19, 3
    g = _gen(cols)
    places, order = _places(tokens, k)
    x, dy = _randn(g, tokens, cols, dtype=dtype), _randn(g, tokens * k, cols, dtype=dtype)
    _check_dispatch(x, places, order, dy)
    w = torch.rand((tokens, k), generator=g, device=DEV)
    _check_combine(dy, places, w, x, x)
    _check_combine(dy, places, w, None, x)
    _check_combine(dy, places, None, x, x)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 6, 8, 9, 16])
@pytest.mark.parametrize("tokens", [1, 2, 33, 2050])
def test_tokens_and_picks(tokens, k, dtype):
    """A workgroup a token and a wave a token, every count of picks; picks of nobody among them."""
    for idle in (0.0, 0.3, 1.0):
        places, order = _places(tokens, k, idle=idle)
        g = _gen(tokens + k)
        x, rows = _randn(g, tokens, 192, dtype=dtype), _randn(g, tokens * k, 192, dtype=dtype)
        _check_dispatch(x, places, order, rows)
        _check_combine(rows, places, torch.rand((tokens, k), generator=g, device=DEV), x, x)


def test_rows_of_nobody_are_not_looked_at():
    """NaN in rows of nobody and in their weights reaches nothing; their gradients are zeros."""
    places, order = _places(40, 4, idle=0.4)
    g = _gen(3)
    rows, dy = _randn(g, 160, 72, dtype=BF16), _randn(g, 40, 72, dtype=BF16)
    w = torch.rand((40, 4), generator=g, device=DEV)
    clean = _check_combine(rows, places, w, None, dy)
    rows[order < 0] = NAN
    w[places < 0] = NAN
    leaves = [rows.requires_grad_(), w.requires_grad_()]
    y = combine_rows(rows, places, w)
    assert torch.equal(y.detach(), clean[0])
    drows, dw = torch.autograd.grad([y], leaves, [dy])
    assert torch.equal(drows, clean[1]) and torch.equal(dw, clean[2])
    assert not drows[order < 0].any() and not dw[places < 0].any()


def test_a_row_stays_its_own():
    places, _ = _places(30, 3)
    rows, dy = _randn(_gen(4), 90, 40), _randn(_gen(5), 30, 40)
    w = torch.rand((30, 3), generator=_gen(6), device=DEV)
    clean = _check_combine(rows, places, w, None, dy)
    rows = rows.clone()
    rows[int(places[7, 1]), 5] = NAN
    y = combine_rows(rows, places, w)
    keep = torch.arange(30, device=DEV) != 7
    assert torch.equal(y[keep], clean[0][keep]) and y[7, 5].isnan() and y[7].isnan().sum() == 1


def test_places_outside_are_left_out():
    """Places past the last row are no rows: nothing outside the tensors is read or written."""
    places, order = _places(20, 2)
    places[3, 1], places[4, 0], places[5, 0] = 40, 2 ** 31 - 1, -2 ** 31
    room = torch.full((60, 24), 7.0, device=DEV)
    rows = room[10:50]
    rows.copy_(_randn(_gen(1), 40, 24))
    w = torch.rand((20, 2), generator=_gen(2), device=DEV)
    check(combine_rows(rows, places, w), *combine(rows, places, w, None, F32)["y"])
    leaves = [rows.detach().clone().requires_grad_(), w.clone().requires_grad_()]
    y = combine_rows(leaves[0], places, leaves[1])
    _, dw = torch.autograd.grad([y], leaves, [torch.ones_like(y)])
    assert float(dw[3, 1]) == float(dw[4, 0]) == float(dw[5, 0]) == 0.0
    got = dispatch_rows(w, places)  # (rows that no place holds are not written)
    at = torch.tensor([int(p) for p in places.flatten().tolist() if 0 <= p < 40], device=DEV)
    tok = torch.tensor([i // 2 for i, p in enumerate(places.flatten().tolist()) if 0 <= p < 40], device=DEV)
    assert torch.equal(got[at], w[tok])
    assert (room[:10] == 7).all() and (room[50:] == 7).all()


def test_strides():
    g = _gen(9)
    places, order = _places(25, 2)
    for dtype in (BF16, F32):
        wide, rows = _randn(g, 25, 200, dtype=dtype), _randn(g, 50, 208, dtype=dtype)
        for lo in (0, 1, 8):
            _check_dispatch(wide[:, lo:lo + 96], places, order, rows[:, lo:lo + 96])
            w = torch.rand((2, 25), generator=g, device=DEV).t()
            _check_combine(rows[:, lo:lo + 96], places, w, wide[:, 64:160], wide[:, lo:lo + 96])
        _check_dispatch(_randn(g, 96, 25, dtype=dtype).t(), places, order, rows[:1, :96].expand(50, 96))
        _check_combine(_randn(g, 96, 50, dtype=dtype).t(), places, None, wide[:1, :96].expand(25, 96), wide[:1, :96].expand(25, 96))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty_batches(dtype):
    places = torch.empty((0, 3), dtype=torch.int32, device=DEV)
    x = torch.empty((0, 16), dtype=dtype, device=DEV, requires_grad=True)
    w = torch.empty((0, 3), device=DEV, requires_grad=True)
    rows = dispatch_rows(x, places)
    y = combine_rows(rows, places, w, x)
    assert rows.shape == y.shape == (0, 16)
    dx, dw = torch.autograd.grad([y], [x, w], [torch.empty_like(y)])
    assert dx.shape == (0, 16) and dw.shape == (0, 3)


def test_offsets_beyond_4_gib():
    """Rows whose elements lie past 2^31."""
    tokens, k, cols = 70000, 8, 4096
    places = torch.arange(tokens * k, dtype=torch.int32, device=DEV).flip(0).view(tokens, k)
    x = _randn(_gen(1), 64, cols, dtype=BF16).repeat(tokens // 64 + 1, 1)[:tokens]
    rows = dispatch_rows(x, places)
    for t in (0, 1, tokens // 2, tokens - 1):
        assert all(torch.equal(rows[int(p)], x[t]) for p in places[t])
    w = torch.full((tokens, k), 0.125, device=DEV)
    assert torch.equal(combine_rows(rows, places, w), x)  # the mean of eight equal rows
    leaf = w.requires_grad_()
    (dw,) = torch.autograd.grad([combine_rows(rows, places, leaf)], [leaf], [x])
    want = (x[:64].double() ** 2).sum(1)
    for t in (0, tokens - 1):
        check(dw[t], want[t % 64].expand(k), (cols + 24) * 2.0 ** -24 * want[t % 64].expand(k))


def test_repeated_calls_agree_bit_for_bit():
    places, order = _places(3000, 6, 64)
    rows, dy = _randn(_gen(1), 18000, 264, dtype=BF16), _randn(_gen(2), 3000, 264, dtype=BF16)
    w = torch.rand((3000, 6), generator=_gen(3), device=DEV)
    runs = [_check_combine(rows, places, w, dy, dy) + _check_dispatch(dy, places, order, rows) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_gradients_against_differences():
    """The sums are linear in each operand: differences are exact up to the loss's rounding."""
    places, _ = _places(12, 3, idle=0.2)
    g = _gen(8)
    named = [_randn(g, 36, 20), torch.rand((12, 3), generator=g, device=DEV), _randn(g, 12, 20)]
    dy = _randn(g, 12, 20)
    leaves = [t.clone().requires_grad_() for t in named]
    grads = torch.autograd.grad([combine_rows(leaves[0], places, leaves[1], leaves[2])], leaves, [dy])
    for i, grad in enumerate(grads):
        way = _randn(g, *named[i].shape)
        loss = []
        for step in (0.5, -0.5):
            rows, w, r = [v + step * way if j == i else v for j, v in enumerate(named)]
            loss.append(float((combine_rows(rows, places, w, r).to(F64) * dy.to(F64)).sum()))
        # 240 terms of some units, off by 2^-22 each
        assert abs(loss[0] - loss[1] - float((grad.to(F64) * way.to(F64)).sum())) < 240 * 16 * 2.0 ** -22


def test_differentiable_once_and_moved_tensors():
    places, _ = _places(20, 2)
    x = _randn(_gen(1), 20, 32).requires_grad_()
    w = torch.rand((20, 2), generator=_gen(2), device=DEV).requires_grad_()
    dy = _randn(_gen(3), 20, 32)
    want = torch.autograd.grad(combine_rows(dispatch_rows(x, places), places, w, x), [x, w], [dy])
    with torch.autograd.graph.save_on_cpu():
        y = combine_rows(dispatch_rows(x, places), places, w, x)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, [x, w], [dy]), want))
    # the gradients depend on the outputs' gradients, those of the weights and rows on each other
    for y, leaf in ((combine_rows(dispatch_rows(x.detach(), places), places, w), w), (dispatch_rows(x, places), x)):
        dy = torch.ones_like(y, requires_grad=True)
        (d,) = torch.autograd.grad(y, [leaf], [dy], create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(d.sum(), [dy])
    rows = dispatch_rows(x.detach(), places).requires_grad_()
    y = combine_rows(rows, places, w)
    (d,) = torch.autograd.grad(y, [rows], [torch.ones_like(y)], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(d.sum(), [w])


def test_refusals_on_the_gpu():
    x, p = torch.zeros(4, 8, device=DEV), torch.zeros(4, 17, dtype=torch.int32, device=DEV)
    with pytest.raises(SmxError, match="supported"):
        dispatch_rows(x, p)
    with pytest.raises(SmxError, match="supported"):
        combine_rows(torch.zeros(68, 8, device=DEV), p)
    with pytest.raises(ValueError, match="places is on"):
        dispatch_rows(x, p.cpu())
    with pytest.raises(ValueError, match="weights on"):
        combine_rows(x[:4], p[:2, :2].contiguous(), torch.zeros(2, 2))


# ---- together ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens", [1, 9, 150])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_expert_block_beside_the_fused_one(tokens, dtype):
    """Routing, dispatch, grouped products over the pool's pages and combine: the fused operator's result."""
    E, H, I, k = 8, 256, 128, 2
    pool, slots = make_pool(E, H, I, dtype, num_slots=10, seed=4)
    x = _randn(_gen(tokens), tokens, H, dtype=dtype)
    logits = _randn(_gen(7), tokens, E, dtype=dtype, scale=2.0)
    r = route_experts(logits, k)
    rows = dispatch_rows(x, r.places)
    h = grouped_linear(rows, pool[:, :2 * I * H].unflatten(1, (2 * I, H)), r.offsets, activation="swiglu", weight_slots=slots)
    d = grouped_linear(h, pool[:, 2 * I * H:].unflatten(1, (H, I)), r.offsets, weight_slots=slots)
    got = combine_rows(d, r.places, r.weights).to(F64)
    want = stack_fused_moe(x, pool, slots, logits, r.weights, r.ids, True).to(F64)
    # both round gate, up (the fused operator only), their product, the terms and the sum: about 6 roundings of u each
    # on sums whose terms are all as large as the largest output
    u = torch.finfo(dtype).eps / 2
    assert float((got - want).abs().max()) <= (12 * u + 2e-5) * float(want.abs().max())


def _block(norm, x, r, w, k, scoring, bias):
    """A pre-norm mixture-of-experts block with a residual stream."""
    s = None
    if norm == "rms":
        y, s = rms_norm(x, w["norm"], 1e-6, residual=r)
    else:
        y, s = layer_norm(x, w["norm"], w["shift"], 1e-6, residual=r)
    logits = fused_linear(y, w["gate"])
    p = route_experts(logits, k, scoring, bias, scale=1.5)
    h = grouped_linear(dispatch_rows(y, p.places), w["up"], p.offsets, activation="swiglu")
    return combine_rows(grouped_linear(h, w["down"], p.offsets), p.places, p.weights, residual=s), p


def _block64(norm, x, r, w, ids, scoring):
    s = x + r
    if norm == "rms":
        y = s * torch.rsqrt(s.square().mean(1, keepdim=True) + 1e-6) * w["norm"]
    else:
        y = torch.nn.functional.layer_norm(s, s.shape[1:], w["norm"], w["shift"], 1e-6)
    logits = y @ w["gate"].t()
    score = torch.softmax(logits, 1) if scoring == "softmax" else torch.sigmoid(logits)
    p = score.gather(1, ids)
    p = 1.5 * p / p.sum(1, keepdim=True)
    half = w["up"].shape[1] // 2
    out = s
    for j in range(ids.shape[1]):
        up, down = w["up"][ids[:, j]], w["down"][ids[:, j]]
        z = torch.matmul(up, y[:, :, None])[:, :, 0]
        h = torch.nn.functional.silu(z[:, :half]) * z[:, half:]
        out = out + p[:, j:j + 1] * torch.matmul(down, h[:, :, None])[:, :, 0]
    return out


@pytest.mark.parametrize("norm,scoring", [("rms", "softmax"), ("layer", "sigmoid")])
@pytest.mark.parametrize("tokens", [1, 70])
def test_trained_block_together(norm, scoring, tokens):
    """Norm, router, dispatch, experts and combine differentiated together, against torch in 64 bits on the CPU."""
    H, I, E, k = 96, 64, 8, 3
    g = _gen(11)
    w = {"norm": _randn(g, H, scale=0.2) + 1, "shift": _randn(g, H, scale=0.1), "gate": _randn(g, E, H, scale=0.2),
         "up": _randn(g, E, 2 * I, H, scale=0.1), "down": _randn(g, E, H, I, scale=0.1)}
    if norm == "rms":
        del w["shift"]
    x, r, dy = (_randn(g, tokens, H) for _ in range(3))
    bias = _randn(g, E, scale=0.1) if scoring == "sigmoid" else None
    leaves = [t.requires_grad_() for t in (x, r, *w.values())]
    y, p = _block(norm, x, r, w, k, scoring, bias)
    got = torch.autograd.grad(y, leaves, dy)
    host = [t.detach().double().cpu().requires_grad_() for t in leaves]
    want = _block64(norm, host[0], host[1], dict(zip(w, host[2:])), p.ids.long().cpu(), scoring)
    grads = torch.autograd.grad(want, host, dy.double().cpu())
    # fp32 sums of up to 192 terms through six layers, on the largest output or gradient: 6 * 192 * 2^-24
    bound = 6 * 192 * 2.0 ** -24
    check(y.detach().cpu(), want.detach(), torch.full_like(want.detach(), bound * float(want.detach().abs().max())))
    for name, a, b in zip(("x", "r", *w), got, grads):
        assert float((a.double().cpu() - b).abs().max()) <= bound * float(b.abs().max()), name


@pytest.mark.parametrize("tokens", [5, 400])
def test_captured_block(tokens):
    """The whole block's training step in a graph, replayed over new inputs (and new loads) between eager calls."""
    H, I, E, k = 128, 64, 8, 2
    g = _gen(12)
    w = {"norm": (_randn(g, H, scale=0.2) + 1).to(BF16), "gate": _randn(g, E, H, scale=0.2, dtype=BF16),
         "up": _randn(g, E, 2 * I, H, scale=0.1, dtype=BF16), "down": _randn(g, E, H, I, scale=0.1, dtype=BF16)}
    x, r, dy = (_randn(g, tokens, H, dtype=BF16) for _ in range(3))
    leaves = [t.requires_grad_() for t in (x, r, *w.values())]

    def step():
        y, p = _block("rms", x, r, w, k, "softmax", None)
        return [y.detach(), p.ids, *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(_randn(_gen(90 + i), tokens, H, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i


def test_block_checkpointed_and_accumulated():
    """Recomputed in the backward pass, and twice into the same gradients: what one pass gives, twice."""
    H, I, E, k, tokens = 64, 32, 4, 2, 33
    g = _gen(15)
    w = {"norm": _randn(g, H, scale=0.2) + 1, "gate": _randn(g, E, H, scale=0.2), "up": _randn(g, E, 2 * I, H, scale=0.1),
         "down": _randn(g, E, H, I, scale=0.1)}
    x, r, dy = (_randn(g, tokens, H) for _ in range(3))
    leaves = [t.requires_grad_() for t in (x, r, *w.values())]

    def block(x, r):
        return _block("rms", x, r, w, k, "softmax", None)[0]

    want = torch.autograd.grad(block(x, r), leaves, dy)
    for _ in range(2):
        torch.utils.checkpoint.checkpoint(block, x, r, use_reentrant=False).backward(dy)
    for t, v in zip(leaves, want):
        assert torch.equal(t.grad, 2 * v)


def test_threads_at_once():
    """Blocks of several Python threads, each on a stream of its own."""
    H, E, k = 128, 16, 4
    up, down = _randn(_gen(1), E, 64, H, scale=0.1), _randn(_gen(2), E, H, 32, scale=0.1)
    inputs = [(_randn(_gen(10 + i), 200 + i, H), _randn(_gen(20 + i), 200 + i, E), _randn(_gen(30 + i), 200 + i, H)) for i in range(4)]

    def step(i):
        x, logits, dy = (t.detach().requires_grad_(j < 2) for j, t in enumerate(inputs[i]))
        y, s = layer_norm(x, residual=x)
        p = route_experts(logits, k)
        h = grouped_linear(dispatch_rows(y, p.places), up, p.offsets, activation="swiglu")
        out = combine_rows(grouped_linear(h, down, p.offsets), p.places, p.weights, residual=s)
        return [out.detach(), *torch.autograd.grad(out, [x, logits], dy)]

    want = [step(i) for i in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = step(i)
            stream.synchronize()
        except Exception as e:  # (shown in the main thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_padded_batch():
    """Padding rows of -inf logits: no expert sees them, the residual passes them on, no gradient enters them."""
    H, I, E, k, tokens, pad = 64, 32, 4, 2, 50, 13
    g = _gen(14)
    up, down = _randn(g, E, 2 * I, H, scale=0.1).requires_grad_(), _randn(g, E, H, I, scale=0.1).requires_grad_()
    y, res, dy = (_randn(g, tokens, H) for _ in range(3))
    logits = _randn(g, tokens, E)
    logits[tokens - pad:] = -float("inf")
    y[tokens - pad:] = NAN

    def block(y, logits, res):
        p = route_experts(logits, k)
        h = grouped_linear(dispatch_rows(y, p.places), up, p.offsets, activation="swiglu")
        return combine_rows(grouped_linear(h, down, p.offsets), p.places, p.weights, residual=res), p

    a = [t.detach().requires_grad_() for t in (y, logits, res)]
    out, p = block(*a)
    assert int(p.offsets[-1]) == (tokens - pad) * k
    assert torch.equal(out.detach()[tokens - pad:], res[tokens - pad:])
    got = torch.autograd.grad(out, [*a, up, down], dy)
    b = [t.detach()[:tokens - pad].clone().requires_grad_() for t in (y, logits, res)]
    out2, _ = block(*b)
    want = torch.autograd.grad(out2, [*b, up, down], dy[:tokens - pad])
    # the same products, perhaps split otherwise: sums of up to 74 terms through three layers, on the largest value
    pairs = [(out.detach()[:tokens - pad], out2.detach()), *((t[:tokens - pad], v) for t, v in zip(got[:3], want[:3])),
             *zip(got[3:], want[3:])]
    for t, v in pairs:
        assert float((t - v).abs().max()) <= 2 * 3 * 74 * 2.0 ** -24 * float(v.abs().max())
    assert not got[0][tokens - pad:].any() and not got[1][tokens - pad:].any()


def _need(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of GPU memory")


def test_tokens_beyond_a_grid_s_threads():
    """A wave a token in the weights' gradient: 2^32 threads and more. Small whole numbers, so all results are exact."""
    _need(40)
    tokens = (1 << 26) + 5
    at = torch.arange(tokens - 1, -1, -1, device=DEV)
    rows = ((at[:, None] * torch.arange(1, 9, device=DEV)) % 7 - 3).to(BF16).requires_grad_()
    w = ((at % 3) + 1).float()[:, None].requires_grad_()
    y = combine_rows(rows, at.int()[:, None], w)
    dy = ((at[:, None] + torch.arange(8, device=DEV)) % 5 - 2).to(BF16)
    drows, dw = torch.autograd.grad([y], [rows, w], [dy])
    with torch.no_grad():
        assert torch.equal(y, rows.flip(0) * w.to(BF16))
        assert torch.equal(drows, (dy * w.to(BF16)).flip(0))
        assert torch.equal(dw[:, 0], (rows.flip(0).float() * dy.float()).sum(1))
    (only,) = torch.autograd.grad([combine_rows(rows, at.int()[:, None], w.detach())], [rows], [dy])
    assert torch.equal(only, drows)


def test_wide_rows_beyond_a_grid_s_threads():
    """A workgroup a token where rows are wide."""
    _need(120)
    tokens, cols = (1 << 24) + 3, 1032
    at = torch.arange(tokens - 1, -1, -1, device=DEV)
    tag = (at % 251).to(BF16)[:, None]
    x = torch.empty((tokens, cols), dtype=BF16, device=DEV)
    x.copy_(tag)
    x[:, -1] = 1.0
    rows = dispatch_rows(x, at.int()[:, None])
    want = tag.flip(0).expand(tokens, cols - 1)
    assert all(torch.equal(rows[i:i + (1 << 20), :-1], want[i:i + (1 << 20)]) for i in range(0, tokens, 1 << 20))
    assert bool((rows[:, -1] == 1.0).all())
    x.zero_()
    del x
    y = combine_rows(rows, at.int()[:, None])
    want = tag.expand(tokens, cols - 1)
    assert all(torch.equal(y[i:i + (1 << 20), :-1], want[i:i + (1 << 20)]) for i in range(0, tokens, 1 << 20))
    assert bool((y[:, -1] == 1.0).all())
    del rows, y, want
    torch.cuda.empty_cache()


def test_signs_kept_in_a_flag():
    """The imaginary part of a conjugate is the memory's numbers with the other sign."""
    g = _gen(3)
    z = torch.complex(_randn(g, 12, 1), _randn(g, 12, 1))
    column = z.conj().imag
    assert column.is_neg()
    places, order = _places(12, 2)
    assert torch.equal(dispatch_rows(column, places), dispatch_rows(-z.imag, places))

    x, r, w, b, dy, rows, dr = (_randn(g, *s) for s in ((12, 64), (12, 64), (64,), (64,), (12, 64), (24, 64), (24, 64)))
    share = torch.rand((12, 2), generator=g, device=DEV)

    def grads(call, leaves, given):
        leaves = [t.detach().requires_grad_() for t in leaves]
        outs = call(*leaves)
        outs = outs if isinstance(outs, tuple) else (outs,)
        return [*outs, *torch.autograd.grad(outs, leaves, given)]

    for call, leaves, given in ((lambda x, r, w: rms_norm(x, w, residual=r), (x, r, w), (dy, x)),
                                (lambda x, w, b: layer_norm(x, w, b), (x, w, b), (dy,)),
                                (lambda x: route_experts(x, 2, "sigmoid", torch._neg_view(-w)).weights, (x,), (share,)),
                                (lambda x: dispatch_rows(x, places), (x,), (dr,)),
                                (lambda x, s, r: combine_rows(x, places, s, r), (rows, share, r), (dy,))):
        want = grads(call, leaves, given)
        got = grads(call, [torch._neg_view(-t) for t in leaves], [torch._neg_view(-t) for t in given])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    with pytest.raises(TypeError, match="places"):
        dispatch_rows(x, torch._neg_view(-places))

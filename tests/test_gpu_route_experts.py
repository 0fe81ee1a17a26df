"""route_experts against the 64-bit reference: choices and order exactly, weights and gradients within bounds."""
import itertools

import pytest
import torch

from ae_amd import _lib
from ae_amd._lib import SmxError
from ae_amd.layers import route_experts, select_experts
from tests.block_ref import F64, INF, choose, order_of, route, scores
from tests.product_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(t, e, dtype=F32, scale=1.5, seed=0):
    return (torch.randn((t, e), generator=_gen(seed + 7 * t + e), device=DEV) * scale).to(dtype)


def _check(logits, k, scoring="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0, train=True,
           what=""):
    top = groups if top_groups is None else top_groups
    leaf = logits.detach().requires_grad_(train)
    r = route_experts(leaf, k, scoring, bias, groups, top_groups, renormalize, scale)
    ids = choose(logits, k, scoring, bias, groups, top)
    assert r.ids.dtype == torch.int32 and torch.equal(r.ids.long(), ids), what
    for got, want in zip((r.places, r.order, r.offsets), order_of(r.ids, logits.shape[1])):
        assert got.dtype == want.dtype and torch.equal(got, want), what
    dw = torch.randn(r.weights.shape, generator=_gen(5), device=DEV) if train else None
    ref = route(logits, ids, scoring, renormalize, scale, dw)
    check(r.weights.detach(), *ref["weights"], what=f"{what} weights")
    if not train:
        return [*r]
    (d,) = torch.autograd.grad([r.weights], [leaf], [dw])
    assert d.dtype == logits.dtype
    check(d, *ref["dlogits"], what=f"{what} dlogits")
    return [r.weights.detach(), *r[1:], d]


# every width of the kernels' lanes and experts, on both sides of each border
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("experts,k", [(1, 1), (2, 2), (8, 2), (15, 3), (16, 16), (17, 4), (60, 4), (64, 6), (65, 5), (128, 8), (130, 1),
                                       (160, 6), (255, 16), (256, 8), (257, 7), (384, 8), (512, 10), (513, 2), (1000, 16), (1024, 8)])
def test_experts(experts, k, dtype):
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            _check(_logits(37, experts, dtype), k, scoring, renormalize=renormalize, scale=2.5, what=f"{scoring} {renormalize}")


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 15, 16, 17, 63, 85, 86, 87, 333, 1025, 8191, 8193, 20001])
def test_tokens(tokens):
    """One workgroup, many, several steps of each."""
    bias = torch.randn(64, generator=_gen(1), device=DEV) * 0.1
    _check(_logits(tokens, 64), 6, renormalize=False)
    _check(_logits(tokens, 64, BF16), 6, "sigmoid", bias, 8, 3)
    _check(_logits(tokens, 300, BF16), 9)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("experts,k,groups,top_groups", [(65, 5, 1, 1), (65, 5, 13, 3), (100, 16, 1, 1), (128, 8, 8, 3), (130, 1, 1, 1),
                                                         (160, 6, 8, 3), (255, 16, 17, 4), (256, 8, 1, 1), (256, 8, 8, 4),
                                                         (256, 16, 64, 9), (256, 2, 2, 1)])
def test_experts_of_many_tokens(experts, k, groups, top_groups, dtype):
    """Several tokens a wave, where few tokens have one each."""
    logits = _logits(1100, experts, dtype)
    logits[200] = 0.0
    logits[300:310] = -INF
    bias = torch.randn(experts, generator=_gen(experts), device=DEV) * 0.2
    for scoring in ("softmax", "sigmoid"):
        for b in (None, bias, torch.zeros(experts, device=DEV)):
            _check(logits, k, scoring, b, groups, top_groups, renormalize=b is not None, scale=1.5)


@pytest.mark.parametrize("experts", [100, 256])
@pytest.mark.parametrize("k", [1, 7, 16])
def test_near_choices_of_many_tokens(experts, k):
    g = _gen(experts + k)
    logits = _logits(1, experts)
    step = torch.randint(0, experts // 3 + 1, (experts,), generator=g, device=DEV).double() / 8
    bias = (step - torch.sigmoid(logits[0].double())).float()
    other = (step - torch.softmax(logits[0].double(), 0)).float()
    logits = logits + torch.randn((1100, experts), generator=g, device=DEV) * 1e-7
    for groups, top_groups in ((1, 1), (4, 2)):
        _check(logits, k, "sigmoid", bias, groups, top_groups)
        _check(logits, k, "softmax", other, groups, top_groups)
    _check((logits * 2 ** 20).round() / 2 ** 20, k)  # and plain ones that lie close or tie


def test_many_tokens():
    """More workgroups than hold all tokens' ranks at one step each."""
    _check(_logits(140001, 20, BF16), 16)
    _check(_logits(300007, 8), 2, "sigmoid")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(8, 2, 1, 3), (12, 4, 2, 5), (64, 8, 3, 6), (64, 64, 7, 7), (160, 8, 3, 6),
                                                         (256, 8, 4, 8), (255, 17, 4, 8), (256, 64, 9, 8), (320, 5, 2, 16), (512, 8, 4, 8),
                                                         (1024, 64, 3, 16), (18, 6, 6, 4)])
def test_groups(experts, groups, top_groups, k, dtype):
    bias = torch.randn(experts, generator=_gen(experts), device=DEV) * 0.2
    logits = _logits(200, experts, dtype)
    for scoring in ("softmax", "sigmoid"):
        _check(logits, k, scoring, None, groups, top_groups)
        if experts > groups:
            _check(logits, k, scoring, bias, groups, top_groups, renormalize=False, scale=0.5)
    _check(logits, k, "sigmoid", bias, groups, top_groups, renormalize=True)


def test_a_group_of_one():
    """With a bias too, a group of one expert ranks by that expert."""
    bias = torch.randn(32, generator=_gen(2), device=DEV)
    _check(_logits(50, 32), 3, "sigmoid", bias, 32, 5)


@pytest.mark.parametrize("experts", [16, 64, 256, 512])
def test_ties(experts):
    """Equal choices go to the lower expert: few distinct logits, no bias, one bias for all, and few distinct biases."""
    g = _gen(experts)
    logits = torch.randint(0, 4, (300, experts), generator=g, device=DEV).float()
    bias = torch.randint(0, 3, (experts,), generator=g, device=DEV).float() * 0.25
    for scoring in ("softmax", "sigmoid"):
        for b in (None, torch.zeros(experts, device=DEV), bias):
            _check(logits, 8, scoring, b)
            _check(logits, 8, scoring, b, 8, 4)
            _check(logits.repeat(4, 1), 8, scoring, b, 8, 4)
    _check(torch.zeros(20, experts, device=DEV), 8, "sigmoid", torch.zeros(experts, device=DEV), 4, 2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("experts,groups,top_groups", [(16, 8, 2), (64, 1, 1), (64, 8, 3), (256, 8, 4), (160, 8, 3), (512, 8, 4)])
def test_a_router_of_zeros(experts, groups, top_groups, dtype):
    """Every choice of every token ties: the first experts of the first groups."""
    logits = torch.zeros((500, experts), dtype=dtype, device=DEV)
    size = experts // groups
    k = min(8, size * top_groups)
    for bias in (None, torch.zeros(experts, device=DEV)):
        for scoring in ("softmax", "sigmoid"):
            out = _check(logits, k, scoring, bias, groups, top_groups)
            assert (out[1] == torch.arange(k, device=DEV, dtype=torch.int32)).all()


@pytest.mark.parametrize("k", [1, 2, 15, 16])
@pytest.mark.parametrize("experts", [16, 60, 256, 300])
def test_near_choices(experts, k):
    """Runs of choices that 32 bits cannot tell apart, inside the picks, across their end and past it."""
    g = _gen(experts + k)
    logits = _logits(64, experts)
    score = torch.sigmoid(logits[0].double())
    step = torch.randint(0, experts // 3 + 1, (experts,), generator=g, device=DEV).double() / 8
    bias = (step - score).float()  # the choices of a step lie within some 2^-25
    logits = logits[:1] + torch.randn((64, experts), generator=g, device=DEV) * 1e-7
    _check(logits, k, "sigmoid", bias)
    _check(logits, k, "softmax", (step - torch.softmax(logits[0].double(), 0)).float())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_choices_that_32_bits_cannot_tell_apart(scoring, groups, top_groups):
    """Biases that make the choices of all experts equal but for some 1e-9: the exact scores decide."""
    experts, tokens = 64, 40
    logits = _logits(1, experts, scale=0.7)
    x = logits.double()
    score = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
    bias = (1.0 - score[0]).float()  # off by up to 2^-25 each, which now decides
    logits = logits.repeat(tokens, 1)
    if scoring == "sigmoid":
        logits[1:] += torch.randn((tokens - 1, experts), generator=_gen(3), device=DEV) * 1e-6
    _check(logits, 6, scoring, bias, groups, top_groups)
    large = bias + 1000.0  # and biases that leave scores only a few bits
    _check(_logits(tokens, experts), 6, scoring, large, groups, top_groups)


def test_logits_far_apart():
    """Scores that vanish in 32 bits still rank, and their ratios are the weights."""
    logits = _logits(50, 32, scale=60.0)
    bias = torch.zeros(32, device=DEV)
    bias[:8] = 5.0  # picks of vanishing scores
    for scoring in ("softmax", "sigmoid"):
        ids = choose(logits, 4, scoring, bias, 1, 1)
        r = route_experts(logits, 4, scoring, bias)
        assert torch.equal(r.ids.long(), ids)
        check(r.weights, *route(logits, ids, scoring, True, 1.0)["weights"], what=scoring)
        assert torch.isfinite(r.weights).all()
        _check(logits, 4, scoring)


def _masked(tokens, experts, dtype):
    logits = _logits(tokens, experts, dtype)
    gone = torch.rand((tokens, experts), generator=_gen(9), device=DEV) < 0.6
    logits[gone] = -INF
    logits[3] = -INF              # nobody at all
    logits[5, 1:] = -INF          # one expert
    logits[tokens - 20:] = -INF   # padding
    return logits


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [60, 700])
@pytest.mark.parametrize("experts,groups,top_groups", [(8, 1, 1), (64, 8, 2), (300, 1, 1)])
def test_masked_experts_and_rows(experts, groups, top_groups, tokens, dtype):
    logits = _masked(tokens, experts, dtype)
    bias = torch.randn(experts, generator=_gen(4), device=DEV) * 0.1
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            for b in (None, bias):
                out = _check(logits, 6, scoring, b, groups, top_groups, renormalize)
                assert (out[1][3] == -1).all() and (out[0][3] == 0).all() and not out[5][3].any()
                assert torch.isfinite(out[5]).all()


def test_a_type_s_lowest_value_is_a_logit():
    """Only -inf masks: experts of the lowest finite logit are picked where nothing better is left."""
    for dtype in (BF16, F16, F32):
        logits = torch.full((4, 16), torch.finfo(dtype).min, dtype=dtype, device=DEV)
        logits[1, 3] = 2.0
        out = _check(logits, 4, "softmax", train=False)
        assert out[1].tolist() == [[0, 1, 2, 3], [3, 0, 1, 2], [0, 1, 2, 3], [0, 1, 2, 3]]


def test_biases_of_infinity():
    bias = torch.zeros(16, device=DEV)
    bias[2], bias[5] = -INF, INF
    out = _check(_logits(30, 16), 15, "sigmoid", bias, train=False)
    assert (out[1] != 2).all() and (out[1][:, 0] == 5).all()
    out = _check(_logits(30, 16), 16, "softmax", bias, train=False)
    assert (out[1][:, 15] == -1).all()


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("biased", [True, False])
def test_a_row_stays_its_own(bad, biased):
    """A bad logit shows in its token's weights, is picked first, and reaches no other token."""
    bias = torch.zeros(64, device=DEV) if biased else None
    logits = _logits(21, 64)
    clean = route_experts(logits, 6, bias=bias)
    worse = logits.clone()
    worse[7, 40] = bad
    leaf = worse.requires_grad_()
    r = route_experts(leaf, 6, bias=bias)
    keep = torch.arange(21, device=DEV) != 7
    assert torch.equal(r.ids[keep], clean.ids[keep]) and torch.equal(r.weights.detach()[keep], clean.weights[keep])
    assert r.weights[7].isnan().all()
    assert int(r.ids[7, 0]) == (40 if not biased else 0)  # (with a bias every score of the row is NaN)
    assert len(set(r.ids[7].tolist())) == 6
    (d,) = torch.autograd.grad([r.weights], [leaf], [torch.ones_like(r.weights)])
    assert torch.isfinite(d[keep]).all() and (biased or d[7].isnan().any())
    s = route_experts(worse.detach(), 6, "sigmoid", bias, renormalize=False)
    assert int(s.ids[7, 0]) == 40 or bad == INF and biased  # (sigmoid(inf) = 1 ties with other scores of 1)
    assert torch.isfinite(s.weights[7, 1:]).all()


def test_strides():
    wide = _logits(90, 200, BF16)
    for lo, hi in ((0, 64), (8, 72), (1, 65), (3, 63), (64, 192)):
        _check(wide[:, lo:hi], 4)
    _check(_logits(64, 90).t(), 5, "sigmoid")
    _check(_logits(1, 64).expand(33, 64), 5)


def test_empty_batches():
    leaf = torch.empty((0, 40), device=DEV, requires_grad=True)
    r = route_experts(leaf, 3)
    assert r.weights.shape == r.ids.shape == r.places.shape == (0, 3) and r.order.shape == (0,)
    assert torch.equal(r.offsets, torch.zeros(41, dtype=torch.int64, device=DEV))
    (d,) = torch.autograd.grad([r.weights], [leaf], [torch.empty((0, 3), device=DEV)])
    assert d.shape == (0, 40)


def test_repeated_calls_agree_bit_for_bit():
    logits = _logits(9000, 256, BF16)
    bias = torch.randn(256, generator=_gen(6), device=DEV) * 0.1
    runs = [_check(logits, 8, "sigmoid", bias, 8, 4) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_offsets_beyond_4_gib():
    tokens, experts, pitch = 40000, 64, 65536
    buf = torch.empty((tokens, pitch), dtype=BF16, device=DEV)
    logits = buf[:, 100:100 + experts]
    logits.copy_(_logits(tokens, experts, BF16))
    _check(logits, 6)


@pytest.mark.parametrize("tokens", [1, 50, 3000])
def test_captured_training_step(tokens):
    """Forward and backward in a graph, replayed over new logits between eager calls."""
    logits = _logits(tokens, 64, BF16).requires_grad_()
    bias = torch.randn(64, generator=_gen(6), device=DEV) * 0.1
    dw = torch.randn((tokens, 6), generator=_gen(7), device=DEV)

    def step():
        r = route_experts(logits, 6, "sigmoid", bias, 8, 4)
        return [r.weights.detach(), *r[1:], *torch.autograd.grad([r.weights], [logits], [dw])]

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
            logits.copy_(_logits(tokens, 64, BF16, seed=100 + i))
            bias.copy_(torch.randn(64, generator=_gen(80 + i), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(p, q) for p, q in zip(got, step())), i


def test_two_streams_at_once():
    logits = _logits(5000, 64).requires_grad_()
    dw = torch.randn((5000, 6), generator=_gen(7), device=DEV)

    def step():
        r = route_experts(logits, 6)
        return [r.weights.detach(), *r[1:], *torch.autograd.grad([r.weights], [logits], [dw])]

    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(p, q) for p, q in zip(one, want))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradients_against_differences(scoring, renormalize):
    """Directional derivatives of the kernels' own fp32 weights, where no choice changes."""
    logits = _logits(30, 24, scale=0.5)
    logits[:, :5] += 6.0  # the picks, in any order
    dw = torch.zeros((30, 24), device=DEV)
    dw[:, :5] = torch.randn((30, 5), generator=_gen(1), device=DEV)
    h = 2.0 ** -6

    def loss(x):
        r = route_experts(x, 5, scoring, renormalize=renormalize)
        return r, (r.weights.to(F64) * dw.to(F64).gather(1, r.ids.long())).sum()

    leaf = logits.clone().requires_grad_()
    r, _ = loss(leaf)
    (d,) = torch.autograd.grad([r.weights], [leaf], [dw.gather(1, r.ids.long())])
    for i in range(3):
        way = torch.randn(logits.shape, generator=_gen(20 + i), device=DEV)
        slope = float((loss(logits + h * way)[1] - loss(logits - h * way)[1]) / (2 * h))
        want = float((d.to(F64) * way.to(F64)).sum())
        # 150 weights below 1, off by 2^-21 each: 150 * 4 * 2^-21 / (2 h) = 0.01; h^2 / 6 of third derivatives of some units
        assert abs(slope - want) < 0.01 + 150 * 4 * h * h / 6, (slope, want)


def test_two_graphs_in_one_pool():
    """Captured calls whose workspaces share memory, replayed in turn."""
    sets = [(_logits(t, e), k) for t, e, k in ((3000, 64, 6), (9000, 256, 8))]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, k in sets:
            route_experts(x, k)
    torch.cuda.current_stream().wait_stream(side)
    for x, k in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(route_experts(x, k))
        graphs.append(graph)
    for i in range(3):
        for j, (x, k) in enumerate(sets):
            x.copy_(_logits(*x.shape, seed=200 + i))
        for j, (x, k) in enumerate(sets):
            graphs[j].replay()
        torch.cuda.synchronize()
        for j, (x, k) in enumerate(sets):
            assert all(torch.equal(p, q) for p, q in zip(outs[j], route_experts(x, k))), (i, j)


@pytest.mark.parametrize("tokens", [1, 700])
def test_picks_without_an_order(tokens):
    """The C call without places, order and offsets: weights and ids alone."""
    x = _logits(tokens, 64, BF16)
    want = route_experts(x, 6, "sigmoid")
    w, ids = torch.empty_like(want.weights), torch.empty_like(want.ids)
    lib = _lib.lib()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.smx_route(x.data_ptr(), 64, 2, tokens, 64, 6, 1, None, 1, 1, 1, 1.0, w.data_ptr(), ids.data_ptr(), None, None,
                         None, None, 0, stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(w, want.weights) and torch.equal(ids, want.ids)


def test_differentiable_once_and_moved_tensors():
    logits = _logits(40, 16).requires_grad_()
    dw = torch.randn((40, 3), generator=_gen(1), device=DEV)
    (want,) = torch.autograd.grad(route_experts(logits, 3).weights, [logits], [dw])
    with torch.autograd.graph.save_on_cpu():
        r = route_experts(logits, 3)
    assert torch.equal(torch.autograd.grad(r.weights, [logits], [dw])[0], want)
    (d,) = torch.autograd.grad(route_experts(logits, 3).weights, [logits], [dw], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(d.sum(), [logits])
    assert not route_experts(logits, 3).ids.requires_grad


def test_refusals_on_the_gpu():
    x = _logits(4, 64)
    with pytest.raises(SmxError, match="supported"):
        route_experts(x, 17)
    with pytest.raises(SmxError, match="supported"):
        route_experts(_logits(2, 1025), 2)
    with pytest.raises(SmxError, match="supported"):
        route_experts(_logits(2, 130), 2, num_groups=65)
    with pytest.raises(ValueError, match="bias on"):
        route_experts(x, 2, bias=torch.zeros(64))
    with pytest.raises(ValueError, match="detached"):
        route_experts(x, 2, bias=torch.zeros(64, device=DEV, requires_grad=True))
    with torch.no_grad():
        route_experts(x, 2, bias=torch.zeros(64, device=DEV, requires_grad=True))


@pytest.mark.parametrize("renormalize", [True, False])
def test_the_serving_router_beside_it(renormalize):
    """select_experts' choice where its fp32 scores differ, and its weights within rounding."""
    logits = _logits(100, 64)
    w, ids = select_experts(logits, logits, 6, renormalize=renormalize)
    r = route_experts(logits, 6, renormalize=renormalize)
    assert torch.equal(r.ids, ids)
    # both are within the bound of the same value
    value, bound = route(logits, r.ids, "softmax", renormalize, 1.0)["weights"]
    check(r.weights, value, bound)
    check(w, value, 4 * bound)


def _few_above(tokens, experts, base, step, most, seed, dtype=F32):
    """Rows of `base`, with up to `most` experts of a row one to eight steps above it."""
    g = _gen(seed + experts)
    at = torch.rand((tokens, experts), generator=g, device=DEV).argsort(1) < torch.randint(0, most + 1, (tokens, 1), generator=g, device=DEV)
    up = torch.randint(1, 9, (tokens, experts), generator=g, device=DEV)
    return (base + torch.where(at, up, 0).double() * step).to(dtype)


def _check_near_groups(logits, k, scoring, bias, what):
    """Two of four groups, whose sums 64 bits may not tell apart.

    A score in 64 bits is off by 2^-52 of itself in exp and 2^-53 in each of the sum 1 + exp and the quotient (a softmax's
    sum is off too, but for all experts of a token alike), the sum of two by 2^-53 more: 5 * 2^-53 in all. Sums of two groups
    that differ by less than twice that, 2^-49 of them to be safe, may come out in either order, here as there (two experts 8
    and 2 steps of 1e-8 above zero, and two 6 and 4 above it, differ by 6e-16). Such tokens may take either group, and are
    few: none of the tokens whose groups lie further apart is let off."""
    ids = route_experts(logits, k, scoring, bias, 4, 2).ids.long()
    want = choose(logits, k, scoring, bias, 4, 2)
    two = torch.topk(scores(logits.to(F64), scoring).view(len(logits), 4, -1), 2, dim=2).values.sum(2)
    size = logits.shape[1] // 4
    for t in (ids != want).any(1).nonzero().flatten().tolist():
        cut = two[t].sort(descending=True).values[1]
        sure, able = two[t] > cut * (1 + 2.0 ** -49), two[t] >= cut * (1 - 2.0 ** -49)
        assert int(able.sum()) > 2, (what, scoring, t)
        ways = []
        for kept in itertools.combinations(range(4), 2):
            if all(bool(able[g]) for g in kept) and all(g in kept for g in range(4) if bool(sure[g])):
                x = logits[t:t + 1].clone()
                x.view(4, size)[[g for g in range(4) if g not in kept]] = -INF
                ways.append(choose(x, k, scoring, bias, 1, 1)[0].tolist())
        assert ids[t].tolist() in ways, (what, scoring, t)


@pytest.mark.parametrize("tokens", [150, 1100])
@pytest.mark.parametrize("k", [1, 4, 8, 16])
@pytest.mark.parametrize("experts", [16, 64, 256, 512])
def test_ties_beside_near_choices(experts, k, tokens):
    """Choices that tie across the end of the picks, and a few that are larger by less than the keys hold."""
    bias = torch.zeros(experts, device=DEV)
    for most in (1, 5, experts):
        ones = _few_above(tokens, experts, 1.0, 2.0 ** -23, most, k)
        zeros = _few_above(tokens, experts, 0.0, 1e-7 / 8, most, k + 1)
        what = f"up to {most}"
        _check(ones, k, what=what, train=False)
        for scoring in ("softmax", "sigmoid"):
            for x in (ones, zeros, zeros.to(BF16)):
                _check(x, k, scoring, bias, what=f"{what} {scoring}", train=False)
            if k <= experts // 2:
                _check(zeros, k, scoring, None, 4, 2, what=f"{what} {scoring}", train=False)
                _check_near_groups(zeros, k, scoring, bias, what)


@pytest.mark.parametrize("tokens", [500, 1500])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_routers_of_very_small_weights(dtype, tokens):
    """A balance bias as it is initialised: scores that differ by little or nothing decide."""
    for experts, k in ((256, 8), (64, 6), (512, 8), (128, 4)):
        bias = torch.zeros(experts, device=DEV)
        for spread in (1e-6, 3e-5, 1e-4, 1e-2):
            x = _logits(tokens, experts, dtype, spread)
            for scoring in ("softmax", "sigmoid"):
                _check(x, k, scoring, bias, what=f"{experts} {spread} {scoring}", train=False)
                _check(x, k, scoring, bias + 0.25, 4, 2, what=f"{experts} {spread} {scoring}", train=False)


@pytest.mark.parametrize("tokens", [1, 1100])
def test_the_one_larger_choice_behind_a_tie(tokens):
    """One expert that the list of the nearest does not hold, or holds last."""
    up = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0)).item()
    for experts, at in ((64, 63), (64, 2), (256, 255), (512, 300), (16, 15)):
        x = torch.ones((tokens, experts), device=DEV)
        x[:, at] = up
        for k in (1, 2, 6):
            assert (_check(x, k, what=f"{experts} {at} {k}", train=False)[1][:, 0] == at).all()
    zero = torch.zeros(256, device=DEV)
    x = torch.full((tokens, 256), -2.0, device=DEV, dtype=BF16)
    x[:, :9], x[:, 9] = 13.0, 13.0625  # sigmoids that saturate
    assert (_check(x, 8, "sigmoid", zero, train=False)[1][:, 0] == 9).all()
    x = torch.zeros((tokens, 64), device=DEV)
    x[:, 40] = 1e-7
    assert _check(x, 6, "sigmoid", zero[:64], train=False)[1][0].tolist() == [40, 0, 1, 2, 3, 4]
    x[:, 40] = -1e-7  # a smaller one among the ties, in front of most of them
    x[:, 2] = -1e-7
    assert _check(x, 6, "sigmoid", zero[:64], train=False)[1][0].tolist() == [0, 1, 3, 4, 5, 6]
    x[:, 2] = -INF
    assert _check(x, 6, "sigmoid", zero[:64], train=False)[1][0].tolist() == [0, 1, 3, 4, 5, 6]
    x[0, 30] = NAN
    assert route_experts(x, 6, "sigmoid", zero[:64]).ids[0].tolist() == [30, 0, 1, 3, 4, 5]


@pytest.mark.parametrize("tokens", [3, 1100])
@pytest.mark.parametrize("experts,groups", [(64, 8), (60, 5), (128, 4), (256, 8), (256, 64), (512, 8)])
def test_groups_whose_sums_leave_32_bits(experts, groups, tokens):
    """Finite biases whose sum of two is behind the largest number of 32 bits: larger groups are still larger."""
    size = experts // groups
    bias = torch.zeros(experts, device=DEV).view(groups, size)
    bias[:, :2] = torch.linspace(2e38, 3e38, groups, device=DEV)[:, None]
    one = bias.clone()
    one[groups - 1, 0] = INF  # (a sum of infinity is larger still)
    low = torch.where(bias == 0, -3.2e38, -bias)
    for order in (bias, bias.flip(0), bias[torch.randperm(groups, generator=_gen(groups), device=DEV)], low, low.flip(0), one):
        for scoring in ("softmax", "sigmoid"):
            _check(_logits(tokens, experts), 2, scoring, order.flatten(), groups, 1, train=False)
            _check(_logits(tokens, experts), 3, scoring, order.flatten(), groups, 2, train=False)

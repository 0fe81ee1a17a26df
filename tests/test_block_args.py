"""CPU checks of the norms, the routing and the rows' way: the 64-bit references against torch's own differentiation, the
C entry points' refusals (before the device is touched) and the Python operators' checks."""
import os
import re
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from ae_amd import _lib
from ae_amd.build import BINDING_PATH
from ae_amd.layers import combine_rows, dispatch_rows, layer_norm, rms_norm, route_experts
from tests.block_ref import F64, INF, choose, combine, norm, order_of, route

HEADER = os.path.join(os.path.dirname(os.path.dirname(__file__)), "include", "specmoe_mi355x_blocks.h")
L = _lib.lib()
A = 0x10000  # an aligned address that the calls below never follow
OK, BAD, UNS, WS, MIS = (_lib.SMX_OK, _lib.SMX_ERR_INVALID_ARG, _lib.SMX_ERR_UNSUPPORTED,
                         _lib.SMX_ERR_WORKSPACE, _lib.SMX_ERR_MISALIGNED)


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


def _close(a, b):
    assert float((a - b).abs().max()) < 1e-10 * (1 + float(b.abs().max()))


@pytest.mark.parametrize("rms", [True, False])
def test_reference_norm(rms):
    s, w, b, dy, ds = _randn(1, 7, 12), _randn(2, 12), _randn(3, 12), _randn(4, 7, 12), _randn(5, 7, 12)
    leaves = [t.requires_grad_() for t in (s, w, b)]
    if rms:
        y = s * torch.rsqrt(s.square().mean(1, keepdim=True) + 1e-3) * w + b
    else:
        y = torch.nn.functional.layer_norm(s, (12,), w, b, 1e-3)
    ref = norm(s.detach(), w.detach(), b.detach(), 1e-3, rms, torch.float32, None, dy, ds)
    _close(y.detach(), ref["y"][0])
    for g, key in zip(torch.autograd.grad([y, s * 1.0], leaves, [dy, ds]), ("dx", "dw", "db")):
        _close(g, ref[key][0])


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_reference_routing(scoring, renormalize):
    x, dw = _randn(6, 9, 10).requires_grad_(), _randn(7, 9, 3)
    ids = choose(x.detach(), 3, scoring, None, 5, 3)
    score = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
    p = score.gather(1, ids)
    w = 2.5 * (p / p.sum(1, keepdim=True) if renormalize else p)
    ref = route(x.detach(), ids, scoring, renormalize, 2.5, dw)
    _close(w.detach(), ref["weights"][0])
    _close(torch.autograd.grad(w, x, dw)[0], ref["dlogits"][0])


def test_reference_choice():
    """Against the definition, expert by expert."""
    x = torch.randint(0, 3, (40, 12), generator=torch.Generator().manual_seed(1)).double()
    x[3] = -INF
    x[4, 2:] = -INF
    bias = torch.tensor([0.0, 0.25, 0.5] * 4, dtype=F64)
    for b in (None, bias):
        for groups, top in ((1, 1), (4, 2), (3, 2)):
            ids = choose(x, 3, "sigmoid", b, groups, top)
            for t in range(40):
                c = [(-INF if x[t, e] == -INF else float(torch.sigmoid(x[t, e]) + (0 if b is None else b[e]))) for e in range(12)]
                size = 12 // groups
                rank = []
                for g in range(groups):
                    v = sorted((v for v in c[g * size:(g + 1) * size] if v > -INF), reverse=True)
                    rank.append(-INF if not v else v[0] if b is None else sum(v[:2]))
                kept = sorted(range(groups), key=lambda g: (-rank[g], g))[:top]
                able = [e for e in range(12) if e // size in kept and c[e] > -INF]
                want = sorted(able, key=lambda e: (-c[e], e))[:3]
                assert ids[t].tolist() == want + [-1] * (3 - len(want))


def test_reference_order():
    ids = torch.tensor([[2, 0], [0, -1], [1, 2]])
    places, order, offsets = order_of(ids, 4)
    assert order.tolist() == [1, 2, 4, 0, 5, ~3] and offsets.tolist() == [0, 2, 3, 5, 5]
    assert places.tolist() == [[3, 0], [1, ~5], [2, 4]]


def test_reference_combine():
    places, _, _ = order_of(torch.tensor([[2, 0], [0, -1], [1, 2]]), 4)
    rows, w, r, dy = _randn(1, 6, 5).requires_grad_(), _randn(2, 3, 2).requires_grad_(), _randn(3, 3, 5), _randn(4, 3, 5)
    y = torch.stack([r[0] + w[0, 0] * rows[3] + w[0, 1] * rows[0], r[1] + w[1, 0] * rows[1],
                     r[2] + w[2, 0] * rows[2] + w[2, 1] * rows[4]])
    ref = combine(rows.detach(), places, w.detach(), r, torch.float32, dy)
    _close(y.detach(), ref["y"][0])
    drows, dw = torch.autograd.grad(y, [rows, w], dy)
    _close(drows, ref["drows"][0])
    _close(dw, ref["dw"][0])


def test_exports_every_declared_symbol():
    with open(HEADER) as f:
        names = re.findall(r"^(?:int|size_t)\s+(smx_\w+)\s*\(", f.read(), re.M)
    assert sorted(names) == sorted(n for n, _, _ in _lib.BLOCK_SIGNATURES)
    assert all(hasattr(L, n) for n in names)


def test_binding_beside_the_library():
    """Loaded first, the binding leaves one HIP runtime and one copy of the library in the process."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys; sys.path.insert(0, %r); from ae_amd import _lib; b = _lib.blocks(); import ae_amd.layers; "
            "maps = {l.split()[-1] for l in open('/proc/self/maps').read().splitlines()}; "
            "print(b.__file__, *(len([m for m in maps if n in m]) for n in ('libamdhip64', 'libspecmoe_mi355x')))" % root)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == [BINDING_PATH, "1", "1"], out.stdout


def _norm(**kw):
    a = dict(kind=1, x=A, xs=64, r=None, rs=0, dt=2, rows=4, H=64, w=A, b=None, wdt=2, eps=1e-6, y=A, sum=None, stats=None)
    a.update(kw)
    return L.smx_norm(a["kind"], a["x"], a["xs"], a["r"], a["rs"], a["dt"], a["rows"], a["H"], a["w"], a["b"], a["wdt"],
                      a["eps"], a["y"], a["sum"], a["stats"], None)


def _norm_grad(**kw):
    a = dict(kind=0, dy=A, ds=64, g=None, gs=0, s=A, ss=64, dt=2, rows=4, H=64, w=A, wdt=2, stats=A, dx=A, dw=A, db=A,
             work=A, bytes=1 << 30)
    a.update(kw)
    return L.smx_norm_grad(a["kind"], a["dy"], a["ds"], a["g"], a["gs"], a["s"], a["ss"], a["dt"], a["rows"], a["H"], a["w"],
                           a["wdt"], a["stats"], a["dx"], a["dw"], a["db"], a["work"], a["bytes"], None)


@pytest.mark.parametrize("call", [_norm, _norm_grad])
def test_norm_sizes_refused(call):
    assert call(kind=2) == BAD
    assert call(rows=-1) == BAD
    assert call(H=0) == BAD
    assert call(dt=3) == BAD
    assert call(wdt=1) == BAD                     # fp16 parameters of bf16 rows
    assert call(H=16385, xs=1 << 20, ds=1 << 20, ss=1 << 20) == UNS


def test_norm_refused():
    assert _norm(xs=63) == BAD                    # rows would overlap
    assert _norm(eps=-1.0) == BAD and _norm(eps=float("nan")) == BAD
    assert _norm(x=None) == BAD and _norm(y=None) == BAD
    assert _norm(r=A, rs=64) == BAD               # a residual without its sum
    assert _norm(sum=A) == BAD                    # a sum without a residual
    assert _norm(r=A, rs=63, sum=A) == BAD
    for name in ("x", "y", "w", "b", "sum"):
        assert _norm(**{"r": A, "rs": 64, "sum": A, name: A + 1}) == MIS
    assert _norm(stats=A + 2) == MIS
    assert _norm(rows=0, x=None, y=None) == OK    # nothing to do, nothing launched


def test_norm_grad_refused():
    assert _norm_grad(ds=63) == BAD and _norm_grad(ss=63) == BAD and _norm_grad(g=A, gs=63) == BAD
    assert _norm_grad(kind=1) == BAD              # an RMS norm has no bias
    assert _norm_grad(dy=None) == BAD and _norm_grad(s=None) == BAD and _norm_grad(stats=None) == BAD
    for name in ("dy", "s", "dx", "dw", "db", "w"):
        assert _norm_grad(**{name: A + 1}) == MIS
    need = L.smx_norm_grad_workspace_size(0, 4, 64, 2)
    assert need > 0 and need == 2 * L.smx_norm_grad_workspace_size(1, 4, 64, 2)
    assert _norm_grad(bytes=need - 1) == WS and _norm_grad(work=None) == WS
    assert _norm_grad(work=A + 4) == MIS
    assert _norm_grad(rows=0, dx=None, dw=None, db=None) == OK
    assert L.smx_norm_grad_workspace_size(0, 4, 16385, 2) == 0


def _route(**kw):
    a = dict(x=A, xs=64, dt=2, T=1000, E=64, k=6, sc=0, bias=None, ng=1, tg=1, ren=1, scale=1.0, w=A, ids=A, places=A,
             order=A, off=A, work=A, bytes=1 << 30)
    a.update(kw)
    return L.smx_route(a["x"], a["xs"], a["dt"], a["T"], a["E"], a["k"], a["sc"], a["bias"], a["ng"], a["tg"], a["ren"],
                       a["scale"], a["w"], a["ids"], a["places"], a["order"], a["off"], a["work"], a["bytes"], None)


def _route_grad(**kw):
    a = dict(dw=A, x=A, xs=64, dt=2, T=1000, E=64, k=6, sc=0, ren=1, scale=1.0, ids=A, d=A)
    a.update(kw)
    return L.smx_route_grad(a["dw"], a["x"], a["xs"], a["dt"], a["T"], a["E"], a["k"], a["sc"], a["ren"], a["scale"],
                            a["ids"], a["d"], None)


@pytest.mark.parametrize("call", [_route, _route_grad])
def test_routing_sizes_refused(call):
    assert call(T=-1) == BAD
    assert call(E=0) == BAD
    assert call(k=0) == BAD
    assert call(k=65) == BAD                      # more picks than experts
    assert call(dt=5) == BAD
    assert call(sc=2) == BAD
    assert call(xs=63) == BAD
    assert call(k=17) == UNS
    assert call(E=1025, xs=2000) == UNS
    assert call(T=1 << 30) == UNS                 # 2^31 picks and more
    assert call(scale=float("inf")) == BAD and call(scale=float("nan")) == BAD


def test_routing_refused():
    assert _route(ng=0) == BAD and _route(ng=5) == BAD
    assert _route(ng=8, tg=0) == BAD and _route(ng=8, tg=9) == BAD
    assert _route(ng=16, tg=1) == BAD             # 6 picks of 4 selectable experts
    assert _route(E=128, xs=128, ng=128, tg=128) == UNS
    for name in ("x", "w", "ids", "places", "order", "off"):
        assert _route(**{name: None}) == BAD, name
    for name in ("w", "ids", "places", "order", "bias"):
        assert _route(**{name: A + 2}) == MIS, name
    assert _route(x=A + 1) == MIS and _route(off=A + 4) == MIS and _route(work=A + 8) == MIS
    need = L.smx_route_workspace_size(1000, 64, 6)
    assert need > 0 and L.smx_route_workspace_size(10, 64, 6) == 0
    assert _route(bytes=need - 1) == WS and _route(work=None) == WS
    assert L.smx_route_workspace_size(1000, 64, 17) == 0


def test_routing_gradient_refused():
    for name in ("dw", "x", "ids", "d"):
        assert _route_grad(**{name: None}) == BAD
    assert _route_grad(x=A + 1) == MIS and _route_grad(d=A + 1) == MIS and _route_grad(dw=A + 2) == MIS
    assert _route_grad(T=0, x=None, d=None, dw=None, ids=None) == OK


def _dispatch(**kw):
    a = dict(x=A, xs=64, dt=2, T=10, H=64, p=A, k=3, y=A)
    a.update(kw)
    return L.smx_dispatch_rows(a["x"], a["xs"], a["dt"], a["T"], a["H"], a["p"], a["k"], a["y"], None)


def _combine(**kw):
    a = dict(x=A, xs=64, dt=2, T=10, H=64, p=A, k=3, w=A, r=A, rs=64, y=A)
    a.update(kw)
    return L.smx_combine_rows(a["x"], a["xs"], a["dt"], a["T"], a["H"], a["p"], a["k"], a["w"], a["r"], a["rs"], a["y"], None)


def _combine_grad(**kw):
    a = dict(dy=A, ds=64, x=A, xs=64, dt=2, T=10, H=64, p=A, k=3, w=A, y=A, dw=A)
    a.update(kw)
    return L.smx_combine_rows_grad(a["dy"], a["ds"], a["x"], a["xs"], a["dt"], a["T"], a["H"], a["p"], a["k"], a["w"],
                                   a["y"], a["dw"], None)


@pytest.mark.parametrize("call", [_dispatch, _combine, _combine_grad])
def test_rows_refused(call):
    assert call(T=-1) == BAD
    assert call(H=0) == BAD
    assert call(k=0) == BAD
    assert call(dt=3) == BAD
    assert call(xs=63) == BAD
    assert call(k=17) == UNS
    assert call(T=1 << 30) == UNS
    assert call(H=(1 << 24) + 1, xs=1 << 25, rs=1 << 25, ds=1 << 25) == UNS
    assert call(x=None) == BAD and call(p=None) == BAD
    assert call(x=A + 1) == MIS and call(y=A + 1) == MIS and call(p=A + 2) == MIS
    assert call(T=0, x=None, p=None, y=None) == OK


def test_rows_refused_by_name():
    assert _dispatch(y=None) == BAD and _combine(y=None) == BAD
    assert _combine(rs=63) == BAD and _combine(r=A + 1) == MIS and _combine(w=A + 2) == MIS
    assert _combine_grad(dy=None) == BAD and _combine_grad(ds=63) == BAD and _combine_grad(dw=A + 2) == MIS
    assert _combine_grad(y=None, dw=None) == OK


def test_norm_python_checks():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="GPU"):
        rms_norm(x, w)
    with pytest.raises(ValueError, match="weight must be"):
        layer_norm(x, torch.zeros(7))
    with pytest.raises(ValueError, match="bias must be"):
        layer_norm(x, w, torch.zeros(1))
    with pytest.raises(ValueError, match="residual must be"):
        rms_norm(x, w, residual=torch.zeros(8))
    with pytest.raises(TypeError, match="mismatch"):
        rms_norm(x, w.half())
    with pytest.raises(TypeError, match="mismatch"):
        rms_norm(x.half(), w, residual=x)
    with pytest.raises(TypeError, match="mismatch"):
        layer_norm(x.half(), w, w.half())
    with pytest.raises(TypeError, match="unsupported"):
        rms_norm(x.double(), w.double())
    with pytest.raises(ValueError, match="H"):
        rms_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, w, eps=float("nan"))


def test_routing_python_checks():
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="GPU"):
        route_experts(x, 2)
    with pytest.raises(ValueError, match="logits must be"):
        route_experts(x[0], 2)
    with pytest.raises(TypeError, match="unsupported"):
        route_experts(x.double(), 2)
    with pytest.raises(ValueError, match="scoring"):
        route_experts(x, 2, "tanh")
    for groups, top in ((3, 1), (0, 1), (4, 5), (4, 0)):
        with pytest.raises(ValueError, match="groups"):
            route_experts(x, 2, num_groups=groups, top_groups=top)
    for k, top in ((0, 4), (9, 4), (3, 1)):
        with pytest.raises(ValueError, match="top_k"):
            route_experts(x, k, num_groups=4, top_groups=top)
    with pytest.raises(ValueError, match="scale"):
        route_experts(x, 2, scale=INF)
    with pytest.raises(ValueError, match="bias must be"):
        route_experts(x, 2, bias=torch.zeros(7))
    with pytest.raises(TypeError, match="bias"):
        route_experts(x, 2, bias=torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError, match="detached"):
        route_experts(x, 2, bias=torch.zeros(8, requires_grad=True))


def test_rows_python_checks():
    x, p = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        dispatch_rows(x, p)
    with pytest.raises(ValueError, match="GPU"):
        combine_rows(torch.zeros(8, 8), p)
    with pytest.raises(TypeError, match="int32"):
        dispatch_rows(x, p.long())
    with pytest.raises(TypeError, match="int32"):
        dispatch_rows(x, p.t().contiguous().t())
    with pytest.raises(ValueError, match="tokens"):
        dispatch_rows(x[:3], p)
    with pytest.raises(ValueError, match="picks"):
        dispatch_rows(x, p[:, :0])
    with pytest.raises(ValueError, match="picks"):
        combine_rows(x, p)
    with pytest.raises(ValueError, match="weights must be"):
        combine_rows(torch.zeros(8, 8), p, torch.zeros(2, 4))
    with pytest.raises(TypeError, match="fp32"):
        combine_rows(torch.zeros(8, 8), p, torch.zeros(4, 2).half())
    with pytest.raises(ValueError, match="residual must be"):
        combine_rows(torch.zeros(8, 8), p, residual=torch.zeros(8, 8))
    with pytest.raises(TypeError, match="mismatch"):
        combine_rows(torch.zeros(8, 8), p, residual=x.half())
    with pytest.raises(ValueError, match="H"):
        dispatch_rows(x[:, :0], p)
    with pytest.raises(TypeError, match="unsupported"):
        dispatch_rows(x.long(), p)


def test_forward_mode_refused():
    x, p = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: rms_norm(d), lambda: layer_norm(x, residual=d), lambda: route_experts(d, 2),
                     lambda: dispatch_rows(d, p), lambda: combine_rows(torch.zeros(8, 8), p, residual=d)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def _calls(x, p):
    w, rows = torch.ones(8), torch.zeros(8, 8)
    return {"rms_norm": lambda t: rms_norm(t, w), "layer_norm": lambda t: layer_norm(x, residual=t),
            "route": lambda t: route_experts(t, 2).weights, "dispatch": lambda t: dispatch_rows(t, p),
            "combine": lambda t: combine_rows(rows, p, residual=t)}


@pytest.mark.parametrize("name", ["rms_norm", "layer_norm", "route", "dispatch", "combine"])
def test_traces_and_transforms_refused(name):
    """A trace would hold an empty result without its kernel, and a transform's tensors stand for others."""
    x, p = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    call = _calls(x, p)[name]
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call)(x)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call, tracing_mode="fake")(x)
    with FakeTensorMode(), pytest.raises(RuntimeError, match="traced"):
        call(torch.empty(4, 8))
    for transform in (lambda f: torch.vmap(f)(x[None]), lambda f: torch.func.grad(lambda t: f(t).sum())(x),
                      lambda f: torch.func.functionalize(f)(x), lambda f: torch.func.jacrev(f)(x)):
        with pytest.raises(RuntimeError, match="torch.func"):
            transform(call)
    with pytest.raises(ValueError, match="GPU"):  # and again as before
        call(x)


def test_other_modes_stay():
    """A mode that only looks on (of a checkpoint's, a counter of operations) is no trace."""
    class Looks(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Looks(), pytest.raises(ValueError, match="GPU"):
        rms_norm(torch.zeros(4, 8))

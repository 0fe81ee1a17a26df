"""CPU checks of the matrix products: the 64-bit reference against differences, the C entry points'
refusals (before the device is touched) and the Python operators' checks."""
import ctypes
import os
import re

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from ae_amd import _lib
from ae_amd.layers import fused_linear, grouped_linear
from tests.product_ref import ACTS, F64, act, act_grad, product

HEADER = os.path.join(os.path.dirname(os.path.dirname(__file__)), "include", "specmoe_mi355x_products.h")
L = _lib.lib()
A = 0x10000  # an aligned address that the calls below never follow
OK, BAD, UNS, WS, MIS = (_lib.SMX_OK, _lib.SMX_ERR_INVALID_ARG, _lib.SMX_ERR_UNSUPPORTED,
                         _lib.SMX_ERR_WORKSPACE, _lib.SMX_ERR_MISALIGNED)


@pytest.mark.parametrize("name", [a for a in ACTS if a != "swiglu"])
def test_reference_slopes_against_differences(name):
    z = torch.linspace(-6, 6, 4001, dtype=F64) + 1e-3  # off relu's corner
    h = 1e-5
    d = (act(name, z + h) - act(name, z - h)) / (2 * h)
    # a central difference errs by h^2 / 6 times a third derivative (below 3 for all) and 2^-52 |act| / h
    far = torch.where(z.abs() > 2 * h, (d - act_grad(name, z)).abs(), torch.zeros_like(z))
    assert float(far.max()) < 1e-9


@pytest.mark.parametrize("name", ACTS)
def test_reference_gradients_against_differences(name):
    g = torch.Generator().manual_seed(3)
    rows, k, n = 3, 5, 4
    nw = 2 * n if name == "swiglu" else n
    t = [torch.randn(s, generator=g, dtype=F64) for s in ((rows, k), (nw, k), (nw,), (rows, n))]
    ref = product(t[0], t[1], t[2], name, None, torch.float32, t[3])
    h = 1e-6

    def loss(x, w, b):
        return float((product(x, w, b, name, None, torch.float32)["y"][0] * t[3]).sum())

    for i, key in enumerate(("dx", "dw", "db")):
        for j in range(t[i].numel()):
            a = [v.clone() for v in t[:3]]
            a[i].view(-1)[j] += h
            b = [v.clone() for v in t[:3]]
            b[i].view(-1)[j] -= h
            # differences of a smooth loss: rounding of the loss, 2^-52 * 100 / h, dominates
            assert abs((loss(*a) - loss(*b)) / (2 * h) - float(ref[key][0].view(-1)[j])) < 1e-7


def test_exports_every_declared_symbol():
    with open(HEADER) as f:
        names = re.findall(r"^(?:int|size_t)\s+(smx_\w+)\s*\(", f.read(), re.M)
    assert sorted(names) == sorted(n for n, _, _ in _lib.PRODUCT_SIGNATURES)
    assert all(hasattr(L, n) for n in names)


def _linear(**kw):
    a = dict(x=A, xs=64, dt=2, rows=4, K=64, w=A, ws=64, N=32, b=None, act=0, r=None, rs=0, y=A, ys=32, z=None,
             work=A, bytes=1 << 40)
    a.update(kw)
    return L.smx_linear(a["x"], a["xs"], a["dt"], a["rows"], a["K"], a["w"], a["ws"], a["N"], a["b"], a["act"],
                        a["r"], a["rs"], a["y"], a["ys"], a["z"], a["work"], a["bytes"], None)


def _grouped(**kw):
    a = dict(x=A, xs=64, dt=2, rows=4, K=64, w=A, ws=64, gs=64 * 32, P=3, N=32, b=None, act=0, r=None, rs=0, off=A,
             G=3, slots=None, fill=1, y=A, ys=32, z=None, work=A, bytes=1 << 40)
    a.update(kw)
    return L.smx_grouped_linear(a["x"], a["xs"], a["dt"], a["rows"], a["K"], a["w"], a["ws"], a["gs"], a["P"],
                                a["N"], a["b"], a["act"], a["r"], a["rs"], a["off"], a["G"], a["slots"], a["fill"],
                                a["y"], a["ys"], a["z"], a["work"], a["bytes"], None)


def _grad(**kw):
    a = dict(dy=A, ds=32, z=A, x=A, xs=64, dt=2, rows=4, K=64, w=A, ws=64, gs=64 * 32, P=3, N=32, act=2, off=A, G=3,
             slots=None, dx=A, dw=A, db=A, work=A, bytes=1 << 40)
    a.update(kw)
    if a["G"] is None:
        return L.smx_linear_grad(a["dy"], a["ds"], a["z"], a["x"], a["xs"], a["dt"], a["rows"], a["K"], a["w"],
                                 a["ws"], a["N"], a["act"], a["dx"], a["dw"], a["db"], a["work"], a["bytes"], None)
    return L.smx_grouped_linear_grad(a["dy"], a["ds"], a["z"], a["x"], a["xs"], a["dt"], a["rows"], a["K"], a["w"],
                                     a["ws"], a["gs"], a["P"], a["N"], a["act"], a["off"], a["G"], a["slots"],
                                     a["dx"], a["dw"], a["db"], a["work"], a["bytes"], None)


@pytest.mark.parametrize("call", [_linear, _grouped, _grad])
def test_sizes_refused(call):
    assert call(rows=-1) == BAD
    assert call(K=0) == BAD
    assert call(N=0) == BAD
    assert call(dt=3) == BAD
    assert call(act=6) == BAD
    assert call(act=-1) == BAD
    assert call(rows=(1 << 30) + 1) == UNS
    assert call(xs=63) == BAD                     # rows would overlap
    assert call(ws=63) == BAD
    assert call(xs=1 << 23) == UNS                # 16 MiB pitch
    assert call(ws=1 << 23) == UNS


def test_forward_refused():
    for call in (_linear, _grouped):
        assert call(x=None) == BAD
        assert call(w=None) == BAD
        assert call(y=None) == BAD
        assert call(ys=31) == BAD
        assert call(r=A, rs=31) == BAD
        for name in ("x", "w", "y", "b", "z"):
            assert call(**{name: A + 1}) == MIS
        assert call(r=A + 1, rs=32) == MIS
        assert call(rows=0, x=None, w=None, y=None, work=None, bytes=0) == OK  # nothing to do
    assert _linear(ws=1 << 21, N=1 << 20, K=64, ys=1 << 20) == UNS  # a weight of 2 GiB and more


def test_groups_refused():
    for call in (_grouped, _grad):
        assert call(off=None) == BAD
        assert call(G=0) == BAD
        assert call(G=-1) == BAD
        assert call(P=4) == BAD                   # weights and groups differ without a slot map
        assert call(P=0, slots=A) == BAD
        assert call(gs=-1) == BAD
        assert call(off=A + 4) == MIS
    assert _grouped(slots=A + 4, P=9) == MIS


def test_gradients_refused():
    for G in (None, 3):
        assert _grad(G=G, dy=None) == BAD
        assert _grad(G=G, x=None) == BAD
        assert _grad(G=G, w=None) == BAD
        assert _grad(G=G, z=None) == BAD          # an activation needs the pre-activations
        assert _grad(G=G, ds=31) == BAD
        assert _grad(G=G, work=None) == WS
        assert _grad(G=G, bytes=16) == WS
        assert _grad(G=G, work=A + 4) == MIS
        assert _grad(G=G, dw=A + 1) == MIS
        assert _grad(G=G, rows=0, dx=None, dw=None, db=None) == OK
    assert _grad(slots=A, P=9, dw=None) == BAD    # weights behind a slot map have no gradient
    assert _grad(slots=A, P=9, db=None) == BAD


def test_workspace_sizes():
    for query in (L.smx_linear_workspace_size, L.smx_linear_grad_workspace_size):
        assert query(-1, 64, 32, 0, 0, 2) == 0
        assert query(4, 0, 32, 0, 0, 2) == 0
        assert query(4, 64, 32, 0, 9, 2) == 0
        assert query(4, 64, 32, 0, 0, 7) == 0
    g = L.smx_linear_grad_workspace_size
    assert g(128, 64, 32, 0, 5, 2) >= 128 * 64 * 2      # dz of 2 N columns
    assert g(128, 64, 32, 0, 5, 0) >= 128 * 64 * 4
    assert g(128, 64, 32, 64, 0, 2) >= g(128, 64, 32, 0, 0, 2)


def _cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def test_python_checks_refuse():
    x, w, off = _cpu(4, 8), _cpu(6, 8), torch.tensor([0, 2, 4])
    w3 = _cpu(2, 6, 8)
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="columns"):
        fused_linear(x, _cpu(6, 9))
    with pytest.raises(ValueError, match="weight"):
        fused_linear(x, w3)
    with pytest.raises(ValueError, match="weight"):
        grouped_linear(x, w, off)
    with pytest.raises(ValueError, match="odd"):
        fused_linear(x, _cpu(7, 8), activation="swiglu")
    with pytest.raises(ValueError, match="bias"):
        fused_linear(x, w, _cpu(5))
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, w, residual=_cpu(4, 5))
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, w, residual=_cpu(1, 6))           # no broadcasting: expand it
    with pytest.raises(ValueError, match="out"):
        fused_linear(x, w, out=_cpu(4, 5))
    with pytest.raises(ValueError, match="adjacent"):
        fused_linear(x, _cpu(8, 6).t())
    with pytest.raises(ValueError, match="adjacent"):
        fused_linear(x, _cpu(1, 8).expand(6, 8))
    with pytest.raises(ValueError, match="empty"):
        fused_linear(_cpu(4, 0), _cpu(6, 0))
    with pytest.raises(TypeError, match="float"):
        fused_linear(x.to(F64), w.to(F64))
    with pytest.raises(ValueError, match="GPU"):
        fused_linear(x, w)
    with pytest.raises(TypeError, match="group_offsets"):
        grouped_linear(x, w3, None)


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual", "out"])
def test_forward_mode_refused(which):
    """A dual tensor's tangent would be dropped: the call says so, before anything else."""
    t = {"x": _cpu(4, 8), "weight": _cpu(6, 8), "bias": _cpu(6), "residual": _cpu(4, 6), "out": _cpu(4, 6)}
    g = {"x": t["x"], "weight": _cpu(2, 6, 8), "bias": _cpu(2, 6), "residual": t["residual"], "out": t["out"]}
    with forward_ad.dual_level():
        for call, args in ((fused_linear, t), (grouped_linear, {**g, "group_offsets": torch.tensor([0, 2, 4])})):
            dual = {**args, which: forward_ad.make_dual(args[which], torch.ones_like(args[which]))}
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(**dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(**dual)
            with pytest.raises(ValueError, match="GPU"):  # within a level, but no duals: the next check
                call(**args)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: fused_linear(**{**t, which: v}), (t[which],), (t[which],))


@pytest.mark.parametrize("which", ["fused", "grouped"])
def test_traces_refused(which):
    """A trace would hold an empty result without its kernel."""
    x, w, off = torch.zeros(4, 8), torch.zeros(2, 8, 8), torch.tensor([0, 2, 4])
    call = (lambda t: fused_linear(t, w[0])) if which == "fused" else (lambda t: grouped_linear(t, w, off))
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call)(x)
    with pytest.raises(ValueError, match="GPU"):  # and again as before
        call(x)

"""Gradients of the matrix products where a call's form is at its edges: a single group whose weight gradient is
split along the contraction, into results that hold NaN before the call. Against 64 bits within the bounds of
tests/product_ref.py."""
import pytest
import torch
from torch.autograd import forward_ad

from ae_amd import _lib
from ae_amd.layers import fused_linear, grouped_linear
from tests.product_ref import check, product
from tests.test_gpu_linear import BF16, DEV, F16, F32, _check_grouped, _inputs

pytestmark = pytest.mark.gpu
CODES = {F32: _lib.SMX_F32, F16: _lib.SMX_F16, BF16: _lib.SMX_BF16}


class Room:
    """A contiguous tensor of `fill` (its bytes, for scratch memory) with a margin of a known pattern on both sides."""

    MARGIN = 4096

    def __init__(self, shape, dtype, fill=float("nan")):
        n = torch.Size(shape).numel()
        self.mark = 0xA5 if dtype == torch.uint8 else 5.0
        self.all = torch.full((n + 2 * self.MARGIN,), self.mark, dtype=dtype, device=DEV)
        self.t = self.all[self.MARGIN:self.MARGIN + n].view(shape)
        self.t.fill_(fill)

    def margins_whole(self):
        m = self.MARGIN
        return bool((self.all[:m] == self.mark).all()) and bool((self.all[-m:] == self.mark).all())


def _grad_into(dy, z, x, w, off, act):
    """The C gradient call of a grouped product (contiguous operands, a weight per group) into tensors of NaN; their
    margins and the workspace's stay as they were."""
    (rows, k), (groups, nw, _), n = x.shape, w.shape, dy.shape[1]
    code, a = CODES[x.dtype], _lib.ACTIVATIONS[act]
    nbytes = _lib.lib().smx_linear_grad_workspace_size(rows, k, n, groups, a, code)
    dx, dw, db = Room((rows, k), x.dtype), Room((groups, nw, k), x.dtype), Room((groups, nw), x.dtype)
    ws = Room((nbytes,), torch.uint8, 0xFF)
    _lib.call("smx_grouped_linear_grad", dy.data_ptr(), n, None if z is None else z.data_ptr(), x.data_ptr(), k, code,
              rows, k, w.data_ptr(), k, nw * k, groups, n, a, off.data_ptr(), groups, None, dx.t.data_ptr(),
              dw.t.data_ptr(), db.t.data_ptr(), ws.t.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert all(r.margins_whole() for r in (dx, dw, db, ws))
    return dx.t, dw.t, db.t


# More rows than columns by far: the plan splits the weight gradient 2 to 8 ways. fp32 and 16-bit types; rows of whole
# 16-byte slots and odd ones; fewer rows than weight rows, and more.
ONE_GROUP = [(900, 64, 1024, F32), (640, 64, 2816, F32), (1000, 128, 2048, F32), (900, 61, 1001, F32),
             (2000, 256, 256, BF16), (2300, 64, 2816, BF16), (1500, 99, 2048, BF16), (5000, 333, 1000, BF16),
             (8192, 256, 2048, BF16), (2000, 64, 2048, F16), (16000, 1000, 4096, F16)]
BOUNDS = {"all": lambda r: (0, r), "inside": lambda r: (37, r - 37), "few": lambda r: (7, 50), "empty": lambda r: (9, 9),
          "late": lambda r: (r - 20, r), "clamped": lambda r: (-4, r + 100)}


@pytest.mark.parametrize("bounds", BOUNDS)
@pytest.mark.parametrize("rows,k,n,dtype", ONE_GROUP)
def test_weight_gradient_of_one_group(rows, k, n, dtype, bounds):
    """Every row of the weight's gradient, whatever rows of x the group has."""
    lo, hi = BOUNDS[bounds](rows)
    x, w, _, _, dy = _inputs(rows, k, n, None, dtype, groups=1, bias=False, residual=False)
    off = torch.tensor([lo, hi], device=DEV)
    dx, dw, db = _grad_into(dy, None, x, w, off, None)
    lo, hi = max(lo, 0), min(hi, rows)
    ref = product(x[lo:hi], w[0], None, None, None, dtype, dy[lo:hi])
    check(dw[0], *ref["dw"], what="dw")
    check(db[0], *ref["db"], what="db")
    check(dx[lo:hi], *ref["dx"], what="dx")
    assert not bool(dx[:lo].any()) and not bool(dx[hi:].any())


@pytest.mark.parametrize("rows,k,n,dtype,act", [(900, 64, 1024, F32, "gelu"), (2000, 256, 256, BF16, "silu"),
                                                (1500, 99, 1024, BF16, "swiglu")])
def test_training_of_one_group(rows, k, n, dtype, act):
    """The same through grouped_linear: an expert-parallel rank with one local expert and a padded batch."""
    x, w, b, r, dy = _inputs(rows, k, n, act, dtype, groups=1)
    _check_grouped(x, w, torch.tensor([5, rows - 300], device=DEV), b, r, act, dy, what=act)


def test_forward_mode_refused():
    """Tangents of the operands, and of the gradient that comes in, would be dropped."""
    x, w, _, _, dy = _inputs(8, 16, 24, "silu", F32)
    off = torch.tensor([0, 8], device=DEV)
    y = fused_linear(x.requires_grad_(), w, None, "silu")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        for call in (lambda: fused_linear(dual, w), lambda: grouped_linear(dual, w[None], off)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, [x], forward_ad.make_dual(dy, torch.ones_like(dy)))
        fused_linear(x.detach(), w)  # no duals


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("grouped", [False, True])
def test_closed_relu_passes_nothing_on(grouped, dtype):
    """Where z is negative or zero the gradient is zero whatever comes in, infinities and NaN too; elsewhere they
    pass."""
    x, w, b, _, dy = _inputs(40, 64, 48, "relu", dtype, residual=False)
    w[:8] = 0
    b[:4], b[4:8] = -2, 0
    leaves = [t.requires_grad_() for t in (x, w, b)]
    off = torch.tensor([0, 40], device=DEV)

    def grads(dy):
        y = grouped_linear(x, w[None], off, b[None], "relu") if grouped else fused_linear(x, w, b, "relu")
        return torch.autograd.grad(y, leaves, dy)

    bad = torch.tensor([float("inf"), float("nan"), float("-inf"), 1.0] * 2, device=DEV, dtype=dtype)
    dy[:, :8] = 0
    want = grads(dy)
    dy[3, :8] = bad
    for p, q in zip(grads(dy), want):
        assert bool(torch.isfinite(p).all()) and torch.equal(p, q)
    with torch.no_grad():
        b[8] = 60.0  # (far beyond any product here)
    dy[3, 8] = float("inf")
    dx, dw, db = grads(dy)
    assert not bool(torch.isfinite(dx[3]).any()) and not bool(torch.isfinite(dw[8]).any()) and not bool(torch.isfinite(db[8]))
    assert bool(torch.isfinite(dx[4:]).all()) and bool(torch.isfinite(dw[9:]).all()) and bool(torch.isfinite(db[9:]).all())


# Products of 1 and 1 + 2^-15: every sum of up to 288 of them is exact in fp32 (a multiple of 2^-15 below 512), while one
# chain of n loses the low bits of whatever it adds once it has passed 4096 (steps of 2^-11): at least 2^-13 of every four
# products, 0.24 in all at n = 12000. Sums of chains of 256 to 288 of them round by at most 2^-11 (half a step below 16384)
# per chain, and per split or wave of the walk, of which there are at most 20.
TERM = 1 + 2.0 ** -15


def _check_chains(got, n):
    assert 8000 < n < 16000
    off = float((got.to(torch.float64) - n * TERM).abs().max())
    assert off <= (n / 256 + 20) * 2.0 ** -11, (off, n)


# one group has nearly all rows: groups of few rows by their mean (aligned and not), of more, and a single one
@pytest.mark.parametrize("rows,k,n,groups", [(12800, 256, 256, 64), (12100, 512, 640, 64), (12100, 511, 640, 64),
                                             (12100, 257, 512, 64), (12000, 256, 256, 16), (12000, 128, 256, 1)])
def test_long_fp32_weight_gradients_run_in_chains(rows, k, n, groups):
    x = torch.ones(rows, k, device=DEV)
    w = torch.zeros(groups, n, k, device=DEV)
    dy = torch.full((rows, n), TERM, device=DEV)
    hot = groups // 3
    off = torch.tensor([g if g <= hot else rows - groups + g for g in range(groups + 1)], device=DEV)
    _, dw, _ = _grad_into(dy, None, x, w, off, None)
    _check_chains(dw[hot], rows - groups + 1)
    assert all(bool((dw[g] == TERM).all()) for g in range(groups) if g != hot)


@pytest.mark.parametrize("rows,k,n", [(3, 12000, 2048), (3, 12001, 2048), (40, 12000, 1024), (3, 12000, 64), (300, 12001, 65)])
def test_long_fp32_products_run_in_chains(rows, k, n):
    y = fused_linear(torch.ones(rows, k, device=DEV), torch.full((n, k), TERM, device=DEV))
    _check_chains(y, k)


def test_long_fp32_groups_of_random_values():
    """The same tiles walked over groups of many and of few rows in turn, into results of whole slots and odd ones."""
    for k, n, many in ((264, 200, 32), (511, 640, 56)):
        cut = [0, 3, 3, 4000, 4031, 4032, 5000] + [5000 + 8 * i for i in range(many)] + [8990, 9000]
        x, w, _, _, dy = _inputs(9000, k, n, None, F32, groups=len(cut) - 1, bias=False, residual=False)
        off = torch.tensor(cut, device=DEV)
        _, dw, _ = _grad_into(dy, None, x, w, off, None)
        for g, (lo, hi) in enumerate(zip(cut, cut[1:])):
            check(dw[g], *product(x[lo:hi], w[g], None, None, None, F32, dy[lo:hi])["dw"], what=f"{k} x {n}, group {g}")


@pytest.mark.parametrize("rows,k,n", [(40, 128, 96), (700, 128, 96), (5000, 128, 96), (5000, 131, 77)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_gradients_of_bounds_that_decrease_stay_inside(act, dtype, rows, k, n):
    """Bounds that mean nothing name rows twice: more row tiles than rows, whose column sums and results have no place.
    Nothing outside the results and the workspace is written (_grad_into looks), and a call that means something
    comes out right behind it."""
    x, w, b, _, dy = _inputs(rows, k, n, act, dtype, groups=6, residual=False)
    z = torch.randn(rows, w.shape[1], device=DEV, generator=torch.Generator(device=DEV).manual_seed(rows))
    for bounds in ([2, rows - 9, 3, rows + 70, -5, rows // 2, 4], [rows, 0, rows, 0, rows, 0, rows],
                   [0, rows, 0, rows, 0, rows, 0], [2 ** 40, -2 ** 40, 2 ** 62, 0, rows, 1, 2 ** 62]):
        off = torch.tensor(bounds, device=DEV)
        y = Room((rows, n), dtype)
        with torch.no_grad():
            grouped_linear(x, w, off, b, act, out=y.t)
        assert y.margins_whole()
        _grad_into(dy, z, x, w, off, act)
    _check_grouped(x, w, torch.tensor([0, 1, 9, 9, 20, 30, rows], device=DEV), b, None, act, dy)

"""layer_norm and rms_norm against the 64-bit reference, with their gradients."""
import pytest
import torch

from ae_amd import _lib
from ae_amd._lib import SmxError
from ae_amd.layers import RMSNorm, layer_norm, rms_norm
from tests.block_ref import F64, norm
from tests.product_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-6


def _randn(gen, *shape, dtype=F32, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale + mean).to(dtype)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inputs(rows, cols, dtype, rms=False, residual=False, wtype=None, affine=True, mean=0.3):
    g = _gen(rows * 31 + cols)
    x = _randn(g, rows, cols, dtype=dtype, scale=1.5, mean=mean)
    r = _randn(g, rows, cols, dtype=dtype, scale=2.0) if residual else None
    w = _randn(g, cols, dtype=wtype or dtype, scale=0.3, mean=1.0) if affine else None
    b = _randn(g, cols, dtype=wtype or dtype, scale=0.2) if affine and not rms else None
    dy = _randn(g, rows, cols, dtype=dtype)
    ds = _randn(g, rows, cols, dtype=dtype) if residual else None
    return x, r, w, b, dy, ds


def _call(rms, x, w, b, r, eps=EPS):
    return rms_norm(x, w, eps, residual=r) if rms else layer_norm(x, w, b, eps, residual=r)


def _check(rms, x, r, w, b, dy=None, ds=None, eps=EPS, what=""):
    """The norm, and with dy its gradients; returns the outputs."""
    named = {"x": x, "r": r, "w": w, "b": b}
    leaves = {n: t.detach().requires_grad_(dy is not None) for n, t in named.items() if t is not None}
    out = _call(rms, leaves["x"], leaves.get("w"), leaves.get("b"), leaves.get("r"), eps)
    y, s = out if r is not None else (out, x)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    if r is not None:
        assert torch.equal(s.detach(), x + r)
    h = x.shape[-1]
    flat = [None if t is None else t.detach().reshape(-1, h) for t in (s, dy, ds)]
    params = None if w is None and b is None else (w if w is not None else b).dtype
    ref = norm(flat[0], w, b, eps, rms, x.dtype, params, flat[1], flat[2])
    check(y.detach().reshape(-1, h), *ref["y"], what=f"{what} y")
    if dy is None:
        return [y]
    got = dict(zip(leaves, torch.autograd.grad([y] if r is None else [y, s], list(leaves.values()),
                                               [dy] if r is None else [dy, ds])))
    for n, key in (("x", "dx"), ("r", "dx"), ("w", "dw"), ("b", "db")):
        if n in got:
            assert got[n].dtype == named[n].dtype
            check(got[n].reshape(ref[key][0].shape), *ref[key], what=f"{what} {key}")
    return [y.detach(), *got.values()]


# every width of the kernels' threads and chunks, on both sides of each border
COLS = [1, 2, 7, 63, 64, 65, 128, 136, 250, 256, 264, 512, 520, 1000, 1001, 1024, 1032, 2047, 2048, 2056, 4096, 4104, 5120,
        8192, 8200, 16383, 16384]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("cols", COLS)
def test_widths(cols, rms, dtype):
    _check(rms, *_inputs(5, cols, dtype, rms))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("rows,cols", [(1, 2048), (2, 129), (17, 96), (257, 384), (1025, 128), (2049, 1024), (4111, 64), (1030, 1001)])
def test_rows_with_a_residual(rows, cols, rms, dtype):
    x, r, w, b, dy, ds = _inputs(rows, cols, dtype, rms, residual=True)
    _check(rms, x, r, w, b, dy, ds)
    with torch.no_grad():
        _check(rms, x, r, w, b)


@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("cols", [128, 333, 4096, 6001])
def test_parameters_in_32_bits(cols, rms):
    for dtype in (BF16, F16):
        _check(rms, *_inputs(33, cols, dtype, rms, residual=True, wtype=F32))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_without_parameters(dtype):
    for rms in (True, False):
        _check(rms, *_inputs(9, 300, dtype, rms, affine=False))
    x, r, w, b, dy, ds = _inputs(9, 300, dtype)
    _check(False, x, r, None, b, dy, ds)
    _check(False, x, r, w, None, dy, ds)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rms", [True, False])
def test_long_columns(rms, dtype):
    """The parameters' gradients over many rows, several walks of each workgroup."""
    _check(rms, *_inputs(70001, 128, dtype, rms))
    _check(rms, *_inputs(5000, 2048, dtype, rms, residual=True))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_mean_far_from_zero(dtype):
    """Differences of a hundredth of the mean: the variance is that of the differences."""
    _check(False, *_inputs(40, 1536, dtype, mean=200.0))


@pytest.mark.parametrize("rms", [True, False])
def test_constant_rows(rms):
    for dtype in (BF16, F32):
        for value in (0.0, 3.0):
            x = torch.full((3, 200), value, dtype=dtype, device=DEV)
            _, _, w, b, dy, _ = _inputs(3, 200, dtype, rms)
            _check(rms, x, None, w, b, dy, eps=1e-5)


def test_far_values():
    """Rows whose squares leave the type's range, but not that of 32 bits."""
    for dtype, scale in ((F16, 3e4), (BF16, 1e15), (F32, 1e15), (F32, 1e-12)):
        x = _randn(_gen(3), 6, 520, dtype=F32).clamp(-2, 2).mul(scale).to(dtype)
        _, _, w, b, dy, _ = _inputs(6, 520, dtype)
        for rms in (True, False):
            _check(rms, x, None, w, None if rms else b, dy if dtype == F16 else None, eps=0.0)


def test_shapes_and_strides():
    g = _gen(4)
    for dtype in (BF16, F32):
        for rms in (True, False):
            _, _, w, b, _, _ = _inputs(1, 96, dtype, rms)
            x3, d3 = _randn(g, 3, 5, 96, dtype=dtype), _randn(g, 3, 5, 96, dtype=dtype)
            _check(rms, x3, None, w, b, d3)
            _check(rms, x3, d3, w, b, d3, x3)
            one = _randn(g, 96, dtype=dtype)
            _check(rms, one, None, w, b, one)
            wide, dwide = _randn(g, 20, 160, dtype=dtype), _randn(g, 20, 104, dtype=dtype)
            for lo in (0, 1, 8):  # rows apart, unaligned, aligned again
                _check(rms, wide[:, lo:lo + 96], wide[:, 64 - lo:160 - lo], w, b, dwide[:, lo:lo + 96], dwide[:, 8:])
            _check(rms, _randn(g, 96, 20, dtype=dtype).t(), None, w, b, dwide[:1, :96].expand(20, 96))
            _check(rms, x3.transpose(0, 1), None, w.flip(0)[::1], b, d3.transpose(0, 1))
            off = torch.cat([w, w])[1:97]  # parameters off 16 bytes
            _check(rms, x3, None, off, None if rms else off, d3)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty_batches(dtype):
    x = torch.empty((0, 64), dtype=dtype, device=DEV, requires_grad=True)
    w = torch.ones(64, dtype=dtype, device=DEV, requires_grad=True)
    y, s = rms_norm(x, w, residual=x)
    assert y.shape == s.shape == (0, 64)
    dx, dw = torch.autograd.grad([y, s], [x, w], [y.detach(), s.detach()])
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("cols", [64, 200, 4096])
def test_a_row_stays_its_own(cols, bad):
    """What is wrong in one row is in no other, in any output."""
    for rms in (True, False):
        x, r, w, b, dy, ds = _inputs(9, cols, BF16, rms, residual=True)
        keep = torch.arange(9, device=DEV) != 4
        clean = [t[:, :] if t.dim() == 2 else t for t in _check(rms, x, r, w, b, dy, ds)[:2]]
        x = x.clone()
        x[4, cols // 2] = bad
        leaves = [t.detach().requires_grad_() for t in (x, r, w)]
        y, s = _call(rms, leaves[0], leaves[2], b, leaves[1])
        dx, _, dw = torch.autograd.grad([y, s], leaves, [dy, ds])
        assert torch.equal(y.detach()[keep], clean[0][keep])
        assert torch.equal(dx[keep], clean[1][keep])
        assert not torch.isfinite(y.detach()[4]).all() and dw.isnan().any()


def test_parts_of_the_outputs():
    """Only the sum is used, only y is, only some inputs want gradients."""
    x, r, w, b, dy, ds = _inputs(30, 160, BF16, residual=True)
    leaves = [t.requires_grad_() for t in (x, r, w, b)]
    y, s = layer_norm(x, w, b, EPS, residual=r)
    got = torch.autograd.grad([s], leaves, [ds], retain_graph=True)
    assert torch.equal(got[0], ds) and torch.equal(got[1], ds)
    assert not got[2].any() and not got[3].any()
    ref = norm(s.detach(), w, b, EPS, False, BF16, None, dy)
    for t, key in zip(torch.autograd.grad([y], leaves, [dy]), ("dx", "dx", "dw", "db")):
        check(t, *ref[key], what=key)
    for i in range(4):
        one = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        y, s = layer_norm(one[0], one[2], one[3], EPS, residual=one[1])
        assert s.requires_grad == y.requires_grad
        (t,) = torch.autograd.grad([y], [one[i]], [dy])
        check(t, *ref[("dx", "dx", "dw", "db")[i]], what=str(i))


def test_one_tensor_as_x_and_residual():
    x, _, w, _, dy, _ = _inputs(12, 128, F32, rms=True)
    x.requires_grad_()
    y, s = rms_norm(x, w, EPS, residual=x)
    (dx,) = torch.autograd.grad([y], [x], [dy])
    value, bound = norm(2 * x.detach(), w, None, EPS, True, F32, None, dy)["dx"]
    check(dx, 2 * value, 2 * bound + 2.0 ** -24 * value.abs())


@pytest.mark.parametrize("rows,cols", [(3000, 128), (700, 4096), (513, 1001)])
def test_repeated_calls_agree_bit_for_bit(rows, cols):
    a = _inputs(rows, cols, BF16, residual=True)
    runs = [_check(False, *a) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_offsets_beyond_4_gib():
    """Rows whose elements lie past 2^31, through a pitch."""
    rows, cols, pitch = 70000, 128, 32768
    buf = torch.empty((rows, pitch), dtype=BF16, device=DEV)
    x = buf[:, 1000:1000 + cols]
    x.copy_(_randn(_gen(2), rows, cols, dtype=BF16))
    _, _, w, b, _, _ = _inputs(1, cols, BF16)
    tail = x[-200:].contiguous()
    y = layer_norm(x, w, b, EPS)
    check(y[-200:], *norm(tail, w, b, EPS, False, BF16)["y"])
    leaf = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad([layer_norm(leaf, w, b, EPS)], [leaf], [buf[:, 1000:1000 + cols]])
    check(dx[-200:], *norm(tail, w, b, EPS, False, BF16, None, tail)["dx"])


def test_side_stream_and_two_at_once():
    x, r, w, b, dy, ds = _inputs(900, 1000, BF16, residual=True)
    leaves = [t.requires_grad_() for t in (x, r, w, b)]

    def step():
        y, s = layer_norm(x, w, b, EPS, residual=r)
        return [y.detach(), *torch.autograd.grad([y, s], leaves, [dy, ds])]

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


@pytest.mark.parametrize("rows", [1, 40, 3000])
def test_captured_training_step(rows):
    """Forward and backward in a graph, replayed over new inputs between eager calls."""
    x, r, w, b, dy, ds = _inputs(rows, 264, BF16, residual=True)
    leaves = [t.requires_grad_() for t in (x, r, w, b)]

    def step():
        y, s = layer_norm(x, w, b, EPS, residual=r)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [dy, ds])]

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
            x.copy_(_randn(_gen(60 + i), rows, 264, dtype=BF16))
            w.copy_(_randn(_gen(70 + i), 264, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(p, q) for p, q in zip(got, step())), i


def test_margins_are_left_alone():
    """The C calls write their results and nothing around them, and the workspace within its bytes."""
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for rows, cols, dtype in ((37, 1001, F32), (130, 264, BF16), (5, 16384, BF16), (2000, 64, F16)):
        code = {F32: 0, F16: 1, BF16: 2}[dtype]
        x, r, w, b, dy, ds = _inputs(rows, cols, dtype, residual=True)
        want = _check(False, x, r, w, b, dy, ds)
        room = [torch.full((rows * cols + 256,), 5.0, dtype=dtype, device=DEV) for _ in range(3)]
        y, s, dx = (t[128:128 + rows * cols] for t in room)
        vectors = torch.full((3, cols + 256), 5.0, dtype=dtype, device=DEV)
        dw, db = vectors[0, 128:128 + cols], vectors[1, 128:128 + cols]
        stats = torch.full((2 * rows + 64,), 5.0, device=DEV)
        need = lib.smx_norm_grad_workspace_size(0, rows, cols, code)
        ws = torch.full((need + 512,), 77, dtype=torch.uint8, device=DEV)
        assert lib.smx_norm(0, x.data_ptr(), cols, r.data_ptr(), cols, code, rows, cols, w.data_ptr(), b.data_ptr(), code, EPS,
                            y.data_ptr(), s.data_ptr(), stats.data_ptr(), stream) == 0
        assert lib.smx_norm_grad(0, dy.data_ptr(), cols, ds.data_ptr(), cols, s.data_ptr(), cols, code, rows, cols, w.data_ptr(),
                                 code, stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need, stream) == 0
        torch.cuda.synchronize()
        for t, v in zip((y, dx, dx, dw, db), want):
            assert torch.equal(t, v.flatten())
        assert all((t[:128] == 5).all() and (t[-128:] == 5).all() for t in room)
        assert (vectors[:2, :128] == 5).all() and (vectors[:2, 128 + cols:] == 5).all() and (vectors[2] == 5).all()
        assert (stats[2 * rows:] == 5).all() and (ws[need:] == 77).all()


def test_gradients_against_differences():
    """Directional derivatives of the kernels' own fp32 loss, in each input."""
    g = _gen(8)
    for rms in (True, False):
        x, r, w, b, dy, ds = _inputs(20, 48, F32, rms, residual=True)
        named = [t for t in (x, r, w, b) if t is not None]
        leaves = [t.detach().requires_grad_() for t in named]

        def loss(v):
            y, s = _call(rms, v[0], v[2], v[3] if not rms else None, v[1])
            return (y.to(F64) * dy.to(F64)).sum() + (s.to(F64) * ds.to(F64)).sum()

        y, s = _call(rms, leaves[0], leaves[2], leaves[3] if not rms else None, leaves[1])
        grads = torch.autograd.grad([y, s], leaves, [dy, ds])
        for i, grad in enumerate(grads):
            way = _randn(g, *named[i].shape)
            h = 2.0 ** -7
            up = [t + h * way if j == i else t for j, t in enumerate(named)]
            down = [t - h * way if j == i else t for j, t in enumerate(named)]
            slope = float((loss(up) - loss(down)) / (2 * h))
            want = float((grad.to(F64) * way.to(F64)).sum())
            # the loss's terms (about 2000, of a few units) are off by 2^-22 each, in random directions at best and all
            # one way at worst: 2000 * 8 * 2^-22 / h = 0.5; the curve by h^2 / 6 of a third derivative, some units a row
            assert abs(slope - want) < 0.5 + 20 * h * h * 10, (rms, i, slope, want)


def test_differentiable_once():
    x, _, w, _, dy, _ = _inputs(8, 40, F32, rms=True)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(rms_norm(x, w), [x], dy, create_graph=True)
    check(dx.detach(), *norm(x.detach(), w, None, EPS, True, F32, None, dy)["dx"])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(dx.sum(), [x])


def test_saved_tensors_may_move():
    """Activations kept on the host between the passes."""
    x, r, w, b, dy, ds = _inputs(40, 128, BF16, residual=True)
    leaves = [t.requires_grad_() for t in (x, r, w, b)]
    want = torch.autograd.grad(layer_norm(x, w, b, residual=r), leaves, [dy, ds])
    with torch.autograd.graph.save_on_cpu():
        outs = layer_norm(x, w, b, residual=r)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(outs, leaves, [dy, ds]), want))


def test_refusals_on_the_gpu():
    x = torch.zeros(3, 16385, device=DEV)
    with pytest.raises(SmxError, match="supported"):
        layer_norm(x)
    with pytest.raises(ValueError, match="weight on"):
        rms_norm(x[:, :64], torch.ones(64))
    with pytest.raises(TypeError, match="mismatch"):
        rms_norm(x[:, :64].bfloat16(), torch.ones(64, device=DEV).half())


def test_a_changed_sum_is_noticed():
    """The backward pass reads the kept sum: changing it in between is torch's error, not a wrong gradient."""
    x, r, w, _, dy, ds = _inputs(8, 64, F32, rms=True, residual=True)
    x.requires_grad_()
    y, s = rms_norm(x, w, residual=r)
    s.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([y], [x], [dy])


def test_the_serving_norm_beside_it():
    """RMSNorm's own result, within the one rounding of the sum that rms_norm normalises."""
    x, r, w, _, _, _ = _inputs(7, 256, F32, rms=True, residual=True)
    layer = RMSNorm(256, EPS).to(DEV)
    layer.weight.data.copy_(w)
    a, b = x.clone(), r.clone()
    layer(a, b)
    y, s = rms_norm(x, w, EPS, residual=r)
    assert torch.equal(s, b)
    want, bound = norm(s, w, None, EPS, True, F32)["y"]
    check(y, want, bound)
    check(a, want, bound)


@pytest.mark.parametrize("cols", [2, 4, 32])
def test_a_large_mean_over_fewer_columns_than_threads(cols):
    # Columns are a power of two, so the mean of equal values is exact and n is 0; mean * rstd = 2^113 1e6 passes fp32's range,
    # and nothing behind the row's end may take part with it. dx = rstd (dy - mean of dy), dw = 0.
    dy = torch.randint(-8, 9, (5, cols), generator=torch.Generator().manual_seed(cols)).float().cuda()
    x = torch.full((5, cols), 2.0 ** 113, device="cuda").requires_grad_()
    w = torch.ones(cols, device="cuda").requires_grad_()
    b = torch.full((cols,), 0.5, device="cuda").requires_grad_()
    y = layer_norm(x, w, b, 1e-12)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    assert torch.equal(y, torch.full_like(y, 0.5)) and torch.equal(dw, torch.zeros_like(dw)) and torch.equal(db, dy.sum(0))
    want = (dy.double() - dy.double().mean(1, keepdim=True)) * 1e6
    # Sums of small integers are exact; roundings: eps to fp32 (half of it in its root), rsqrt (1 ulp, two half steps),
    # and the product: 3.5 half steps.
    assert ((dx.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


def test_batched_gradients_refused():
    """torch.autograd.grad over a batch of gradients runs the backward pass on tensors that stand for others."""
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    y = rms_norm(x)
    with pytest.raises(RuntimeError, match="vmap"):
        torch.autograd.grad(y, x, torch.ones(2, 3, 8, device=DEV), is_grads_batched=True)


def test_compiled_around():
    """torch.compile leaves the call as it is, between what it compiles."""
    x, w = torch.randn(30, 64, device=DEV), torch.randn(64, device=DEV)
    call = torch.compile(lambda t: 2.0 * rms_norm(t + 1.0, w), backend="eager")
    assert torch.equal(call(x), 2.0 * rms_norm(x + 1.0, w))
    assert torch.equal(call(x + 1.0), 2.0 * rms_norm((x + 1.0) + 1.0, w))  # (rounded in the same steps)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols,offset", [(70001, 128, 0), (70001, 128, 1), (131077, 64, 0), (40003, 256, 0), (20011, 512, 3),
                                              (30001, 1024, 0), (20011, 2048, 0), (9001, 4096, 0), (5003, 16384, 0)])
def test_no_row_is_left_out_of_the_column_sums(rows, cols, offset, dtype):
    """Rows of +-1 whose mean is 0 and whose variance is 1, small whole gradients: every sum is a whole number below
    2^24, so the parameters' gradients in 32 bits are exact, and a row too few or too many shows."""
    g = _gen(rows + cols)
    sign = torch.where(torch.randperm(cols, generator=g, device=DEV) < cols // 2, 1.0, -1.0)
    flip = torch.where(torch.rand((rows, 1), generator=g, device=DEV) < 0.5, 1.0, -1.0)
    wide = torch.empty((rows, cols + 8), dtype=dtype, device=DEV)
    x = wide[:, offset:offset + cols] if offset else torch.empty((rows, cols), dtype=dtype, device=DEV)
    x.copy_(flip * sign)
    dy = torch.randint(-2, 3, (rows, cols), generator=g, device=DEV).to(dtype)
    w = torch.ones(cols, device=DEV, requires_grad=True)
    b = torch.zeros(cols, device=DEV, requires_grad=True)
    sums = (dy.float() * x.float()).sum(0, dtype=F64), dy.sum(0, dtype=F64)
    y = rms_norm(x, w, 0.0)
    assert torch.equal(y.detach(), x)
    assert torch.equal(torch.autograd.grad(y, w, dy)[0].double(), sums[0])
    y = layer_norm(x, w, b, 0.0)
    assert torch.equal(y.detach(), x)
    assert all(torch.equal(p.double(), q) for p, q in zip(torch.autograd.grad(y, [w, b], dy), sums))

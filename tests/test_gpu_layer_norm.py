"""Layer norm (``nsr_hip.ops.layer_norm*``, ``nsr.layers.LayerNorm``) against its formula in 64 bits.

Tolerances are worst-case bounds: u = 2^-24 is a rounding of fp32; a lane adds at most ceil(width / 64) values of a row before
the lanes are added in 6 steps, so a row's sum of terms t is off by at most (ceil(width / 64) + 6) u sum|t| (+ the roundings of
each term); a value stored in a type with spacing eps is off by eps / 2 relative to itself (+ half its smallest subnormal).  A
column's sum over the rows adds at most rows / 1024 + 264 values in one chain."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _store(v, dtype):
    """bound of the rounding of values v to dtype"""
    return v.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _inputs(rows, width, dtype, affine, seed=0, mean=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return ((1.5 * new(rows, width) + mean * new(rows, 1)).to(dtype), (1 + 0.2 * new(width)).to(affine),
            (0.1 * new(width)).to(affine), new(rows, width).to(dtype))


def _reference(x, w, b, eps):
    """y, its bound, mean, rstd and their bounds"""
    x64 = x.double()
    n = x.shape[-1]
    k = math.ceil(n / 64) + 6
    mean = x64.mean(-1, keepdim=True)
    var = (x64 - mean).square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    d_mean = (k + 2) * U * x64.abs().mean(-1, keepdim=True)
    rel = (k + 10) * U + (d_mean * rstd).square()  # of the variance with eps: its sum, the division, what the mean adds
    h = (x64 - mean) * rstd
    w64 = 1.0 if w is None else w.double()
    y = h * w64 + (0.0 if b is None else b.double())
    d_h = rstd * d_mean * (1 + rel) + h.abs() * (rel + 6 * U)
    tol = d_h * abs(w64) + 3 * U * (h * w64).abs() + U * y.abs()
    return y, tol + _store(y, x.dtype), mean[..., 0], rstd[..., 0], (d_mean[..., 0] + U * mean[..., 0].abs(),
                                                                   rstd[..., 0] * (rel[..., 0] + 4 * U))


def _reference_backward(dy, x, w, mean, rstd):
    n, rows = x.shape[-1], x.numel() // x.shape[-1]
    k = math.ceil(n / 64) + 6
    d, s = dy.double(), rstd.double()[..., None]
    h = (x.double() - mean.double()[..., None]) * s
    g = d * (1.0 if w is None else w.double())
    a, c = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = s * (g - a - h * c)
    tol = s.abs() * (k + 12) * U * (g.abs() + g.abs().mean(-1, keepdim=True) + h.abs() * (g * h).abs().mean(-1, keepdim=True))
    chain = rows / 1024 + 264 + 8
    flat = lambda t: t.reshape(-1, n)  # noqa: E731
    dw, db = flat(d * h).sum(0), flat(d).sum(0)
    return (dx, tol + _store(dx, x.dtype)), (dw, chain * U * flat(d * h).abs().sum(0)), (db, chain * U * flat(d).abs().sum(0))


def _close(got, want, tol, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = float((off - tol).max()) if off.numel() else 0.0
    assert worst <= 0.0, (what, float(off.max()), worst)


SHAPES = [(1, 1), (1, 64), (3, 2), (5, 7), (64, 64), (257, 65), (1000, 8), (33, 777), (2, 1024), (9, 1025), (4, 4096), (3, 5000),
          (2, 20000), (2, 65537), (1030, 96), (5000, 33), (70000, 64), (7, 16384), (20, 2048), (3000, 16), (513, 512)]


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype,affine", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_forward_and_backward_match_the_formula(rows, width, dtype, affine):
    from nsr_hip import ops
    x, w, b, dy = _inputs(rows, width, dtype, affine)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, 1e-5)
    want, tol, m64, s64, (dm, ds) = _reference(x, w, b, 1e-5)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == F32 and mean.shape == (rows,)
    _close(y, want, tol, "y")
    _close(mean, m64, dm, "mean")
    _close(rstd, s64, ds, "rstd")
    assert torch.equal(ops.layer_norm(x, w, b, 1e-5), y)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    (r, t), (rw, tw), (rb, tb) = _reference_backward(dy, x, w, mean, rstd)
    _close(dx, r, t, "dx")
    _close(dw, rw, tw + _store(rw, affine), "dweight")
    _close(db, rb, tb + _store(rb, affine), "dbias")
    again = ops.layer_norm_backward(dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))  # the same bits


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_missing_affine_parts(weight, bias, dtype):
    from nsr_hip import ops
    x, w, b, dy = _inputs(129, 130, dtype, dtype, 1)
    w, b = (w if weight else None), (b if bias else None)
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    want, tol = _reference(x, w, b, 1e-5)[:2]
    _close(y, want, tol, "y")
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, want_dweight=weight, want_dbias=bias)
    (r, t), (rw, tw), (rb, tb) = _reference_backward(dy, x, w, mean, rstd)
    _close(dx, r, t, "dx")
    assert (dw is None) == (not weight) and (db is None) == (not bias)
    if weight:
        _close(dw, rw, tw + _store(rw, dtype), "dweight")
    if bias:
        _close(db, rb, tb + _store(rb, dtype), "dbias")
    only = ops.layer_norm_backward(dy, x, w, mean, rstd, want_dx=False)
    assert only[0] is None and only[1].dtype == only[2].dtype == dtype


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width,stride,offset", [(64, 80, 0), (64, 67, 0), (64, 64, 3), (100, 101, 1), (777, 800, 5), (4096, 4099, 1),
                                                 (128, 136, 8)])
def test_row_strides_and_unaligned_rows(dtype, width, stride, offset):
    """rows that are slices of wider ones, at addresses that no vector load takes; what lies between the rows stays"""
    from nsr_hip import ops
    x, w, b, dy = _inputs(50, width, dtype, dtype, 2)
    wide = torch.full((50 * stride + offset,), float("nan"), dtype=dtype, device="cuda")
    dwide = wide.clone()
    xs, ds = (t[offset:].as_strided((50, width), (stride, 1)) for t in (wide, dwide))
    xs.copy_(x)
    ds.copy_(dy)
    y, mean, rstd = ops.layer_norm_forward(xs, w, b)
    dx, dw, db = ops.layer_norm_backward(ds, xs, w, mean, rstd)
    want, tol = _reference(x, w, b, 1e-5)[:2]
    _close(y, want, tol, "y")
    (r, t), (rw, tw), (rb, tb) = _reference_backward(dy, x, w, mean, rstd)
    _close(dx, r, t, "dx")
    _close(dw, rw, tw + _store(rw, dtype), "dweight")
    _close(db, rb, tb + _store(rb, dtype), "dbias")
    # weights and gradients at odd addresses too
    wo, bo = (torch.cat([t[:1], t])[1:] for t in (w, b))
    assert torch.equal(ops.layer_norm(xs, wo, bo), y)


def test_shapes_layouts_and_batches():
    from nsr_hip import ops
    x, w, b, dy = _inputs(24, 40, F32, F32, 3)
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    y3, m3, _ = ops.layer_norm_forward(x.view(2, 3, 4, 40), w, b)
    assert y3.shape == (2, 3, 4, 40) and m3.shape == (2, 3, 4) and torch.equal(y3.view(24, 40), y)
    xt = x.t().contiguous().t()  # columns dense, not rows
    assert torch.equal(ops.layer_norm(xt, w, b), y)
    assert torch.equal(ops.layer_norm(x[0], w, b), y[0])
    same = ops.layer_norm(x[:1].expand(5, 40), w, b)
    assert torch.equal(same, y[:1].expand(5, 40))
    want = ops.layer_norm_backward(dy[:1].expand(24, 40).contiguous(), x, w, mean, rstd)
    got = ops.layer_norm_backward(dy[:1].expand(24, 40), xt, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    w2 = torch.stack([w, w], 1)[:, 0]  # a strided weight
    assert torch.equal(ops.layer_norm(x, w2, b), y)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_rows(dtype):
    from nsr_hip import ops
    x = torch.empty(0, 64, dtype=dtype, device="cuda")
    w = torch.ones(64, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x, w, w)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = ops.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 64) and float(dw.abs().max()) == 0.0 and float(db.abs().max()) == 0.0


def test_rows_without_spread_and_large_values():
    """constant rows have no variance but eps; rows of 1e18 have squares past fp32 only after centring, rows of 1e-20 none"""
    from nsr_hip import ops
    x = torch.full((4, 96), 3.25, device="cuda")
    x[1] = 0.0
    x[2] = torch.linspace(-1e18, 1e18, 96, device="cuda")
    x[3] = torch.linspace(-1e-20, 1e-20, 96, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x, None, None, 1e-5)
    want, tol, _, s64, _ = _reference(x, None, None, 1e-5)
    _close(y, want, tol, "y")
    assert abs(float(rstd[1]) / float(s64[1]) - 1) < 1e-6 and abs(float(rstd[2]) / float(s64[2]) - 1) < 1e-5
    # one NaN or infinity stays in its row
    x = torch.randn(6, 70, device="cuda")
    clean = ops.layer_norm(x)
    x[2, 5], x[4, 69] = float("nan"), float("inf")
    y = ops.layer_norm(x)
    assert torch.isnan(y[2]).all() and torch.isnan(y[4, 69]) and torch.equal(y[[0, 1, 3, 5]], clean[[0, 1, 3, 5]])


@pytest.mark.parametrize("rows,width", [(6, 5), (3, 70)])
def test_gradients_against_differences(rows, width):
    """the gradient of sum(y dy) against central differences of the formula in 64 bits: step h, truncation h^2 / 6 f''' and
    rounding 2^-53 f / h leave under 1e-6 of the gradient's scale at h = 1e-5; the kernel's own fp32 bound comes on top"""
    from nsr_hip import ops
    x, w, b, dy = _inputs(rows, width, F32, F32, 4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    ops.layer_norm(*leaves, 1e-5).backward(dy)

    def f(x, w, b):
        c = x - x.mean(-1, keepdim=True)
        return float((((c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt()) * w + b) * dy.double().cpu()).sum())

    at = [t.double().cpu() for t in (x, w, b)]
    for k, leaf in enumerate(leaves):
        flat = at[k].view(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 17)):
            keep = float(flat[i])
            flat[i] = keep + 1e-5
            up = f(*at)
            flat[i] = keep - 1e-5
            down = f(*at)
            flat[i] = keep
            assert abs(float(leaf.grad.view(-1)[i]) - (up - down) / 2e-5) < 1e-4 * max(1.0, float(leaf.grad.abs().max())), (k, i)


def test_module_autograd_and_once_differentiable():
    from nsr.layers import LayerNorm
    from nsr_hip import ops
    ln = LayerNorm(48).cuda()
    assert sorted(ln.state_dict()) == ["bias", "weight"] and LayerNorm(48, bias=False).bias is None
    x, w, b, dy = _inputs(30, 48, BF16, F32, 5)
    with torch.no_grad():
        ln.weight.copy_(w)
        ln.bias.copy_(b)
    xl = x.clone().requires_grad_()
    y = ln(xl)
    assert y.dtype == BF16 and torch.equal(y, ops.layer_norm(x, w, b))
    y.backward(dy)
    _, mean, rstd = ops.layer_norm_forward(x, w, b)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    assert torch.equal(xl.grad, dx) and torch.equal(ln.weight.grad, dw) and torch.equal(ln.bias.grad, db)
    only_bias = b.clone().requires_grad_()
    ops.layer_norm(x, None, only_bias).backward(dy)
    assert only_bias.grad.dtype == F32 and torch.equal(only_bias.grad, db)
    g, = torch.autograd.grad(ln(xl).float().sum(), xl, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_graph_replays_other_stream_and_two_graphs():
    from nsr_hip import ops
    x, w, b, dy = _inputs(300, 200, F32, F32, 6)
    eager = ops.layer_norm_forward(x, w, b) + ops.layer_norm_backward(dy, x, w, *ops.layer_norm_forward(x, w, b)[1:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = ops.layer_norm_forward(x, w, b) + ops.layer_norm_backward(dy, x, w, *eager[1:3])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(there, eager))
    graphs = []
    for _ in range(2):
        xi, di = x.clone(), dy.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, mean, rstd = ops.layer_norm_forward(xi, w, b)
            out = ops.layer_norm_backward(di, xi, w, mean, rstd)
        graphs.append((g, xi, di, (y, mean, rstd) + out))
    for k in range(4):
        for g, xi, di, _ in graphs:
            xi.copy_(x * (k + 1)), di.copy_(dy - k)
            g.replay()
        f = ops.layer_norm_forward(x * (k + 1), w, b)
        want = f + ops.layer_norm_backward(dy - k, x * (k + 1), w, *f[1:])
        torch.cuda.synchronize()
        for *_, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_offsets_past_32_bits():
    """2^32 elements and a few rows more: the last rows are those of a small call"""
    from nsr_hip import ops
    width = 4096
    rows = (1 << 20) + 3
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    tail, w, b, dt = _inputs(5, width, BF16, BF16, 7)
    x[-5:] = tail
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    small = ops.layer_norm_forward(tail, w, b)
    assert torch.equal(y[-5:], small[0]) and torch.equal(mean[-5:], small[1]) and torch.equal(y[0], b)
    del y
    dy = torch.zeros_like(x)
    dy[-5:] = dt
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    ref = ops.layer_norm_backward(dt, tail, w, *small[1:])
    assert torch.equal(dx[-5:], ref[0]) and float(dx[:-5].float().abs().max()) == 0.0
    for got, want, terms in ((dw, ref[1], 5), (db, ref[2], 5)):  # (other orders of the same five terms, rounded to bf16)
        assert float((got.float() - want.float()).abs().max()) <= float(want.float().abs().max()) * 2.0 ** -7


def test_refusals_on_the_gpu():
    from nsr_hip import NsrError, ops
    x, w, b, dy = _inputs(4, 32, F32, F32, 8)
    _, mean, rstd = ops.layer_norm_forward(x, w, b)
    for bad in (lambda: ops.layer_norm(x.double(), None, None), lambda: ops.layer_norm(x, w[:31], b),
                lambda: ops.layer_norm(x, w.half(), b.half()), lambda: ops.layer_norm(x, w, b.cpu()),
                lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x.half(), w, b.half()),
                lambda: ops.layer_norm_backward(dy[:3], x, w, mean, rstd),
                lambda: ops.layer_norm_backward(dy.half(), x, w, mean, rstd),
                lambda: ops.layer_norm_backward(dy, x, w, mean[:3], rstd),
                lambda: ops.layer_norm_backward(dy, x, w, mean.double(), rstd), lambda: ops.layer_norm(x, w, b, -1.0)):
        with pytest.raises((NsrError, ValueError)):
            bad()


@pytest.mark.parametrize("rows,width", [(37, 9001), (33, 12288), (21, 12289), (600, 5001), (300, 129), (1200, 1001), (530, 16384),
                                        (700, 8192), (2100, 17), (257, 4), (1025, 7), (8200, 9), (300, 513), (70, 2049)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_and_access_boundaries(rows, width, dtype):
    """widths around the sizes where rows go to larger groups of lanes, to the element-wise and to the long form; 16-bit rows at odd
    addresses; row counts that leave the last tile of rows partly empty"""
    from nsr_hip import ops
    x, w, b, dy = _inputs(rows, width, dtype, F32, 11)
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    want, tol, m64, s64, (dm, ds) = _reference(x, w, b, 1e-5)
    _close(y, want, tol, "y")
    _close(mean, m64, dm, "mean")
    _close(rstd, s64, ds, "rstd")
    assert torch.equal(ops.layer_norm(x, w, b), y)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    (r, t), (rw, tw), (rb, tb) = _reference_backward(dy, x, w, mean, rstd)
    _close(dx, r, t, "dx")
    _close(dw, rw, tw + _store(rw, F32), "dweight")
    _close(db, rb, tb + _store(rb, F32), "dbias")
    for wants in ((True, False, False), (False, True, False), (False, False, True)):
        part = ops.layer_norm_backward(dy, x, w, mean, rstd, *wants)
        assert all((p is None) if not k else torch.equal(p, q) for k, p, q in zip(wants, part, (dx, dw, db)))


@pytest.mark.parametrize("width", [64, 65, 257, 5001])
def test_infinities_stay_in_their_row_and_columns(width):
    """an infinite dy in the last row of a partly filled tile: the columns' sums are infinite there and exact elsewhere"""
    from nsr_hip import ops
    x, w, b, dy = _inputs(131, width, BF16, F32, 12)
    _, mean, rstd = ops.layer_norm_forward(x, w, b)
    clean = ops.layer_norm_backward(dy, x, w, mean, rstd)
    dy[130, 3] = float("inf")
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    assert torch.equal(dx[:130], clean[0][:130])
    keep = torch.arange(width, device="cuda") != 3
    assert torch.equal(dw[keep], clean[1][keep]) and torch.equal(db[keep], clean[2][keep])
    assert float(db[3]) == float("inf") and torch.isinf(dw[3])


def test_one_row_with_any_stride_through_the_c_entry():
    """a single row has no stride: the C entry takes 0 for it (and no row past the end adds to the sums)"""
    from nsr_hip import check, lib, ops, ptr, stream_ptr
    x, w, b, dy = _inputs(1, 64, F32, F32, 13)
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    y0, dx0, dw0, db0 = (torch.empty_like(t) for t in (y, dx, dw, db))
    check(lib.nsr_layer_norm_forward(ptr(x), 0, ptr(w), ptr(b), ptr(y0), None, None, 1, 64, 0, 0, 1e-5, stream_ptr()))
    check(lib.nsr_layer_norm_backward(ptr(dy), 0, ptr(x), 0, ptr(w), ptr(mean), ptr(rstd), ptr(dx0), ptr(dw0), ptr(db0), None, 1, 64,
                                      0, 0, stream_ptr()))
    assert all(torch.equal(p, q) for p, q in ((y, y0), (dx, dx0), (dw, dw0), (db, db0)))


@pytest.mark.parametrize("dtype,width", [(F32, 8), (BF16, 16), (BF16, 9), (F32, 3)])
def test_more_rows_than_workgroups_at_once(dtype, width):
    """so many narrow rows that every workgroup walks several tiles"""
    from nsr_hip import ops
    rows = 4_300_001
    x, w, b, dy = _inputs(rows, width, dtype, F32, 14)
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    want, tol = _reference(x, w, b, 1e-5)[:2]
    _close(y, want, tol, "y")
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    (r, t), (rw, tw), (rb, tb) = _reference_backward(dy, x, w, mean, rstd)
    _close(dx, r, t, "dx")
    _close(dw, rw, tw + _store(rw, F32), "dweight")
    _close(db, rb, tb + _store(rb, F32), "dbias")


@pytest.mark.parametrize("width", [64, 65, 4096])
def test_variances_below_the_smallest_normal_number(width):
    from nsr_hip import ops

    x = torch.randn(9, width, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 1e-20
    y, mean, rstd = ops.layer_norm_forward(x, eps=0.0)
    x64 = x.double()
    mean64 = x64.mean(-1, keepdim=True)
    var = (x64 - mean64).square().mean(-1, keepdim=True)  # about 1e-40
    # each square and the mean of them is rounded to a multiple of 2^-149, so the variance is off by at most 2^-149 more
    # than the roundings and the mean's error that rows of any size have; rstd by half of that relative to itself
    k = math.ceil(width / 64) + 6
    d_mean = (k + 2) * U * x64.abs().mean(-1, keepdim=True)
    rel = (k + 10) * U + 2.0 ** -149 / var + d_mean.square() / var
    assert ((rstd.double()[:, None] - var.rsqrt()).abs() <= var.rsqrt() * (rel + 4 * U)).all()
    h = (x64 - mean64) * var.rsqrt()
    assert ((y.double() - h).abs() <= var.rsqrt() * d_mean * (1 + rel) + h.abs() * (rel + 8 * U)).all()

"""Layer norm of rows whose mean is far above their spread, and of rows without any, in every form of the kernel.

Bounds: u = 2^-24 is a rounding of fp32, k = ceil(width / 64) + 6 the additions that a row's sum takes one after another.  The first
mean is off by at most D = (k + 2) u mean|x|.  The centred values' own mean is taken off again: it is exact to
E = (k + 4) u (mean|c| + D) for c the true centred values (the sum's roundings, the quotient, the fold into one fma), so a centred
value is off by E + 3 u (|c| + D).  The variance loses (k + 10) u (var + D^2) to the sum of squares about the first mean and 2 D E to
the square of the correction."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# element by element, groups of 1 .. 64 lanes, of 128 .. 1024 threads, several vectors a lane, the form that reads a row three times
WIDTHS = [3, 8, 13, 64, 65, 102, 257, 777, 1000, 2047, 2049, 5001, 9000, 16384, 16385, 40001]


def _store(v, dtype):
    return v.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _k(width):
    return math.ceil(width / 64) + 6


def _affine(width, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=g, device="cuda") for s in ((width,), (width,), (9, width))]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_of_one_value(dtype, width):
    """the mean is the value, the centred values are 0 (exactly where the sum is: whole numbers under 2^24), y is the bias"""
    from nsr_hip import ops
    eps = 1e-5
    value = torch.tensor([1000.0, 2047.0, -0.1, 3.3, 1.0, 4096.5, 0.0, 1e-3, -777.0], device="cuda").to(dtype)
    x = value[:, None].repeat(1, width)
    w, b, dy = _affine(width, width)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, eps)
    v, k = value.double()[:, None], _k(width)
    D = (k + 2) * U * v.abs()
    E = (k + 7) * U * D  # (c = 0; its 3 u D among them)
    off = E / math.sqrt(eps)
    want = b.double().expand(9, width)
    assert bool(((y.double() - want).abs() <= off * w.double().abs() + U * want.abs() + _store(want, dtype)).all())
    assert torch.equal(mean, value.float())
    rel = ((k + 10) * U * D * D + 2 * D * E)[:, 0] / eps + 4 * U
    assert bool(((rstd.double() * math.sqrt(eps) - 1).abs() <= rel).all())
    whole = (value.float() == value.float().round()) & (value.float().abs() * width < 2 ** 24)
    assert torch.equal(y[whole], b.to(dtype).expand(9, width)[whole]) and bool(whole.any())
    # h is 0, so the weight's gradient is, whatever dy
    _, dw, db = ops.layer_norm_backward(dy.to(dtype), x, w, mean, rstd)
    assert float(dw.abs().max()) == 0.0 and float(db.abs().max()) > 0.0


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("offset", [0, 1])
def test_mean_far_above_the_spread(dtype, width, offset):
    """means so large that D is about half the spread; offset: rows at addresses that are no multiple of 4 bytes (16 bits)"""
    from nsr_hip import ops
    eps, k, rows = 1e-5, _k(width), 9
    m = min(1.37 * 2.0 ** math.floor(math.log2(0.5 / ((k + 2) * U))), 3e4 if dtype is F16 else 1e9)
    spread = max(1.0, 4 * m * torch.finfo(dtype).eps)
    g = torch.Generator(device="cuda").manual_seed(width)
    x = (m + spread * torch.randn(rows, width, generator=g, device="cuda", dtype=torch.float64)).to(dtype)
    flat = torch.zeros(rows * width + offset, dtype=dtype, device="cuda")
    xs = flat[offset:].view(rows, width)
    xs.copy_(x)
    w, b, _ = _affine(width, 1)
    y, mean, rstd = ops.layer_norm_forward(xs, w, b, eps)
    x64 = x.double()
    m64 = x64.mean(-1, keepdim=True)
    c = x64 - m64
    var = c.square().mean(-1, keepdim=True)
    D = (k + 2) * U * x64.abs().mean(-1, keepdim=True)
    E = (k + 4) * U * (c.abs().mean(-1, keepdim=True) + D)
    s = (var + eps).rsqrt()
    rel = ((k + 10) * U * (var + D * D) + 2 * D * E) * s * s
    h = c * s
    off = s * (E + 3 * U * (c.abs() + D)) * (1 + rel) + h.abs() * (rel + 6 * U)
    want = h * w.double() + b.double()
    assert bool(((y.double() - want).abs() <= off * w.double().abs() + 3 * U * (h * w.double()).abs() + U * want.abs()
                 + _store(want, dtype)).all())
    assert bool(((mean.double() - m64[:, 0]).abs() <= (E + U * m64.abs())[:, 0]).all())
    assert bool(((rstd.double() / s[:, 0] - 1).abs() <= rel[:, 0] + 4 * U).all())


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_squares_past_fp32_and_values_that_are_none(dtype, width):
    """rows whose squares overflow fp32 have a reciprocal deviation of 0, as the sum in fp32 says: y is the bias, nothing is NaN.
    A NaN or an infinity makes its own row NaN and no other"""
    from nsr_hip import ops
    g = torch.Generator(device="cuda").manual_seed(width)
    w, b, _ = _affine(width, 2)
    x = torch.randn(9, width, generator=g, device="cuda")
    clean = ops.layer_norm_forward(x.to(dtype), w, b)
    for k, scale in ((1, 1e21), (3, 1e25), (5, 1e30)):
        x[k] = scale * (1 + torch.rand(width, generator=g, device="cuda"))
        x[k, 0] = -scale
    x[6, width // 2], x[7, width - 1] = float("nan"), float("inf")
    y, mean, rstd = ops.layer_norm_forward(x.to(dtype), w, b)
    for k in (1, 3, 5):
        assert torch.equal(y[k], b.to(dtype)) and float(rstd[k]) == 0.0 and torch.isfinite(mean[k])
    assert torch.isnan(y[6]).all() and torch.isnan(y[7]).all() and torch.isnan(mean[6]) and torch.isnan(rstd[6:8]).all()
    rest = [0, 2, 4, 8]
    assert all(torch.equal(p[rest], q[rest]) for p, q in zip((y, mean, rstd), clean))

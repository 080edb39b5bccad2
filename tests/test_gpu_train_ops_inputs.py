"""Inputs that the training operators (``nsr.optim.AdamW``, layer norm) refuse or have to see, on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _bytes(opt):
    return [t.clone().view(torch.uint8) for t in (*opt.flat32.values(), *opt.flat8.values())]


@pytest.mark.parametrize("kind,other", [(F16, BF16), (BF16, F16)])
@pytest.mark.parametrize("bits,clip", [(32, None), (32, 1.0), (8, None)])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("beside_none", [False, True])
def test_gradient_of_the_other_16_bit_type_is_refused(kind, other, bits, clip, strided, beside_none):
    """refused before any launch: parameters, moments and the step count stay"""
    import nsr.optim
    from nsr_hip import NsrError
    ps = [torch.nn.Parameter(torch.randn(70, 60, device="cuda").to(kind)) for _ in range(2)]
    opt = nsr.optim.AdamW(ps, lr=0.1, state_bits=bits, min_8bit_size=0, max_grad_norm=clip)
    for p in ps:
        p.grad = torch.randn(70, 60, device="cuda").to(kind)
    opt.step()
    before, moments = [p.detach().clone() for p in ps], _bytes(opt)
    if beside_none:
        ps[1].grad = None
    g = torch.randn(70, 60, device="cuda").to(other)
    ps[0].grad.data = g.t().contiguous().t() if strided else g
    with pytest.raises(NsrError, match="another size, type or device"):
        opt.step()
    ps[0].grad = None
    ps[0].grad_dtype = other
    ps[0].grad = g
    with pytest.raises(NsrError, match="another size, type or device"):
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, before)) and opt.taken_steps() == 1
    assert all(torch.equal(a, b) for a, b in zip(_bytes(opt), moments))


def test_layer_norm_refuses_forward_mode():
    from torch.autograd import forward_ad
    from nsr.layers import LayerNorm
    from nsr_hip import NsrError, ops
    x, t = torch.randn(2, 5, 16, device="cuda")
    ln = LayerNorm(16).cuda()
    with forward_ad.dual_level():
        xd = forward_ad.make_dual(x, t)
        for call in (lambda: ops.layer_norm(xd), lambda: ops.layer_norm_forward(xd), lambda: ln(xd),
                     lambda: ops.layer_norm(x, forward_ad.make_dual(x[0], t[0]))):
            with pytest.raises(NsrError, match="forward mode"):
                call()
        with torch.no_grad(), pytest.raises(NsrError, match="forward mode"):
            ln(xd)
        assert ops.layer_norm(x).shape == x.shape  # (no tangent among the inputs)
    with pytest.raises(RuntimeError):
        torch.func.jvp(ops.layer_norm, (x,), (t,))


def test_layer_norm_forward_keeps_the_graph():
    """y of the statistics form has the gradients of layer_norm, whichever inputs want them"""
    from nsr_hip import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, b, dy = (torch.randn(*s, generator=g, device="cuda") for s in ((40, 24), (24,), (24,), (40, 24)))
    for wants in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        grads = []
        for f in (ops.layer_norm, lambda *a: ops.layer_norm_forward(*a)[0]):
            leaves = [t.clone().requires_grad_(bool(k)) for t, k in zip((x, w, b), wants)]
            y = f(*leaves)
            y.backward(dy)
            grads.append([y.detach()] + [t.grad for t in leaves if t.requires_grad])
        assert len(grads[0]) == 1 + sum(wants) and all(torch.equal(p, q) for p, q in zip(*grads))
    y, mean, rstd = ops.layer_norm_forward(x.clone().requires_grad_(), w, b)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
    assert all(torch.equal(p, q) for p, q in zip((y, mean, rstd), ops.layer_norm_forward(x, w, b)))
    with torch.no_grad():
        assert not ops.layer_norm_forward(x.clone().requires_grad_(), w, b)[0].requires_grad


@pytest.mark.parametrize("rows,width", [(5, (1 << 25) + 3), (0, (1 << 25) + 3), (1, (1 << 28) + 4099), (6, (1 << 26) + 16)])
def test_layer_norm_backward_of_very_wide_rows(rows, width):
    """grids past 65535 blocks of columns, past 2^32 threads for the partial sums.  The products and the centred values are those of
    torch's fp32 operations; sums of rows in another order, each of the rows additions off by u of the terms' sum at most.  dx is
    looked at where one value of dy alone is not zero: its row's means are that term over the width."""
    from nsr_hip import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, width, generator=g, device="cuda")
    dy = torch.zeros_like(x)
    mean, rstd = torch.full((rows,), 0.25, device="cuda"), torch.full((rows,), 1.5, device="cuda")
    where = torch.tensor([0, 4095, 4096, width // 2 + 1, width - 4, width - 1], device="cuda")
    for r in range(rows):
        dy[r, where] = torch.randn(where.numel(), generator=g, device="cuda")
    dx, dw, db = ops.layer_norm_backward(dy, x, None, mean, rstd)
    assert dx.shape == x.shape and dw.shape == db.shape == (width,)
    d, h = dy[:, where].double(), ((x[:, where] - 0.25) * 1.5).double()
    bound = (rows + 2) * 2.0 ** -24
    assert bool(((dw[where].double() - (d * h).sum(0)).abs() <= bound * (d * h).abs().sum(0)).all())
    assert bool(((db[where].double() - d.sum(0)).abs() <= bound * d.abs().sum(0)).all())
    assert int(torch.count_nonzero(dw)) <= where.numel() and int(torch.count_nonzero(db)) <= where.numel()
    for r in range(rows):
        a, c = float(d[r].sum()) / width, float((d[r] * h[r]).sum()) / width
        want = 1.5 * (d[r] - a - h[r] * c)
        assert bool(((dx[r, where].double() - want).abs() <= 16 * 2.0 ** -24 * (1.5 * d[r].abs() + want.abs() + 1e-6)).all())
        rest = 1.5 * (-a - ((x[r, 7:4000:13] - 0.25) * 1.5).double() * c)
        assert bool(((dx[r, 7:4000:13].double() - rest).abs() <= 64 * 2.0 ** -24 * (d[r].abs().sum() / width * 20)).all())


@pytest.mark.parametrize("rows,width", [(5, 16385), (129, 40001), (300, 16386), (1100, 16385), (40, 1 << 20)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_column_sums_of_long_rows(rows, width, dtype):
    """shares of several rows each: at most ceil(rows / shares) <= 128 additions a share and 128 over the shares, of terms with two
    roundings of their own"""
    from nsr_hip import ops
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, dy = (torch.randn(rows, width, generator=g, device="cuda").to(dtype) for _ in range(2))
    mean, rstd = (torch.rand(rows, generator=g, device="cuda") for _ in range(2))
    _, dw, db = ops.layer_norm_backward(dy, x, None, mean, rstd, want_dx=False, affine_dtype=F32)
    h = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    for got, terms in ((dw, dy.double() * h), (db, dy.double())):
        bound = (128 + 128 + 4) * 2.0 ** -24 * (terms.abs().sum(0) if got is db
                                                else (dy.double().abs() * (x.double().abs() + 1) * rstd.double()[:, None]).sum(0))
        assert bool(((got.double() - terms.sum(0)).abs() <= bound).all())
    assert all(torch.equal(p, q) for p, q in zip((dw, db), ops.layer_norm_backward(dy, x, None, mean, rstd, affine_dtype=F32)[1:]))

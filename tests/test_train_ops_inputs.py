"""Inputs of the training operators (``nsr.optim.AdamW``, layer norm) that are refused before anything reaches a kernel, on the
CPU."""
import numpy as np
import pytest
import torch


def _gathering(p):
    """an optimizer of one tensor as far as the gathering of its gradients goes (construction needs a GPU)"""
    from nsr import optim
    opt = object.__new__(optim.AdamW)
    opt._ps, opt._addresses, opt._all_contiguous = [p], [p.data_ptr()], p.is_contiguous()
    opt._kinds = [[of(p)] for of in (optim._size, optim._dtype, optim._device)]
    opt._desc = (optim.NsrAdamwTensor * 1)()
    opt._fields = np.frombuffer(opt._desc, dtype=optim._DESCRIPTOR)
    return opt


@pytest.mark.parametrize("kind,other,by", [(torch.float16, torch.bfloat16, "data"), (torch.bfloat16, torch.float16, "data"),
                                           (torch.float32, torch.int32, "data"), (torch.float16, torch.bfloat16, "grad_dtype"),
                                           (torch.bfloat16, torch.float16, "grad_dtype")])
@pytest.mark.parametrize("strided", [False, True])
def test_gradient_of_another_type_of_the_same_size(kind, other, strided, by):
    """the kernel reads a gradient with its parameter's type: one of another type is refused in every layout, none is converted"""
    from nsr_hip import NsrError
    p = torch.nn.Parameter(torch.zeros(4, 6, dtype=kind))
    opt = _gathering(p)
    g = torch.ones(4, 6, dtype=other)
    g = g.t().contiguous().t() if strided else g
    if by == "data":
        p.grad = torch.zeros(4, 6, dtype=kind)
        p.grad.data = g
    else:
        p.grad_dtype = other
        p.grad = g
    assert p.grad.dtype == other and p.grad.nbytes == p.nbytes and p.grad.is_contiguous() != strided
    with pytest.raises(NsrError, match="another size, type or device"):
        opt._gather()
    p.grad = None
    p.grad_dtype = kind
    p.grad = torch.ones(4, 6, dtype=kind)
    assert opt._gather()[1] == 1 and opt._fields["grad"][0] == p.grad.data_ptr()


@pytest.mark.parametrize("strided", [False, True])
def test_gradient_on_another_device(strided):
    """an address in another device's memory reaches no kernel (the optimizer's own device is a GPU, the gradient is not there)"""
    from nsr_hip import NsrError
    p = torch.nn.Parameter(torch.zeros(4, 6))
    opt = _gathering(p)
    opt._kinds[2] = [0]
    p.grad = torch.ones(6, 4).t() if strided else torch.ones(4, 6)
    with pytest.raises(NsrError, match="another size, type or device"):
        opt._gather()


@pytest.mark.parametrize("which", ["x", "weight", "bias", "dy", "mean", "rstd"])
def test_layer_norm_refuses_tangents(which):
    """forward mode: a result without its tangent would be a derivative of zero"""
    from torch.autograd import forward_ad
    from nsr_hip import NsrError, ops
    with forward_ad.dual_level():
        dual = lambda name, *shape: (forward_ad.make_dual(torch.ones(*shape), torch.ones(*shape)) if name == which  # noqa: E731
                                     else torch.ones(*shape))
        x, w, b, dy, mean, rstd = (dual(*a) for a in (("x", 3, 8), ("weight", 8), ("bias", 8), ("dy", 3, 8), ("mean", 3), ("rstd", 3)))
        calls = [lambda: ops.layer_norm_backward(dy, x, w, mean, rstd)] if which != "bias" else []
        if which in ("x", "weight", "bias"):
            leaf = torch.ones(8, requires_grad=True)
            calls += [lambda: ops.layer_norm(x, w, b), lambda: ops.layer_norm_forward(x, w, b)]
            calls += [lambda: ops.layer_norm(x, leaf, b)] if which != "weight" else [lambda: ops.layer_norm(x, w, leaf)]
        for call in calls:
            with pytest.raises(NsrError, match="forward mode"):
                call()


def test_partial_sums_of_long_rows_stay_small():
    """the column sums' workspace of the backward pass, two fp32 rows a share of the rows: past the register form (more than 12288
    columns of fp32, 16384 of 16 bits) a share has 128 rows, or fewer where two workgroups a CU need more shares"""
    import nsr_hip
    floats = nsr_hip.lib.nsr_layer_norm_backward_workspace_floats
    for code, narrow, block in ((0, 12289, 4096), (1, 16385, 8192), (2, 16385, 8192)):
        for width in (narrow, 20000, 65537, 1 << 20, (1 << 28) + 5, 1 << 30):
            for rows in (0, 1, 4, 5, 64, 256, 1000, 5000, 1 << 20):
                shares, left = divmod(floats(rows, width, code), 2 * width)
                assert left == 0 and shares <= min(rows, 256)
                assert shares <= max(-(-rows // 128), -(-512 // -(-width // block))), (rows, width)
    assert 4 * floats(256, 1 << 20, 0) == 1 << 24

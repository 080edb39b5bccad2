"""The encode's fp16 features are one fp32 sum rounded once more, the same in every kernel that makes them: one or two levels a
lane, tables from LDS, with the Jacobian, seven taps at once, in front of the network in one kernel."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L,F", [(16, 1), (16, 2), (8, 4), (4, 8)])
def test_every_form_of_the_encode_gives_the_same_bits(L, F):
    import nsr_hip
    from nsr_hip import check, lib, ops, ptr, stream_ptr
    gd = nsr_hip.make_grid_desc(L, F, 14, 16, 1.4)
    g = torch.Generator().manual_seed(F)
    table = ((torch.rand(gd.n_entries * F, generator=g) * 2 - 1) * 0.5).half().cuda()
    n, radius = 20000, 1.0
    eps = 2 * radius / (16 * 1.4 ** (L - 1))  # one cell of the finest level
    o = ((torch.rand(n, 3, generator=g) * 2 - 1) * radius).cuda()
    t0, x7 = torch.zeros(n, device="cuda"), torch.empty(7 * n, 3, device="cuda")
    check(lib.nsr_neus_points(ptr(o), ptr(torch.zeros_like(o)), ptr(torch.arange(n, device="cuda")), ptr(t0), ptr(t0), radius, eps, 1,
                              ptr(x7), None, n, None, stream_ptr()), "nsr_neus_points")
    want = ops.hashgrid_forward(x7, table, gd)
    got = {}
    try:
        # (a level of 16384 entries of 8 features is more than the LDS holds: the launch is refused)
        for variant in ((0, 1), (4, 1), (4, 2)) if F < 8 else ((0, 1),):
            lib.nsr_hashgrid_forward_variant(*variant)
            got[variant] = ops.hashgrid_forward(x7, table, gd)
    finally:
        lib.nsr_hashgrid_forward_variant(0, 2)
    got["jacobian"], jac = torch.empty_like(want), torch.empty(L * 7 * n * F * 3, device="cuda")
    check(lib.nsr_hashgrid_forward_jac(ptr(x7), ptr(table), ptr(got["jacobian"]), 7 * n, L * F, 0, L, ctypes.byref(gd), ptr(jac), None,
                                       stream_ptr()), "nsr_hashgrid_forward_jac")
    got["taps"] = torch.empty_like(want)
    check(lib.nsr_hashgrid_forward_taps(ptr(x7), ptr(table), ptr(got["taps"]), n, L * F, 0, L, ctypes.byref(gd), None, stream_ptr()),
          "nsr_hashgrid_forward_taps")
    md = nsr_hip.NsrMlpDesc(L * F, 32, 16, 16, 1, 0)
    w = (torch.randn(64 * 32 + 16 * 64, generator=g) * 0.15).half().cuda()
    assert ops.grid_mlp_supported(gd, md)
    got["with network"] = ops.grid_mlp_forward(x7, table, w, gd, md, None, want_enc=True)[2]
    differ = {k: int((v != want).sum()) for k, v in got.items()}
    assert not any(differ.values()), differ

"""``nsr.optim.AdamW`` against its formula in 64 bits, and layer norm + clipping + AdamW as one training step.

Tolerances: u = 2^-24 is a rounding of fp32 (constants count one each).  m' = b1 m + c1 g: 3 roundings of either term; v': 4; the
root halves v's and adds its own; the update m / (r root + eps) * step adds 6 more; p (1 - lr wd) 2 and the difference 1.  A type
with spacing eps rounds by eps / 2.  8-bit codes: see _codes_match.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16, F8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
TOP, LEAST = 448.0, 2.0 ** -100


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _bits(seed, t, e):
    key = _mix(_mix(torch.tensor(t, dtype=torch.int64, device=e.device)) ^ seed)
    return _mix((e & 0xFFFFFFFF) ^ ((key + (e >> 32) * 0x9E3779B9) & 0xFFFFFFFF))


def _blocks(x, fill=0.0):
    n = x.numel()
    return torch.cat([x, x.new_full((-n % 256,), fill)]).view(-1, 256)


def _expected(p, g, m, v, t, lr, b1, b2, eps, wd, factor=1.0):
    """64-bit p', m', v' with their bounds (before the store's rounding)"""
    p, g, m, v = p.double(), g.double() * factor, m.double(), v.double()
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    tm = 6 * U * ((b1 * m).abs() + ((1 - b1) * g).abs()) + 1e-44
    tv = 8 * U * v1 + 1e-44
    r, root = v1.sqrt(), 1 / math.sqrt(1 - b2 ** t)
    step, denom = lr / (1 - b1 ** t), r * root + eps
    tr = 6 * U * r + (1e-44 / r.clamp_min(1e-30))
    upd = step * m1 / denom
    p1 = p * (1 - lr * wd) - upd
    tp = step * tm / denom + upd.abs() * (tr * root / denom + 8 * U) + 4 * U * p.abs() + 1e-44
    return p1, tp, m1, tm, v1, tv


def _store(v, dtype):
    return v.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _within(got, want, tol, what):
    off = (got.detach().double() - want).abs() - tol
    assert torch.isfinite(got.float()).all() and float(off.max()) <= 0.0, (what, float(off.max()))


def _codes_match(codes, scale, x, tx, u16, least):
    """codes / scales of the values x (64-bit, the kernel's off by at most tx) by the 64-bit rule.  tx is no fixed share of x:
    b1 m and c1 g may cancel.  With d = the block's largest tx / top, the largest magnitude is off by at most d top, the scale by
    d + 4 u (its product, 1 / 448, the store), and y = |x| 448 / top by 448 tx / top + y (d + 4 u)"""
    b = _blocks(x)
    top = b.abs().amax(1).clamp_min(LEAST)
    d = _blocks(tx).amax(1) / top
    assert bool(((scale.double() / (top / TOP) - 1).abs() <= d + 4 * U).all())
    y = (b.abs() / top[:, None] * TOP)
    ty = (_blocks(tx) / top[:, None] * TOP + y * (d + 4 * U)[:, None]).view(-1)[:x.numel()]
    y = y.view(-1)[:x.numel()]
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    at = y / step + (u16.double() + 0.5) / 65536
    want = (torch.floor(at) * step).clamp_max(TOP)
    want = torch.where(x != 0, want.clamp_min(least), torch.zeros_like(want))
    got = codes.float().double()
    # (2^-22 of a step: the bits of y under the 20 that the random ones are added to)
    sure = ((at - at.round()).abs() > ty / step + 2.0 ** -22) & (x.abs() > tx)
    assert torch.equal(got.abs()[sure], want[sure])
    assert bool(((got.abs() - want).abs() <= step * 1.001 + ty).all())  # elsewhere: a neighbour
    assert bool((got * x >= 0)[x.abs() > tx].all())
    nought = x == 0  # (no gradient yet: nothing to round)
    assert bool((got[nought] == 0).all())
    assert float((sure | nought).double().mean()) > 0.999 or x.numel() < 5000


SIZES = [[1], [255, 256, 257], [4096, 4097, 3, 1, 8191], [70001], [5] * 41, [1 << 20, 13]]


def _make(sizes, dtype, seed=0, **kw):
    import nsr.optim
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda n: torch.randn(n, generator=gen, device="cuda")  # noqa: E731
    ps = [torch.nn.Parameter((0.1 * new(n)).to(dtype)) for n in sizes]
    opt = nsr.optim.AdamW(ps, **kw)
    grads = lambda: [(new(n) * 10.0 ** (new(n).clamp(-3, 1) - 2)).masked_fill_(new(n) > 1.0, 0.0).to(dtype) for n in sizes]  # noqa: E731
    return ps, opt, grads


def _moments(opt, p):
    s = opt.state[p]
    if "scales" not in s:
        return s["exp_avg"].clone().view(-1), s["exp_avg_sq"].clone().view(-1)
    per = s["scales"].repeat_interleave(256, dim=1)[:, :p.numel()]
    return s["exp_avg"].float().view(-1) * per[0], (s["exp_avg_rms"].float().view(-1) * per[1]).square()


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_steps_match_the_formula(sizes, dtype, bits, clip):
    lr, betas, eps, wd = 0.01, (0.9, 0.99), 1e-15, 0.1
    ps, opt, grads = _make(sizes, dtype, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=bits, min_8bit_size=0,
                           max_grad_norm=clip, rounding_seed=12345)
    places = dict(zip(ps, opt._at))
    for t in range(1, 5):
        gs = grads()
        for p, g in zip(ps, gs):
            p.grad = g
        before = [(p.detach().clone(), *_moments(opt, p)) for p in ps]
        opt.step()
        factor = 1.0
        if clip:
            norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
            assert abs(float(opt.grad_norm) / norm - 1) < 2 * U
            factor = min(1.0, clip / (norm + 1e-6))
        for p, g, (p0, m0, v0) in zip(ps, gs, before):
            p1, tp, m1, tm, v1, tv = _expected(p0, g, m0, v0, t, lr, *betas, eps, wd, factor)
            _within(p, p1, tp + _store(p1, dtype), ("p", t))
            s = opt.state[p]
            if bits == 32:
                _within(s["exp_avg"], m1, tm, ("m", t))
                _within(s["exp_avg_sq"], v1, tv, ("v", t))
            else:
                e = places[p] + torch.arange(p.numel(), device="cuda")
                h = _bits(12345, t, e)
                _codes_match(s["exp_avg"], s["scales"][0], m1, tm, h >> 16, 0.0)
                # |sqrt(a) - sqrt(b)| is at most the root of |a - b|, and tv / (2 r) to first order where that is less
                tr = torch.minimum(tv.sqrt(), tv / v1.sqrt().clamp_min(1e-30)) + 2 * U * v1.sqrt()
                _codes_match(s["exp_avg_rms"], s["scales"][1], v1.sqrt(), tr, h & 0xFFFF, 2.0 ** -9)
                assert bool(((v1 > 0) <= (s["exp_avg_rms"].float() > 0)).all())
    assert opt.taken_steps() == 4


def test_32_bit_steps_follow_torch_and_state_dicts_are_exchanged():
    torch.manual_seed(0)
    shapes = [(64, 35), (64,), (1,), (13, 64), (300, 257)]
    ours, theirs = ([torch.nn.Parameter(torch.full(s, 0.1, device="cuda")) for s in shapes] for _ in range(2))
    import nsr.optim
    kw = dict(betas=(0.9, 0.99), eps=1e-15)
    groups = lambda ps: [dict(params=ps[:2], lr=0.01), dict(params=ps[2:], lr=0.002, weight_decay=0.1)]  # noqa: E731
    a, b = nsr.optim.AdamW(groups(ours), **kw), torch.optim.AdamW(groups(theirs), **kw)
    sched = [torch.optim.lr_scheduler.MultiStepLR(o, milestones=[3, 6], gamma=0.33) for o in (a, b)]

    def steps(n):
        for _ in range(n):
            for p, q in zip(ours, theirs):
                p.grad = torch.randn_like(p)
                q.grad = p.grad.clone()
            a.step(), b.step()
            [s.step() for s in sched]
        for p, q in zip(ours, theirs):
            assert torch.allclose(p, q, rtol=2e-5, atol=2e-6)

    steps(8)
    sd = a.state_dict()
    assert sd["state"][0]["step"].item() == 8 and sd["state"][3]["exp_avg"].shape == (13, 64)
    a2, b2 = nsr.optim.AdamW(groups(ours), **kw), torch.optim.AdamW(groups(theirs), **kw)
    a2.load_state_dict(b.state_dict())  # each continues from the other's state
    b2.load_state_dict(sd)
    assert a2.taken_steps() == 8 and a2.param_groups[1]["lr"] == a.param_groups[1]["lr"]
    a, b = a2, b2
    steps(3)


@pytest.mark.parametrize("clip", [None, 1.0])
def test_8_bit_state_dict_continues_with_the_same_bits(clip):
    sizes = [5000, 77, 20000]
    kw = dict(lr=0.01, state_bits=8, max_grad_norm=clip)
    ps, opt, grads = _make(sizes, F32, **kw)
    assert "scales" not in opt.state[ps[1]] and opt.state[ps[0]]["exp_avg"].dtype == F8  # 77 < min_8bit_size
    gs = [grads() for _ in range(6)]

    def go(ps, opt, gs):
        for g in gs:
            for p, q in zip(ps, g):
                p.grad = q
            opt.step()

    go(ps, opt, gs[:3])
    import io
    f = io.BytesIO()
    torch.save(opt.state_dict(), f)
    f.seek(0)
    saved = torch.load(f, weights_only=True)
    ps2, opt2, _ = _make(sizes, F32, **kw)
    for p, q in zip(ps2, ps):
        p.data.copy_(q.data)
    opt2.load_state_dict(saved)
    go(ps, opt, gs[3:])
    go(ps2, opt2, gs[3:])
    assert all(torch.equal(p, q) for p, q in zip(ps, ps2))
    assert all(torch.equal(opt.flat8[k].view(torch.uint8), opt2.flat8[k].view(torch.uint8)) for k in opt.flat8)
    with pytest.raises(ValueError):
        _make(sizes, F32, lr=0.01)[1].load_state_dict(saved)
    with pytest.raises(ValueError):
        _make([5000, 78, 20000], F32, **kw)[1].load_state_dict(saved)


def test_rounding_is_unbiased_and_moments_do_not_stick():
    """a constant gradient: m tends to g and r to |g|; round-to-nearest codes would stay where they are.  One code is off by at most
    a lattice step (1/8); means over n elements by 5 standard deviations of a uniform step, 5 / 8 / sqrt(12 n) each step, which the
    moments' own averaging never enlarges"""
    n = 1 << 16
    ps, opt, _ = _make([n], F32, lr=1e-4, betas=(0.9, 0.999), state_bits=8)
    g = torch.full((n,), 0.3, device="cuda")
    g[::256] = 1.0  # the blocks' largest value is another one
    ps[0].grad = g
    b1, b2 = 0.9, 0.999
    for t in range(1, 401):
        opt.step()
    m, v = _moments(opt, ps[0])
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[::256] = False
    want = (1 - b1 ** 400) * 0.3
    assert abs(float(m[rest].double().mean()) / want - 1) < 0.01
    # r is held and v = r^2: rounding r without bias adds its variance, at most (1/8)^2 / 4 of v between two codes
    ratio = float(v[rest].double().mean()) / ((1 - b2 ** 400) * 0.09)
    assert 0.99 < ratio < 1.10, ratio
    assert 0.5 < float((v[rest] / ((1 - b2 ** 400) * 0.09)).min()) and float((v[rest] / ((1 - b2 ** 400) * 0.09)).max()) < 2.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_at_odd_addresses_equal_aligned_ones(bits, dtype):
    """parameters and gradients as slices of one buffer at every alignment: the same bits as tensors of their own, and what lies
    between them stays"""
    import nsr.optim
    sizes = [8192, 5000, 1, 4096 * 3 + 1, 300]
    kw = dict(lr=0.01, state_bits=bits, min_8bit_size=0, max_grad_norm=1.0)
    ps, opt, grads = _make(sizes, dtype, **kw)
    flat_p, flat_g = (torch.full((sum(sizes) + 3 * len(sizes) + 1,), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    at, views, gviews, gaps = 1, [], [], torch.ones_like(flat_p, dtype=torch.bool)
    for p in ps:
        views.append(torch.nn.Parameter(flat_p[at:at + p.numel()]))
        views[-1].data.copy_(p.data)
        gviews.append(flat_g[at:at + p.numel()])
        gaps[at:at + p.numel()] = False
        at += p.numel() + 3
    opt2 = nsr.optim.AdamW(views, **kw)
    for _ in range(3):
        for p, v, gv, g in zip(ps, views, gviews, grads()):
            p.grad, v.grad = g, gv
            gv.copy_(g)
        opt.step(), opt2.step()
    assert all(torch.equal(p, v) for p, v in zip(ps, views))
    for k in ("flat32", "flat8"):
        a, b = getattr(opt, k), getattr(opt2, k)
        assert a.keys() == b.keys() and all(torch.equal(a[q].view(torch.uint8), b[q].view(torch.uint8)) for q in a)
    assert bool((flat_p[gaps] == 7).all()) and bool((flat_g[gaps] == 7).all())


def test_layouts_missing_gradients_and_empty_tensors():
    import nsr.optim
    torch.manual_seed(1)
    a = torch.nn.Parameter(torch.randn(40, 30, device="cuda").t())  # dense, columns first
    b = torch.nn.Parameter(torch.randn(7, device="cuda"))
    c = torch.nn.Parameter(torch.zeros(0, device="cuda"))
    d = torch.nn.Parameter(torch.randn(6, 1, 4, device="cuda"))
    ref = [torch.nn.Parameter(t.detach().clone().contiguous()) for t in (a, b, c, d)]
    ours = nsr.optim.AdamW([a, b, c, d], lr=0.01)
    theirs = torch.optim.AdamW(ref, lr=0.01)
    for step in range(3):
        for p, q in zip((a, b, c, d), ref):
            q.grad = torch.randn_like(q)
            p.grad = q.grad.clone() if step else q.grad.clone().as_strided(p.shape, p.stride()).copy_(q.grad)
        a.grad = ref[0].grad.clone().contiguous()  # strides other than the parameter's
        ours.step(), theirs.step()
    for p, q in zip((a, b, d), (ref[0], ref[1], ref[3])):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)
    assert torch.allclose(ours.state[a]["exp_avg"], theirs.state[ref[0]]["exp_avg"], rtol=1e-5, atol=1e-7)
    keep = b.detach().clone(), ours.state[b]["exp_avg"].clone()
    a.grad, b.grad, c.grad = torch.ones_like(a), None, None
    version = a._version
    ours.step()
    assert torch.equal(b, keep[0]) and torch.equal(ours.state[b]["exp_avg"], keep[1]) and a._version > version
    ours.zero_grad(set_to_none=True)
    before = a.detach().clone()
    ours.step()
    assert torch.equal(a, before) and ours.taken_steps() == 4  # no gradient at all: no step


@pytest.mark.parametrize("bits", [32, 8])
def test_elements_and_steps_that_are_left_out(bits):
    sizes = [5000, 300]
    kw = dict(lr=0.01, state_bits=bits, min_8bit_size=0)
    # without clipping: an element with a non-finite gradient keeps its value and moments
    ps, opt, grads = _make(sizes, F32, **kw)
    for _ in range(2):
        for p, g in zip(ps, grads()):
            p.grad = g
        opt.step()
    before = [(p.detach().clone(), *_moments(opt, p)) for p in ps]
    gs = grads()
    gs[0][7], gs[0][4999], gs[1][0] = float("nan"), float("inf"), -float("inf")
    for p, g in zip(ps, gs):
        p.grad = g
    opt.step()
    for p, g, (p0, m0, v0) in zip(ps, gs, before):
        bad = ~torch.isfinite(g)
        assert torch.equal(p[bad], p0[bad]) and torch.isfinite(p).all() and not torch.equal(p, p0)
        m, v = _moments(opt, p)
        if bits == 32:
            assert torch.equal(m[bad], m0[bad]) and torch.equal(v[bad], v0[bad])
        assert torch.isfinite(m).all() and torch.isfinite(v).all()
    # with clipping: the whole step stays out and does not count
    ps, opt, grads = _make(sizes, F32, max_grad_norm=1.0, **kw)
    for p, g in zip(ps, grads()):
        p.grad = g
    opt.step()
    before = [p.detach().clone() for p in ps]
    flat = {k: t.clone().view(torch.uint8) for k, t in {**opt.flat32, **opt.flat8}.items()}
    ps[1].grad[5] = float("nan")
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, before)) and opt.taken_steps() == 1
    assert all(torch.equal(t.view(torch.uint8), flat[k]) for k, t in {**opt.flat32, **opt.flat8}.items())
    assert not math.isfinite(float(opt.grad_norm))
    ps[1].grad[5] = 3e38  # squares past fp32: the norm is finite in 64 bits, the step is taken
    opt.step()
    assert opt.taken_steps() == 2 and abs(float(opt.grad_norm) / 3e38 - 1) < 1e-6 and torch.isfinite(ps[1]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_very_small_and_very_large_gradients(bits):
    ps, opt, _ = _make([1024], F32, lr=0.01, betas=(0.9, 0.99), eps=1e-15, state_bits=bits, min_8bit_size=0)
    g = torch.zeros(1024, device="cuda")
    g[:256] = 3e38      # the squares overflow: no update can blow up, the state stays finite in 8 bits
    g[256:512] = 1e-30  # squares under fp32: m / eps
    g[512] = 1.0        # one element far over the rest of its block
    g[513:768] = 1e-7
    ps[0].grad = g
    p0 = ps[0].detach().clone()
    for _ in range(20):
        opt.step()
    assert torch.isfinite(ps[0]).all() and float((ps[0].detach() - p0).abs().max()) < 20 * 0.01 * 4
    assert torch.equal(ps[0][768:], p0[768:] * 1.0) or float((ps[0][768:] / p0[768:] - (1 - 1e-4) ** 20).abs().max()) < 1e-5
    if bits == 8:
        m, v = _moments(opt, ps[0])
        assert torch.isfinite(m).all() and torch.isfinite(v).all() and bool((v[513:768] > 0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_capture_replays_with_a_learning_rate_on_the_device(bits):
    sizes = [9000, 257] + [33] * 40  # two launches
    kw = dict(betas=(0.9, 0.99), state_bits=bits, max_grad_norm=2.0, capturable=True)
    lrs = [torch.tensor(0.01, device="cuda") for _ in range(2)]
    pair = [_make(sizes, F32, lr=lr, **kw) for lr in lrs]
    (ps, opt, grads), (qs, ref, _) = pair
    static = [torch.zeros_like(p) for p in ps]
    for p, g in zip(ps, static):
        p.grad = g
    gs = [grads() for _ in range(6)]
    for g, s in zip(gs[0], static):
        s.copy_(g)
    opt.step()  # (a first step outside)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for q, g in zip(qs, gs[0]):
        q.grad = g
    ref.step()
    for k in range(1, 6):
        for g, s in zip(gs[k], static):
            s.copy_(g)
        for lr in lrs:
            lr.fill_(0.01 / k)
        graph.replay()
        for q, g in zip(qs, gs[k]):
            q.grad = g
        ref.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k
        assert float(opt.grad_norm) == float(ref.grad_norm)
    assert opt.taken_steps() == 6
    plain = _make([64], F32, lr=0.01)[1]
    plain.param_groups[0]["params"][0].grad = torch.zeros(64, device="cuda")
    from nsr_hip import NsrError
    other = torch.cuda.CUDAGraph()
    with pytest.raises(NsrError):
        with torch.cuda.graph(other):
            plain.step()


def test_two_optimizers_on_two_streams():
    """no state is shared: two optimizers interleaved on two streams give what each gives alone"""
    sizes = [30000, 555]
    runs = []
    gs = [[torch.randn(n, device="cuda") for n in sizes] for _ in range(5)]
    torch.cuda.synchronize()
    for mode in ("alone", "interleaved"):
        pair = [_make(sizes, F32, seed=k, lr=0.01, state_bits=8, max_grad_norm=1.0 + k) for k in range(2)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        order = [(k, i) for k in range(2) for i in range(5)] if mode == "alone" else [(k, i) for i in range(5) for k in range(2)]
        for k, i in order:
            ps, opt, _ = pair[k]
            with torch.cuda.stream(streams[k]):
                for p, g in zip(ps, gs[i]):
                    p.grad = g
                opt.step()
        torch.cuda.synchronize()
        runs.append([p.detach().clone() for ps, *_ in pair for p in ps])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("unscale_first", [False, True])
def test_grad_scaler_skips_and_unscales(unscale_first):
    import nsr.optim
    torch.manual_seed(2)
    p, q = (torch.nn.Parameter(torch.ones(1000, device="cuda")) for _ in range(2))
    ours, theirs = nsr.optim.AdamW([p], lr=0.01), torch.optim.AdamW([q], lr=0.01)
    scalers = [torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=2) for _ in range(2)]
    for step in range(6):
        g = torch.randn(1000, device="cuda")
        if step == 2:
            g[3] = float("inf")
        for par, opt, sc in ((p, ours, scalers[0]), (q, theirs, scalers[1])):
            opt.zero_grad()
            sc.scale((par * g).sum()).backward()
            if unscale_first:
                sc.unscale_(opt)
            sc.step(opt)
            sc.update()
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6), step
        assert scalers[0].get_scale() == scalers[1].get_scale()
    assert ours.taken_steps() == 5 and not hasattr(ours, "found_inf")


def test_tinycudann_modules_get_their_image():
    import nsr.optim
    import tinycudann as tcnn
    from conftest import COLOR_MLP, DENSITY_MLP
    enc = dict(otype="HashGrid", n_levels=4, n_features_per_level=2, log2_hashmap_size=12, base_resolution=4, per_level_scale=2.0)
    torch.manual_seed(3)
    ewn = tcnn.NetworkWithInputEncoding(3, 16, enc, DENSITY_MLP).cuda()
    net = tcnn.Network(16, 3, COLOR_MLP).cuda()
    head = torch.nn.Linear(3, 1).cuda()
    params = [m.params for m in (ewn, net)] + list(head.parameters())
    opt = nsr.optim.AdamW(params, lr=0.01, betas=(0.9, 0.99), eps=1e-15, state_bits=8, max_grad_norm=1.0, modules=[ewn, net])
    x = torch.rand(512, 3, device="cuda")
    for _ in range(3):
        opt.zero_grad()
        head(net(ewn(x).float()).float()).square().mean().backward()
        opt.step()
        for m in (ewn, net):
            assert torch.equal(m.half_params(m.params), m.params.detach().half()) and m._shadow_trusted
    with torch.no_grad():  # written from outside: the next step starts from a fresh image, also where it is left out
        net.params.add_(0.25)
    opt.zero_grad()
    head(net(ewn(x).float()).float()).square().mean().backward()
    head.weight.grad[0, 0] = float("nan")
    opt.step()
    assert torch.equal(net.half_params(net.params), net.params.detach().half())


def test_training_step_of_a_normalised_network():
    """layer norm's gradients into the clip and the update, as a user runs them, against the same network in float64 with torch's
    AdamW.  Three steps; Adam's update is at most lr in size, an error delta of a gradient moves it by lr delta / |g|: elements
    whose gradient is under 1e-3 of the largest are not compared (fp32 gradients are good to about 1e-6 of the largest)"""
    import nsr.optim
    from nsr.layers import LayerNorm
    torch.manual_seed(4)
    x, target = torch.randn(777, 35, device="cuda"), torch.randn(777, 3, device="cuda")
    net = torch.nn.Sequential(torch.nn.Linear(35, 64), LayerNorm(64), torch.nn.ReLU(), torch.nn.Linear(64, 65), LayerNorm(65),
                              torch.nn.ReLU(), torch.nn.Linear(65, 3)).cuda()
    ref = torch.nn.Sequential(torch.nn.Linear(35, 64), torch.nn.LayerNorm(64), torch.nn.ReLU(), torch.nn.Linear(64, 65),
                              torch.nn.LayerNorm(65), torch.nn.ReLU(), torch.nn.Linear(65, 3)).double().cuda()
    ref.load_state_dict({k: v.double() for k, v in net.state_dict().items()})
    kw = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8)
    ours, theirs = nsr.optim.AdamW(net.parameters(), max_grad_norm=0.1, **kw), torch.optim.AdamW(ref.parameters(), **kw)
    seen = [torch.full_like(p, float("inf"), dtype=torch.float64) for p in ref.parameters()]
    for _ in range(3):
        ours.zero_grad(), theirs.zero_grad()
        (net(x) - target).square().mean().backward()
        (ref(x.double()) - target.double()).square().mean().backward()
        for p, q in zip(net.parameters(), ref.parameters()):
            assert float((p.grad - q.grad).abs().max()) < 2e-5 * max(1e-3, float(q.grad.abs().max()))
        norm = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.1)
        seen = [torch.minimum(s, q.grad.abs() / q.grad.abs().max()) for s, q in zip(seen, ref.parameters())]
        ours.step(), theirs.step()
        assert abs(float(ours.grad_norm) / float(norm) - 1) < 1e-5 and float(norm) > 0.1
    for p, q, s in zip(net.parameters(), ref.parameters(), seen):
        big = s > 1e-2
        assert float((p - q)[big].abs().max()) < 3e-3 * 0.05


def test_offsets_past_32_bits():
    """2^32 + 4099 bf16 elements, 8-bit moments: the last elements and those around 2^32 move as the formula says"""
    import nsr.optim
    n = (1 << 32) + 4099
    p = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    p.grad = torch.zeros(n, dtype=BF16, device="cuda")
    opt = nsr.optim.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, max_grad_norm=1e9, rounding_seed=9)
    where = torch.cat([torch.arange(3), torch.arange((1 << 32) - 2, (1 << 32) + 300), torch.arange(n - 5, n)]).cuda()
    g = torch.linspace(0.5, 2.0, where.numel(), device="cuda").to(BF16)
    p.grad[where] = g
    opt.step()
    assert torch.equal(p[where], torch.full_like(g, -0.5)) and int(torch.count_nonzero(p)) == where.numel()
    assert abs(float(opt.grad_norm) / math.sqrt(float(g.double().square().sum())) - 1) < 2 * U
    s = opt.state[p]
    m = torch.zeros(256 * 20, dtype=torch.float64, device="cuda")
    b0 = (1 << 32)
    m[:300], m[4094:4096] = 0.1 * g[5:305].double(), 0.1 * g[305:307].double()  # (2 of the last 5 lie in the window)
    e = b0 + torch.arange(4096, device="cuda")
    _codes_match(s["exp_avg"][b0:b0 + 4096], s["scales"][0, b0 // 256:b0 // 256 + 16], m[:4096], 6 * U * m[:4096].abs(), _bits(9, 1, e) >> 16, 0.0)


def test_refusals_on_the_gpu():
    import nsr.optim
    from nsr_hip import NsrError
    new = lambda *s, **k: torch.nn.Parameter(torch.zeros(*s, device="cuda", **k))  # noqa: E731
    flat = torch.zeros(100, device="cuda")
    for bad in (lambda: nsr.optim.AdamW([new(4, dtype=torch.float64)]),
                lambda: nsr.optim.AdamW([torch.nn.Parameter(torch.zeros(4, 8, device="cuda")[:, ::2])]),
                lambda: nsr.optim.AdamW([torch.nn.Parameter(flat[:60]), torch.nn.Parameter(flat[50:])]),
                lambda: nsr.optim.AdamW([dict(params=[new(4)]), dict(params=[new(4)], betas=(0.5, 0.9))]),
                lambda: nsr.optim.AdamW([new(4)], lr=-1.0), lambda: nsr.optim.AdamW([new(4)], betas=(0.9, 1.0)),
                lambda: nsr.optim.AdamW([new(4)], lr=torch.tensor(0.1), capturable=True),
                lambda: nsr.optim.AdamW([new(4)]).add_param_group(dict(params=[new(4)])),
                lambda: nsr.optim.AdamW([new(4)], modules=[type("M", (), dict(params=new(4)))()])):
        with pytest.raises((NsrError, ValueError, NotImplementedError)):
            bad()
    p = new(6)
    opt = nsr.optim.AdamW([p], lr=0.1)
    p.grad = torch.ones(6, device="cuda")
    p.data = torch.zeros(7, device="cuda")
    with pytest.raises(NsrError):
        opt.step()


def test_replaced_gradients_are_refused_and_copies_too():
    import copy
    import nsr.optim
    from nsr_hip import NsrError
    ps, opt, grads = _make([600, 33], F32, lr=0.01)
    for p, g in zip(ps, grads()):
        p.grad = g
    ps[0].grad.data = torch.zeros(599, device="cuda")  # (torch checks ``p.grad = g``, not this)
    before = [p.detach().clone() for p in ps]
    with pytest.raises(NsrError):
        opt.step()
    ps[1].grad = None
    with pytest.raises(NsrError):
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, before)) and opt.taken_steps() == 0
    ps[1].grad, ps[0].grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1), (33,)).cuda(), None
    with pytest.raises((NsrError, RuntimeError)):
        opt.step()
    with pytest.raises(NotImplementedError):
        copy.deepcopy(opt)
    q = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    theirs = torch.optim.AdamW([q], amsgrad=True)
    with pytest.raises(NotImplementedError):
        nsr.optim.AdamW([torch.nn.Parameter(torch.zeros(5, device="cuda"))]).load_state_dict(theirs.state_dict())


def test_closure_hooks_and_a_rate_that_keeps_its_place():
    import nsr.optim
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    lr = torch.tensor(0.5, device="cuda")
    opt = nsr.optim.AdamW([p], lr=lr, weight_decay=0.0, capturable=True)
    seen = []
    opt.register_step_pre_hook(lambda *a: seen.append("before"))
    opt.register_step_post_hook(lambda *a: seen.append("after"))

    def closure():
        opt.zero_grad()
        loss = (p * 2).sum()
        loss.backward()
        return loss

    assert float(opt.step(closure)) == 600.0 and seen == ["before", "after"]
    assert torch.allclose(p, torch.full_like(p, 0.5), atol=1e-6)
    sd = opt.state_dict()
    sd["param_groups"][0]["lr"] = torch.tensor(0.25)
    opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.25 and opt.taken_steps() == 1


def test_pieces_of_one_tensor():
    """2^33 + 4099 elements are two pieces of one launch each: those around the cut and the last ones move like the others"""
    import nsr.optim
    n = (1 << 33) + 4099
    p = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    p.grad = torch.zeros(n, dtype=BF16, device="cuda")
    opt = nsr.optim.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, rounding_seed=9)
    cut = 1 << 33
    where = torch.cat([torch.arange(3), torch.arange(cut - 300, cut + 300), torch.arange(n - 5, n)]).cuda()
    g = torch.linspace(0.5, 2.0, where.numel(), device="cuda").to(BF16)
    p.grad[where] = g
    opt.step()
    assert torch.equal(p[where], torch.full_like(g, -0.5))
    assert sum(int(torch.count_nonzero(part)) for part in p.detach().split(1 << 31)) == where.numel()
    s = opt.state[p]
    m = torch.zeros(1024, dtype=torch.float64, device="cuda")
    m[212:812] = 0.1 * g[3:603].double()  # elements cut - 512 .. cut + 511
    e = cut - 512 + torch.arange(1024, device="cuda")
    b0 = (cut - 512) // 256
    _codes_match(s["exp_avg"][cut - 512:cut + 512], s["scales"][0, b0:b0 + 4], m, 6 * U * m.abs(), _bits(9, 1, e) >> 16, 0.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(bits):
    """300 tensors: several launches of the update (64, 36) and of the norm (128), against the formula"""
    lr, betas, eps, wd = 0.01, (0.9, 0.99), 1e-15, 0.1
    sizes = [37 + k for k in range(299)] + [9000]
    ps, opt, grads = _make(sizes, F32, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=bits, min_8bit_size=0,
                           max_grad_norm=0.5)
    for t in (1, 2):
        gs = grads()
        for p, g in zip(ps, gs):
            p.grad = g
        before = [(p.detach().clone(), *_moments(opt, p)) for p in ps]
        opt.step()
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
        assert abs(float(opt.grad_norm) / norm - 1) < 2 * U
        for p, g, (p0, m0, v0) in zip(ps, gs, before):
            p1, tp, *_ = _expected(p0, g, m0, v0, t, lr, *betas, eps, wd, min(1.0, 0.5 / (norm + 1e-6)))
            _within(p, p1, tp + _store(p1, F32), ("p", t))

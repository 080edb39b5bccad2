"""State of ``nsr.optim.AdamW``: what it exchanges with torch's, what may change after construction, images beside replayed steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_state_of_16_bit_parameters_is_exchanged_with_torch(dtype):
    """torch keeps the moments in the parameter's type: taken in as they are (every 16-bit value is one of float32), given back they
    are rounded by torch"""
    import nsr.optim
    shapes = [(300, 7), (5,), (64,)]
    g = torch.Generator(device="cuda").manual_seed(2)
    new = lambda s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    ps = [[torch.nn.Parameter(new(s)) for s in shapes] for _ in range(2)]
    kw = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-3)
    theirs, ours = torch.optim.AdamW(ps[0], **kw), nsr.optim.AdamW(ps[1], **kw)
    for _ in range(3):
        for p in ps[0]:
            p.grad = new(p.shape)
        theirs.step()
    ours.load_state_dict(theirs.state_dict())
    assert ours.taken_steps() == 3
    for p, q in zip(*ps):
        for k in ("exp_avg", "exp_avg_sq"):
            assert ours.state[q][k].dtype == F32 and torch.equal(ours.state[q][k], theirs.state[p][k].float())
    for q in ps[1]:
        q.grad = new(q.shape)
    ours.step()
    theirs.load_state_dict(ours.state_dict())
    for p, q in zip(*ps):
        s = theirs.state[p]
        assert s["step"].item() == 4 and all(torch.equal(s[k], ours.state[q][k].to(s[k].dtype)) for k in ("exp_avg", "exp_avg_sq"))
    for p in ps[0]:
        p.grad = new(p.shape)
    theirs.step()
    # what is no floating-point moment is refused still, and 8-bit codes take nothing but codes
    sd = ours.state_dict()
    sd["state"][0]["exp_avg"] = sd["state"][0]["exp_avg"].int()
    with pytest.raises(ValueError):
        ours.load_state_dict(sd)
    eight = nsr.optim.AdamW(ps[1], state_bits=8, min_8bit_size=0, **kw)
    with pytest.raises(ValueError):
        eight.load_state_dict(theirs.state_dict())


def _pair(n, seed=5):
    import nsr.optim
    g = torch.Generator(device="cuda").manual_seed(seed)
    p0 = torch.randn(n, generator=g, device="cuda")
    gs = [torch.randn(n, generator=g, device="cuda") for _ in range(6)]
    kw = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-8)
    return lambda **more: (lambda p: (p, nsr.optim.AdamW([p], **kw, **more)))(torch.nn.Parameter(p0.clone())), gs


def test_clipping_switched_on_and_off_after_construction():
    """the same bits as steps of optimizers built with each setting that hand their state on; a norm that is no norm is refused"""
    new, gs = _pair(3000)
    (p, opt), (q, plain), (r, clipped) = new(), new(), new(max_grad_norm=0.5)
    assert opt.max_grad_norm is None and opt.grad_norm is None

    def go(param, optimizer, g):
        param.grad = g
        optimizer.step()

    def hand_on(a, b, of, to):
        with torch.no_grad():
            b.copy_(a)
        to.load_state_dict(of.state_dict())

    for g in gs[:2]:
        go(p, opt, g), go(q, plain, g)
    opt.max_grad_norm = 0.5
    hand_on(q, r, plain, clipped)
    for g in gs[2:4]:
        go(p, opt, g), go(r, clipped, g)
        assert torch.equal(opt.grad_norm, clipped.grad_norm) and abs(float(opt.grad_norm) / float(g.double().norm()) - 1) < 1e-6
    assert torch.equal(p, r) and opt.taken_steps() == 4
    opt.max_grad_norm = None
    hand_on(r, q, clipped, plain)
    for g in gs[4:]:
        go(p, opt, g), go(q, plain, g)
    # (the unclipped device-side step works 1 / (1 - b^t) out on the device, in 64 bits as on the host, rounded to fp32 once)
    assert opt.grad_norm is None and opt.taken_steps() == 6 and torch.allclose(p, q, rtol=1e-6, atol=1e-8)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            opt.max_grad_norm = bad
    assert opt.max_grad_norm is None
    for name in ("state_bits", "min_8bit_size"):
        with pytest.raises(AttributeError):
            setattr(opt, name, 8)


def test_capture_switched_on_after_construction():
    """the count moves to the device: replays go on counting from where the eager steps stopped"""
    new, gs = _pair(3000)
    (p, opt), (q, ref) = new(), new(capturable=True)
    held = torch.zeros_like(gs[0])
    for g in gs[:2]:
        p.grad = q.grad = g
        opt.step(), ref.step()
    opt.capturable = True
    p.grad = held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for g in gs[2:]:
        held.copy_(g)
        graph.replay()
        q.grad = g
        ref.step()
        torch.cuda.synchronize()
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-8)
    assert opt.taken_steps() == ref.taken_steps() == 6


@pytest.mark.parametrize("size", [1024, 700])
def test_8_bit_moments_beside_a_gradient_that_is_not_finite(size):
    """the parameter stays; the moments are those of before, rounded once more: within one lattice step of the block's new scale
    (steps of e4m3 value y: 2^(max(floor(log2 y), -6) - 3); a code may be rounded up to the next power's), signs kept, and
    positive roots above zero"""
    import nsr.optim
    g = torch.Generator(device="cuda").manual_seed(8)
    p = torch.nn.Parameter(torch.randn(size, generator=g, device="cuda"))
    opt = nsr.optim.AdamW([p], lr=0.01, state_bits=8, min_8bit_size=0)
    for _ in range(3):
        p.grad = torch.randn(size, generator=g, device="cuda")
        opt.step()

    def moments():
        s = opt.state[p]
        per = s["scales"].double().repeat_interleave(256, dim=1)[:, :size]
        return [s[k].double() * sc for k, sc in zip(("exp_avg", "exp_avg_rms"), per)], per

    bad = torch.tensor([0, 5, 255, 300, 511, 600, size - 1], device="cuda")
    for scale in (1.0, 100.0, 0.0):  # the blocks' scales stay about as they are, grow, shrink
        before, _ = moments()
        p0 = p.detach().clone()
        p.grad = scale * torch.randn(size, generator=g, device="cuda")
        p.grad[bad] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").repeat(3)[:bad.numel()]
        opt.step()
        assert torch.equal(p[bad], p0[bad])
        after, per = moments()
        for a, b, sc in zip(after, before, per):
            a, b, sc = a[bad], b[bad], sc[bad]
            y = (b / sc).abs().clamp_min(2.0 ** -9)
            step = torch.exp2(torch.floor(torch.log2(y)).clamp_min(-6) - 3) * sc
            assert bool(((a - b).abs() <= step * (1 + 2.0 ** -20)).all()) and bool((a * b >= 0).all())
        assert bool((after[1][bad] > 0).all())


def _module_and_graph(seed=3):
    """a network whose optimizer's step is captured, its gradients in a buffer of their own"""
    import nsr.optim
    import tinycudann as tcnn
    from conftest import COLOR_MLP
    torch.manual_seed(seed)
    net = tcnn.Network(16, 3, COLOR_MLP).cuda()
    opt = nsr.optim.AdamW([net.params], lr=0.05, capturable=True, modules=[net])
    net.params.grad = torch.randn_like(net.params)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    return net, opt, graph


def test_replayed_steps_and_parameters_written_from_outside():
    """a replay bumps no version counter: a cast that evaluation mode made after a write from outside is not taken for the
    parameters that a replay has changed since"""
    net, opt, graph = _module_and_graph()
    image = lambda: net.half_params(net.params)  # noqa: E731
    now = lambda: net.params.detach().half()  # noqa: E731
    for mode in (net.train, net.eval):
        mode()
        graph.replay()
        assert torch.equal(image(), now())
    with torch.no_grad():
        net.params.add_(0.25)
    for mode in (net.eval, net.train, net.eval):
        mode()
        assert torch.equal(image(), now())
        graph.replay()
        assert torch.equal(image(), now())
    opt.step()  # an eager step puts the image right
    graph.replay()
    assert torch.equal(image(), now()) and net._shadow_trusted


def test_captured_forward_reads_the_refreshed_image():
    net, opt, graph = _module_and_graph()
    x = torch.rand(256, 16, device="cuda")
    with torch.no_grad():
        net(x)
        forward = torch.cuda.CUDAGraph()
        with torch.cuda.graph(forward):
            y = net(x)
        for k in range(3):
            graph.replay()
            forward.replay()
            assert torch.equal(y, net(x))
            net.params.mul_(0.5 + k)
            opt.refresh_images()
            forward.replay()
            assert torch.equal(y, net(x)) and torch.equal(net.half_params(net.params), net.params.half())


def test_state_dict_hooks_see_the_whole_state():
    """as in torch: a hook behind state_dict sees the steps and may change them, one in front of load_state_dict gets and may replace
    the moments, one behind it sees them loaded"""
    new, gs = _pair(300)
    (p, opt), (q, other) = new(), new()
    p.grad = gs[0]
    opt.step()
    seen = []
    opt.register_state_dict_post_hook(lambda o, sd: seen.append(sd["state"][0]["step"].item()))
    sd = opt.state_dict()
    assert seen == [1.0] and set(opt.state[p]) == {"exp_avg", "exp_avg_sq"} and list(sd["state"][0])[0] == "step"

    def double(o, sd):
        state = {0: {**sd["state"][0], "exp_avg": 2 * sd["state"][0]["exp_avg"]}}
        return {**sd, "state": state}

    first = other.register_load_state_dict_pre_hook(double)
    second = other.register_load_state_dict_post_hook(lambda o: seen.append((o.state[q]["exp_avg"].clone(), o.taken_steps())))
    other.load_state_dict(sd)
    assert torch.equal(seen[1][0], 2 * opt.state[p]["exp_avg"]) and seen[1][1] == 1
    assert torch.equal(other.state[q]["exp_avg_sq"], opt.state[p]["exp_avg_sq"])
    first.remove(), second.remove()
    other.load_state_dict(sd)
    assert torch.equal(other.state[q]["exp_avg"], opt.state[p]["exp_avg"]) and len(seen) == 2


def test_two_modules_of_one_parameter():
    """the pass writes one image a parameter: both modules read it, in every step"""
    import nsr.optim
    import tinycudann as tcnn
    from conftest import COLOR_MLP
    torch.manual_seed(4)
    a, b = (tcnn.Network(16, 3, COLOR_MLP).cuda() for _ in range(2))
    b.params = a.params
    opt = nsr.optim.AdamW([a.params], lr=0.05, modules=[a, b])
    for _ in range(4):
        a.params.grad = torch.randn_like(a.params)
        opt.step()
        for m in (a, b):
            assert m._shadow_trusted and torch.equal(m.half_params(m.params), a.params.detach().half())


def test_a_module_with_another_parameter_is_refused():
    """an image of the optimizer's parameter is not handed to a module that holds another one meanwhile"""
    import nsr.optim
    import tinycudann as tcnn
    from conftest import COLOR_MLP
    from nsr_hip import NsrError
    net = tcnn.Network(16, 3, COLOR_MLP).cuda()
    p = net.params
    opt = nsr.optim.AdamW([p], lr=0.05, modules=[net])
    p.grad = torch.ones_like(p)
    opt.step()
    before = p.detach().clone()
    net.params = torch.nn.Parameter(torch.randn_like(p))
    for call in (opt.step, opt.refresh_images):
        with pytest.raises(NsrError, match="another `params`"):
            call()
    assert torch.equal(p, before) and opt.taken_steps() == 1
    assert torch.equal(net.half_params(net.params), net.params.detach().half())


@pytest.mark.parametrize("capturable", [False, True])
def test_step_counts_that_are_none(capturable):
    """a step number of 0 or less would divide by 1 - beta^0"""
    new, gs = _pair(300)
    p, opt = new(capturable=capturable)
    for bad in (-1, -5, 1 << 31):
        with pytest.raises(ValueError):
            opt.set_step(bad)
    opt.set_step(0)
    p.grad = gs[0]
    opt.step()
    assert opt.taken_steps() == 1 and torch.isfinite(p).all()


def test_a_refused_captured_step_leaves_the_step_count_alone():
    """with a GradScaler's scalars: the refusal comes before the step count would be made inside the capture"""
    from nsr_hip import NsrError
    new, gs = _pair(300)
    (p, opt), (q, ref) = new(), new()
    for o in (opt, ref):
        o.found_inf, o.grad_scale = torch.zeros(1, device="cuda"), torch.full((1,), 2.0, device="cuda")
    p.grad = q.grad = gs[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(NsrError):
        with torch.cuda.graph(graph):
            opt.step()
    assert opt.taken_steps() == 0
    for o in (opt, ref):
        o.step()
    assert torch.equal(p, q) and opt.taken_steps() == ref.taken_steps() == 1

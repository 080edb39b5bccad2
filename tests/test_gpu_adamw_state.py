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

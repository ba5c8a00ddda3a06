"""What GlobalHeads keeps from forward to backward is its own."""
import pytest

import slime_amd
from slime_amd import GlobalHeads, Pseudopod

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

CHANGES = {
    "output": lambda y, alive, heads: y.add_(1.0),
    "output by another call": lambda y, alive, heads: heads.ca.forward(y.clone(), out=y),
    "mask": lambda y, alive, heads: alive.logical_not_(),
    "gains": lambda y, alive, heads: (heads.wq.mul_(0.5), heads.wk.add_(1.0)),
    "gains replaced": lambda y, alive, heads: [setattr(heads, n, getattr(heads, n) * 2) for n in ("wq", "wk")],
}


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("what", CHANGES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_changes_between_forward_and_backward(dtype, what):
    """The gradients are the forward's, bit by bit, whatever became of what the caller holds."""
    cfg = slime_amd.CAConfig("heads", B=2, G=16, H=8, D=16, dtype=dtype, steps=1, w_std=0.1)
    with Pseudopod(cfg.B, cfg.G, cfg.H, cfg.D, cfg.dtype, cfg.dt) as ca:
        ca.set_params(slime_amd.make_params(cfg, seed=1))
        x = torch.from_numpy(slime_amd.make_state(cfg, seed=2)).cuda().to(ca.torch_dtype)
        g = torch.Generator(device="cuda").manual_seed(3)
        grad = torch.randn(ca.state_shape, generator=g, device="cuda").to(ca.torch_dtype)
        alive = torch.rand(ca.state_shape[:3], generator=g, device="cuda") < 0.7
        heads = GlobalHeads(ca)
        heads.wq += 0.2 * torch.randn(cfg.D, generator=g, device="cuda")
        heads.forward(x, alive)
        want = [t.clone() for t in (*heads.backward(grad), heads.dwq, heads.dwk)]
        # P's and I's gradients, and so the gains', pass through out
        assert all(bool(t.any()) for t in want)
        y = heads.forward(x, alive)
        CHANGES[what](y, alive, heads)
        got = (*heads.backward(grad), heads.dwq, heads.dwk)
        for a, b, name in zip(got, want, ("dP", "dI", "dV", "dwq", "dwk")):
            assert torch.equal(a, b), name


@pytest.mark.parametrize("fails", ["qk_norm_rotate", "attend"])
def test_a_history_step_that_raises_adds_no_state(monkeypatch, fails):
    """The next step is as if the one that raised had not been made."""
    from slime_amd import CellHistory, global_heads
    cfg = slime_amd.CAConfig("heads", B=1, G=16, H=8, D=16, dtype="bf16", steps=1, w_std=0.1)
    with Pseudopod(cfg.B, cfg.G, cfg.H, cfg.D, cfg.dtype, cfg.dt) as ca:
        ca.set_params(slime_amd.make_params(cfg, seed=1))
        x = torch.from_numpy(slime_amd.make_state(cfg, seed=2)).cuda().to(ca.torch_dtype)
        states = [x, ca.forward(x)]
        plain, past = CellHistory(ca, capacity=2), CellHistory(ca, capacity=2)
        want = [plain.step(s) for s in states]
        for s, y in zip(states, want):
            with monkeypatch.context() as m:
                def refuse(*_, **__):
                    raise slime_amd.SlimeError(-1, "no")
                m.setattr(global_heads, fails, refuse)
                with pytest.raises(slime_amd.SlimeError):
                    past.step(x + 1)
            assert torch.equal(past.step(s), y)
        assert past.length == 2

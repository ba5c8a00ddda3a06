"""Global heads on the projections of a ``Pseudopod``: the attention operators as they are used
together.

``GlobalHeads`` lets every cell of a grid attend to every other (or to the living ones), and gives
the gradients of the projections and of the gains. ``CellHistory`` lets each cell attend to its own
earlier states: one new state at a time over a cache of normed keys and values.

    ca = Pseudopod(B=4, G=64, H=8, D=64, dtype="bf16")
    ca.set_params(make_params(cfg))
    heads = GlobalHeads(ca)
    y = heads.forward(x)                              # [B, G, G, C], as a state
    dP, dI, dV = heads.backward(grad_y)               # and heads.dwq, heads.dwk

    past = CellHistory(ca, capacity=64)
    for x in states:
        y = past.step(x)

``python -m slime_amd.global_heads`` trains the gains of a small grid's heads on a fixed target and
prints the loss, then steps a history and compares it with one attention over all of it.
"""
from __future__ import annotations

import math

from .attention import attend, attend_backward, qk_norm_rotate, qk_norm_rotate_backward, rotation_freqs
from .ca import Pseudopod, _torch


class GlobalHeads:
    """Attention of cells to all cells of their grid, placed by row and column."""

    def __init__(self, ca: Pseudopod, base: float = 10000.0, eps: float = 1e-6):
        torch = _torch()
        self.ca, self.eps = ca, eps
        self.wq, self.wk = (torch.ones(ca.D, device="cuda") for _ in range(2))
        self.freqs = rotation_freqs(ca.D, base, axes=2)
        n = torch.arange(ca.G * ca.G, device="cuda")
        self.positions = torch.stack((n // ca.G, n % ca.G), -1).to(torch.int32).expand(ca.B, -1, -1)
        self._saved = self._gains = None

    def _heads(self, t):
        ca = self.ca
        return t.view(ca.B, ca.G * ca.G, ca.H, ca.D)

    def forward(self, x, alive=None):
        """The heads' output for states x; ``alive``: bool [B, G, G], the cells that are seen. What
        ``backward`` needs is kept here, apart from what the caller has: the output, the mask and
        the gains may be changed in place before it."""
        q0, k0, v = (self._heads(t) for t in self.ca.project(x))
        if alive is not None:
            alive = alive.reshape(self.ca.B, -1).clone()
        gains = self.wq.clone(), self.wk.clone()
        q, k = qk_norm_rotate(q0, k0, *gains, self.positions, self.freqs, eps=self.eps)
        out, lse = attend(q, k, v, alive=alive)
        self._saved = (q0, k0, q, k, v, out, lse, alive)
        self._gains = gains
        return out.clone().view(self.ca.state_shape)

    def backward(self, grad):
        """Gradients of the projections of the last forward, planes as states -> (dP, dI, dV); of the
        gains in ``dwq`` and ``dwk``."""
        if self._saved is None:
            raise RuntimeError("backward without a forward")
        q0, k0, q, k, v, out, lse, alive = self._saved
        dq, dk, dv = attend_backward(self._heads(grad), q, k, v, out, lse, alive=alive)
        dP, dI, self.dwq, self.dwk = qk_norm_rotate_backward(dq, dk, q0, k0, *self._gains, self.positions,
                                                             self.freqs, eps=self.eps)
        return tuple(t.view(self.ca.state_shape) for t in (dP, dI, dv))


class CellHistory:
    """Each cell's attention to its own states so far, one state a call: the cells are the batch,
    and keys are normed and placed as they enter the cache. ``window``: how many states back a
    state looks (0: all)."""

    def __init__(self, ca: Pseudopod, capacity: int, window: int = 0, base: float = 10000.0, eps: float = 1e-6):
        torch = _torch()
        if capacity < 1:
            raise ValueError(f"capacity must be >= 1, got {capacity}")
        self.ca, self.capacity, self.window, self.eps = ca, capacity, window, eps
        self.cells = ca.B * ca.G * ca.G
        self.wq, self.wk = (torch.ones(ca.D, device="cuda") for _ in range(2))
        self.freqs = rotation_freqs(ca.D, base)
        self.keys, self.values = (torch.empty((self.cells, capacity, ca.H, ca.D), dtype=ca.torch_dtype, device="cuda")
                                  for _ in range(2))
        self.times = torch.arange(capacity, dtype=torch.int32, device="cuda")
        self.length = 0

    def step(self, x):
        """Adds state x and returns its heads' output, [B, G, G, C]. A step that raises adds nothing."""
        torch = _torch()
        if self.length == self.capacity:
            raise RuntimeError(f"the history holds its {self.capacity} states")
        t = self.length
        q, k, v = (p.view(self.cells, 1, self.ca.H, self.ca.D) for p in self.ca.project(x))
        at = self.times[t:t + 1].view(1, 1, 1).expand(self.cells, 1, 1)
        q, _ = qk_norm_rotate(q, k, self.wq, self.wk, at, self.freqs, eps=self.eps,
                              out=(torch.empty_like(q), self.keys[:, t:t + 1]))
        self.values[:, t:t + 1].copy_(v)
        out, _ = attend(q, self.keys[:, :t + 1], self.values[:, :t + 1], causal=True, window=self.window)
        self.length = t + 1
        return out.view(self.ca.state_shape)


def main() -> None:
    torch = _torch()
    from .synthetic import CAConfig, make_params, make_state
    cfg = CAConfig("heads", B=2, G=32, H=8, D=32, dtype="bf16", steps=1, w_std=0.1)
    with Pseudopod(cfg.B, cfg.G, cfg.H, cfg.D, cfg.dtype, cfg.dt) as ca:
        ca.set_params(make_params(cfg, seed=1))
        x = torch.from_numpy(make_state(cfg, seed=2)).cuda().to(ca.torch_dtype)

        # The heads of other gains, which the training finds.
        heads = GlobalHeads(ca)
        heads.wq += 0.5 * torch.randn(cfg.D, generator=torch.Generator().manual_seed(3)).cuda()
        target = heads.forward(x).float()
        heads.wq.fill_(1.0)
        first = None
        for i in range(40):
            diff = heads.forward(x).float() - target
            loss = float(diff.square().mean())
            first = first or loss
            heads.backward((2 * diff / diff.square().mean().sqrt()).to(ca.torch_dtype))
            for w, g in ((heads.wq, heads.dwq), (heads.wk, heads.dwk)):
                w -= 0.02 * g / g.square().mean().sqrt()
            if i % 10 == 0:
                print(f"step {i}: loss {loss:.3e}", flush=True)
        print(f"loss {first:.3e} -> {loss:.3e}", flush=True)

        past = CellHistory(ca, capacity=12)
        for _ in range(past.capacity):
            y = past.step(x)
            x = ca.forward(x)
        print(f"history of {past.length} states: {past.cells} cells, output {tuple(y.shape)}, "
              f"largest {float(y.float().abs().max()):.3f}", flush=True)
        if not (math.isfinite(loss) and loss < first and bool(torch.isfinite(y).all())):
            raise SystemExit("the heads did not train")


if __name__ == "__main__":
    main()

"""Attention of cells beyond their 3x3 patch: over a whole grid, or over a history of states.

The CA activation lets a cell attend to its nine neighbours. Here the projections P, I and V of
``Pseudopod.project`` serve as queries, keys and values of any cells::

    q, k, v = (t.view(B, G * G, H, D) for t in ca.project(x))
    q, k = qk_norm_rotate(q, k, wq, wk, positions, rotation_freqs(D, axes=2))
    out, lse = attend(q, k, v)

and ``attend_backward`` and ``qk_norm_rotate_backward`` give the gradients. All arithmetic runs in
``libslime_ca.so`` (include/slime_ca.h, ``slime_ca_attend`` and ``slime_ca_qk_norm_rotate``), which
the module ``_binding`` calls on torch's tensors; nothing synchronises, and every call may be
captured into a graph.

As ``Pseudopod``'s, the calls are outside autograd: outputs require no grad, and the gradients are
calls of their own.

Tensors are CUDA tensors [B, N, heads, D] (N cells or states), float32 or bfloat16, with any
strides but 1 along D: planes [B, G, G, C] viewed per head, parts of one packed product, or heads
first. D is 8, 16, 32, 64 or 128; Hq query heads share Hkv key heads, Hq % Hkv == 0. ``stream``
(default: the current one) is where a call runs and its outputs belong.
"""
from __future__ import annotations

import contextlib
import importlib.util
import math
import operator
import os

from . import _lib
from .ca import _torch

HEAD_DIMS = (8, 16, 32, 64, 128)
PAIRS = ("halves", "adjacent")
ALIGN = ("end", "start")

BINDING_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_binding.so")

_native = None  # the module of csrc/binding.cpp


def load():
    """The module that makes the calls; raises if it has not been built, or for another torch, whose
    tensors it would misread."""
    global _native
    if _native is None:
        _lib.load()
        torch = _torch()  # its libraries are what the module links to
        if not os.path.exists(BINDING_PATH):
            raise ImportError(f"{BINDING_PATH} is missing: build it with `python -m slime_amd.build`")
        spec = importlib.util.spec_from_file_location("slime_amd._binding", BINDING_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        built = getattr(module, "torch_version", "unknown")
        if built != str(torch.__version__):
            raise ImportError(f"{BINDING_PATH} was built for torch {built}, this is {torch.__version__}: "
                              "build it again with `python -m slime_amd.build`")
        _native = module
    return _native


def _call(name, stream, args, check):
    """Makes a call of the native module; ``check`` says what is wrong with arguments that it did not
    take. On another stream than the current one, what it allocates belongs to that stream, and its
    inputs are kept until it is done."""
    native = _native or load()
    if stream is None:
        r = getattr(native, name)(*args)
    else:
        check()
        torch = _torch()
        with contextlib.ExitStack() as stack:
            stack.enter_context(torch.cuda.stream(stream))
            for x in args:
                if isinstance(x, torch.Tensor):
                    x.record_stream(stream)
            r = getattr(native, name)(*args)
    if type(r) is tuple:
        return r
    if r is None:
        check()
        raise ValueError(f"{name}: arguments out of range")
    _lib.check(r)


def _check(t, name, like=None, shape=None) -> None:
    """A CUDA tensor [B, N, heads, D], dense along D, of the type and device of ``like``."""
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dim() != 4 or not t.is_cuda or t.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{name} must be a CUDA tensor [B, N, heads, D] of float32 or bfloat16, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.stride(3) != 1:
        raise ValueError(f"{name} must have stride 1 along its channels, got strides {t.stride()}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _check_vector(t, name, n, dtype, like) -> None:
    if not isinstance(t, _torch().Tensor) or tuple(t.shape) != (n,) or t.dtype != dtype or t.device != like.device \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} values on {like.device}, got "
                         + (f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, _torch().Tensor) else repr(t)))


def _check_heads(Hq, Hkv, D) -> None:
    if D not in HEAD_DIMS:
        raise ValueError(f"heads of {D} channels: must be one of {HEAD_DIMS}")
    if Hkv < 1 or Hq % Hkv or Hq < 1:
        raise ValueError(f"{Hq} query heads cannot share {Hkv} key heads")


def _check_output(t, name, like, itself, apart) -> None:
    """``apart``: what the output may not share memory with, by name; it may be all of ``itself``."""
    _check(t, name, like, like.shape)
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} repeats memory (strides {t.stride()})")
    for other, x in apart.items():
        if x is not None and load().overlaps(t, x, other == itself):
            raise ValueError(f"{name} lies in the memory of {other}")


# ---- norm and rotation ---------------------------------------------------------------------

def rotation_freqs(D: int, base: float = 10000.0, axes: int = 1, device="cuda"):
    """Radians per position of each pair of channels, float64 [D / 2]: base^(-i / n) for pair i
    of the n = D / 2 / axes pairs of each axis."""
    if D not in HEAD_DIMS or axes not in (1, 2):
        raise ValueError(f"heads of {D} channels and {axes} axes: D must be one of {HEAD_DIMS}, axes 1 or 2")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be finite and positive, got {base}")
    torch = _torch()
    n = D // 2 // axes
    f = float(base) ** (-torch.arange(n, dtype=torch.float64) / n)
    return f.repeat(axes).to(device)


def _check_norm(q, k, wq, wk, positions, freqs, eps, pairs, out=None, grads=()):
    torch = _torch()
    _check(q, "q")
    _check(k, "k", q)
    B, N, Hq, D = q.shape
    _check(k, "k", q, (B, N, k.shape[2], D))
    _check_heads(Hq, k.shape[2], D)
    _check_vector(wq, "wq", D, torch.float32, q)
    _check_vector(wk, "wk", D, torch.float32, q)
    _check_vector(freqs, "freqs", D // 2, torch.float64, q)
    if not isinstance(positions, torch.Tensor) or positions.dim() != 3 or tuple(positions.shape[:2]) != (B, N) \
            or positions.shape[2] not in (1, 2) or positions.dtype != torch.int32 or positions.device != q.device:
        raise ValueError(f"positions must be an int32 tensor [{B}, {N}, 1 or 2] on {q.device}")
    if positions.shape[2] == 2 and positions.stride(2) != 1:
        raise ValueError("positions must have stride 1 along its coordinates")
    if pairs not in PAIRS:
        raise ValueError(f"pairs must be one of {sorted(PAIRS)}, got {pairs!r}")
    if out is not None:
        inputs = dict(q=q, k=k, wq=wq, wk=wk, positions=positions, freqs=freqs)
        _check_output(out[0], "out[0]", q, "q", inputs)
        _check_output(out[1], "out[1]", k, "k", {**inputs, "out[0]": out[0]})
    for g, name, like in zip(grads, ("grad_q", "grad_k"), (q, k)):
        _check(g, name, q, like.shape)


def qk_norm_rotate(q, k, wq, wk, positions, freqs, *, eps: float = 1e-6, pairs: str = "halves",
                   out=None, stream=None):
    """Queries and keys normed per head (x w / sqrt(mean(x^2) + eps), gains ``wq``, ``wk``:
    float32 [D]) and rotated by position, in one pass -> (q, k).

    ``positions``: int32 [B, N, 1] (an index), or [B, N, 2] (a cell's y and x: the first half of the
    pairs turns by y, the second by x); any batch and row strides. ``freqs``: float64 [D / 2], radians
    per position of each pair (``rotation_freqs``). ``pairs``: "halves" turns channels (i, i + D / 2),
    "adjacent" (2i, 2i + 1). ``out``: (q, k) to write; each may be its own input, place by place, and
    shares no other memory with the arguments."""
    oq, ok = (None, None) if out is None else out
    return _call("norm", stream, (q, k, wq, wk, positions, freqs, eps, pairs, oq, ok),
                 lambda: _check_norm(q, k, wq, wk, positions, freqs, eps, pairs, out))


def qk_norm_rotate_backward(grad_q, grad_k, q, k, wq, wk, positions, freqs, *, eps: float = 1e-6,
                            pairs: str = "halves", stream=None):
    """The gradient of ``qk_norm_rotate`` at its inputs for these gradients of its outputs ->
    (dq, dk, dwq, dwk): of the inputs in their type, of the gains float32 [D]."""
    return _call("norm_backward", stream, (q, k, wq, wk, positions, freqs, eps, pairs, grad_q, grad_k),
                 lambda: _check_norm(q, k, wq, wk, positions, freqs, eps, pairs, grads=(grad_q, grad_k)))


# ---- attention -----------------------------------------------------------------------------

def _check_attend(q, k, v, scale, window, align, lengths, alive, out=None, back=()):
    torch = _torch()
    _check(q, "q")
    _check(k, "k", q)
    B, Nq, Hq, D = q.shape
    _, Nk, Hkv, _ = k.shape
    _check_heads(Hq, Hkv, D)
    _check(k, "k", q, (B, Nk, Hkv, D))
    _check(v, "v", q, (B, Nk, Hkv, D))
    if align not in ALIGN:
        raise ValueError(f"align must be one of {sorted(ALIGN)}, got {align!r}")
    if operator.index(window) < 0:
        raise ValueError(f"window must be >= 0, got {window}")
    if scale is not None and not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be finite and > 0, got {scale}")
    if lengths is not None:
        _check_vector(lengths, "lengths", B, torch.int32, q)
    if alive is not None and (not isinstance(alive, torch.Tensor) or tuple(alive.shape) != (B, Nk)
                              or alive.dtype not in (torch.bool, torch.uint8)
                              or alive.device != q.device or (Nk > 1 and alive.stride(1) != 1)):
        raise ValueError(f"alive must be a bool or uint8 tensor [{B}, {Nk}] with dense rows on {q.device}")
    if out is not None:
        _check_output(out, "out", q, "q", dict(q=q, k=k, v=v, lengths=lengths, alive=alive))
    if back:
        grad_out, out, lse = back
        _check(grad_out, "grad_out", q, q.shape)
        _check(out, "out", q, q.shape)
        if not isinstance(lse, torch.Tensor) or tuple(lse.shape) != (B, Hq, Nq) or lse.dtype != torch.float32 \
                or lse.device != q.device or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous float32 tensor [{B}, {Hq}, {Nq}] on {q.device}")


def attend(q, k, v, *, scale: float | None = None, causal: bool = False, window: int = 0,
           align: str = "end", lengths=None, alive=None, out=None, stream=None):
    """softmax(scale q . k) over the keys that each query sees, applied to v -> (out, lse): out as
    q, lse float32 [B, Hq, Nq] the log of the sum of exp(scale q . k). ``scale``: 1 / sqrt(D).

    Key j is seen if it is below ``lengths[b]`` (int32 [B]; default all) and ``alive`` (bool or uint8
    [B, Nk], a mask of living cells; default all). Query i sits at position p = i + lengths[b] - Nq
    (``align`` "end": the queries are the last of the keys, as when a history grows) or p = i
    ("start": a padded batch in training); with ``causal`` it sees j <= p, with a ``window`` W > 0
    p - j < W and, unless causal, j - p < W. A query that sees no key gives 0 and -inf.

    ``out``: where to write the output, of q's shape; it may be q itself, and shares no other memory
    with the arguments.

    Few queries over many keys (one new state over a long history) are split over the device."""
    return _call("attend", stream, (q, k, v, scale, causal, window, align, lengths, alive, out),
                 lambda: _check_attend(q, k, v, scale, window, align, lengths, alive, out))


def attend_backward(grad_out, q, k, v, out, lse, *, scale: float | None = None, causal: bool = False,
                    window: int = 0, align: str = "end", lengths=None, alive=None, stream=None):
    """The gradient of ``attend`` at its inputs, from its outputs and the gradient of ``out`` ->
    (dq, dk, dv) in the inputs' type; dk and dv are summed over the query heads of a key head, and
    keys that no query may see get 0. The probabilities are computed again from lse."""
    return _call("attend_backward", stream, (q, k, v, scale, causal, window, align, lengths, alive, grad_out, out, lse),
                 lambda: _check_attend(q, k, v, scale, window, align, lengths, alive, back=(grad_out, out, lse)))


__all__ = ["attend", "attend_backward", "qk_norm_rotate", "qk_norm_rotate_backward", "rotation_freqs",
           "HEAD_DIMS", "PAIRS", "ALIGN"]

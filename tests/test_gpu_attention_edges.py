"""attend and attend_backward where a workgroup's work ends early, or a call outgrows one launch."""
import ctypes
import math

import pytest

from slime_amd import _lib
from tests import attention_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _draw(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _splits(B, Nq, Nk, Hq, Hkv, D, dtype):
    """Of the forward, from its workspace."""
    cfg = _lib.AttendConfig(B, Nq, Nk, Hq, Hkv, D, _lib.SLIME_BF16 if dtype == torch.bfloat16 else _lib.SLIME_F32,
                            1.0, 0, 0, 0, None, None, 0)
    n = ctypes.c_size_t()
    _lib.check(_lib.load().slime_ca_attend_workspace(ctypes.byref(cfg), 0, ctypes.byref(n)))
    return n.value // (4 * B * Hq * Nq * (D + 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 16, 32, 128])
def test_splits_without_a_tile(D, dtype):
    """Few rows over histories of which most are far shorter than the split keys: the splits that
    get no tile (heads below the padded width among them) add nothing."""
    import slime_amd
    B, Nq, Nk, Hq, Hkv = 5, 2, 3000, 4, 2
    dt = DTYPES[dtype]
    assert _splits(B, Nq, Nk, Hq, Hkv, D, dt) >= 4
    lengths = torch.tensor([3000, 130, 1, 0, 129], dtype=torch.int32, device="cuda")
    q, k, v = (_draw((B, n, h, D), dt, s) for n, h, s in ((Nq, Hq, 1), (Nk, Hkv, 2), (Nk, Hkv, 3)))
    r = ref.Reference(q, k, v, 1 / math.sqrt(D), ref.seen_mask(B, Nq, Nk, lengths=lengths))
    first = None
    for _ in range(3):
        out, lse = slime_amd.attend(q, k, v, lengths=lengths)
        ref.within(out, r.out.permute(0, 2, 1, 3), r.out_tol.permute(0, 2, 1, 3), "out")
        ref.within(lse, r.lse, r.lse_tol, "lse")
        first = first or (out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    assert not out[3].any() and bool((lse[3] == -math.inf).all())

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


def _living(B, seed):
    """(lengths, alive) of one key an entry: 0 or 1, and a cell that lives or not."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(2, B, 1, generator=g, device="cuda") < 0.8).unbind(0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_heads_than_a_launch(dtype):
    """2^21 entries of 8 heads, one query and one key each, in views of one packed product: twice what
    a launch of 256 threads a head may hold. With one key the output is its value: its weight and their
    sum are the same number, so in bf16 bit by bit, in fp32 to the product, the quotient and the
    joining of four waves. The value's gradient is the output's; the score's is 0, but for its two
    terms of D products each, rounded apart."""
    import slime_amd
    B, H, D, dt = 2 ** 21 + 5, 8, 8, DTYPES[dtype]
    x = _draw((B, 1, 3 * H, D), dt, 1)
    q, k, v = x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:]
    below, lives = _living(B, 2)
    how = dict(lengths=below[:, 0].int().contiguous(), alive=lives)
    seen = (below & lives)[:, :, None, None]
    out, lse = slime_amd.attend(q, k, v, **how)
    if dt == torch.bfloat16:
        assert torch.equal(out, v * seen)
    else:
        assert bool(((out - v * seen).abs() <= 8 * ref.U32 * v.abs() * seen).all())
    score = (q.float() * k.float()).sum(-1).transpose(1, 2) / math.sqrt(D)
    size = (q.float() * k.float()).abs().sum(-1).transpose(1, 2) / math.sqrt(D)
    live = seen[..., 0].expand_as(lse)
    assert bool((lse[~live] == -math.inf).all())
    # the reference's bound for one key, and as many roundings of the sum here
    bound = ((2 * D + 16) * size + 48 + 8 * score.abs()) * ref.U32
    assert bool(((lse - score).abs() <= bound)[live].all())
    gout = _draw(q.shape, dt, 3)
    dq, dk, dv = slime_amd.attend_backward(gout, q, k, v, out, lse, **how)
    # 2^(s - lse) is 1 but for their roundings, and bf16's one
    off = (2 * D + 24) * ref.U32 * (1 + size + lse.abs().nan_to_num(0, 0, 0)).transpose(1, 2)[..., None]
    u = ref.u_of(dt) * (2 if dt == torch.bfloat16 else 1)
    assert bool(((dv.float() - gout.float() * seen).abs() <= (off + u) * gout.float().abs()).all())
    ds = 4 * (D + 4) * ref.U32 * (gout.float() * v.float()).abs().sum(-1, keepdim=True) * 1.01 / math.sqrt(D)
    for got, other in ((dq, k), (dk, q)):
        assert bool((got.float().abs() <= ds * other.float().abs() * seen).all())


def test_slices_of_a_batch_take_their_own_lengths():
    """As many heads, none to three keys an entry: entries about the slices' ends are as in a call of
    them alone."""
    import slime_amd
    B, H, D = 2 ** 21 + 5, 8, 8
    q, k, v = (_draw((B, 1 if i == 0 else 3, H, D), torch.bfloat16, i) for i in range(3))
    lengths = (torch.arange(B, device="cuda") % 4).int()
    out, lse = slime_amd.attend(q, k, v, lengths=lengths)
    n = 1000
    for at in (0, B // 2 - n // 2, B - n):
        part = slice(at, at + n)
        o, s = slime_amd.attend(q[part], k[part], v[part], lengths=lengths[part])
        assert torch.equal(o, out[part]) and torch.equal(s, lse[part])


@pytest.mark.parametrize("power", [-20, -100, -112, -120, -126])
def test_small_fp32_values_in_three_parts(power):
    """Many rows in fp32: each value as three bf16 parts, of which the last ends at bf16's smallest
    step, 2^-133. So a value is off by half of that at most, beside the reference's bound, and each of a
    sum's products by half of fp32's smallest, 2^-149."""
    import slime_amd
    B, N, H, D = 1, 70, 2, 32
    q, k, v = (_draw((B, N, H, D), torch.float32, s) for s in (1, 2, 3))
    v = (v.double() * 2.0 ** power).float()
    r = ref.Reference(q, k, v, 1 / math.sqrt(D), ref.seen_mask(B, N, N))
    out, _ = slime_amd.attend(q, k, v)
    tol = (2 * r.ds + (N + 32) * ref.U32) * (r.p @ r.v.abs()) + ref.U32 * r.out.abs() + 2.0 ** -134 + 6 * N * 2.0 ** -150
    ref.within(out, r.out.permute(0, 2, 1, 3), tol.permute(0, 2, 1, 3), "out")


@pytest.mark.parametrize("value, fits", [(3.38e38, True), (-3.38e38, True), (3.4e38, False), (math.inf, False)])
def test_the_largest_fp32_values(value, fits):
    """Above the largest bf16, 3.39e38, a value of many rows in fp32 is NaN, in its channel alone; few
    rows take every value."""
    import slime_amd
    q, k, v = (torch.zeros(1, n, 1, 32, device="cuda") for n in (64, 64, 64))
    v[0, 3, 0, 5] = value
    for rows in (64, 8):
        out, _ = slime_amd.attend(q[:, :rows], k, v)
        want = torch.full((rows,), value / 64, device="cuda")
        got = out[0, :, 0, 5]
        if fits or rows == 8:
            # 64 equal weights: their product, the sum's quotient and the split's rest
            assert torch.equal(got, want) or float(((got - want) / want).abs().max()) <= 16 * ref.U32
        else:
            assert bool(torch.isnan(got).all())
        out[0, :, 0, 5] = 0
        assert not out.any()


@pytest.mark.parametrize("Nq,Nk,Hq,Hkv,D", [(1, 65, 8, 8, 64), (1, 4000, 8, 2, 64), (32, 77, 2, 2, 32), (4, 300, 8, 1, 128),
                                            (3, 1000, 4, 4, 16), (1, 2, 8, 8, 8)])
@pytest.mark.parametrize("living", [False, True], ids=["", "alive"])
def test_bf16_weights_of_few_rows_in_two_parts(Nq, Nk, Hq, Hkv, D, living):
    """At most 32 rows a key head: each weight is off by two roundings to bf16, one of the other's
    rest (2^-16), so the output's own rounding is all that is left of that type."""
    import slime_amd
    B, dt = 3, torch.bfloat16
    q, k, v = (_draw((B, n, h, D), dt, s) for n, h, s in ((Nq, Hq, 1), (Nk, Hkv, 2), (Nk, Hkv, 3)))
    g = torch.Generator(device="cuda").manual_seed(4)
    alive = torch.rand(B, Nk, generator=g, device="cuda") < 0.7 if living else None
    r = ref.Reference(q, k, v, 1 / math.sqrt(D), ref.seen_mask(B, Nq, Nk, alive=alive))
    out, _ = slime_amd.attend(q, k, v, alive=alive)
    u = ref.u_of(dt)
    tol = (2 * r.ds + (Nk + 32) * ref.U32 + u * u) * (r.p @ r.v.abs()) + u * r.out.abs() + 1e-30
    ref.within(out, r.out.permute(0, 2, 1, 3), tol.permute(0, 2, 1, 3), "out")

"""CPU checks: calls of more workgroups than a launch takes are refused by name, or go in slices."""
import ctypes

import pytest

from slime_amd import _lib


def _status(back, **kw):
    base = dict(B=1, Nq=1, Nk=1, Hq=8, Hkv=8, D=8, dtype=_lib.SLIME_BF16, scale=1.0)
    base.update(kw)
    n = ctypes.c_size_t()
    rc = _lib.load().slime_ca_attend_workspace(ctypes.byref(_lib.AttendConfig(**base)), back, ctypes.byref(n))
    return rc, _lib.load().slime_ca_last_error()


@pytest.mark.parametrize("back", [0, 1])
@pytest.mark.parametrize("size", [dict(B=2 ** 21), dict(B=2 ** 24), dict(B=2 ** 31 - 1), dict(B=2 ** 27, Nq=33),
                                  dict(B=2 ** 21, Hq=16, Nk=1000), dict(B=2 ** 22, D=128, dtype=_lib.SLIME_F32)])
def test_large_batches_are_taken(back, size):
    """(Without a device: as far as asking for one.)"""
    assert _status(back, **size)[0] in (_lib.SLIME_OK, _lib.SLIME_ENODEV)


# 128 rows a workgroup; a launch of 256 threads each holds 2^24 less one, in eights.
@pytest.mark.parametrize("tiles, taken", [(2 ** 13 - 1, True), (2 ** 13, False), (2 ** 20, False)])
def test_one_entry_is_within_a_launch(tiles, taken):
    rc, message = _status(0, Hq=2048, Hkv=2048, Nq=128 * tiles)
    assert (rc in (_lib.SLIME_OK, _lib.SLIME_ENODEV)) == taken
    if not taken:
        assert rc == _lib.SLIME_EINVAL and b"one batch entry exceeds one launch" in message


def test_one_entry_of_many_keys():
    # Keys' workgroups of 128 count in the gradient only.
    size = dict(Hq=2048, Hkv=2048, Nk=2 ** 20)
    assert _status(0, **size)[0] in (_lib.SLIME_OK, _lib.SLIME_ENODEV)
    assert _status(1, **size)[0] == _lib.SLIME_EINVAL
    assert _status(1, Hq=1024, Hkv=1024, Nk=2 ** 20)[0] in (_lib.SLIME_OK, _lib.SLIME_ENODEV)
    assert _status(1, Hq=1024, Hkv=1024, Nk=2 ** 20, D=128)[0] == _lib.SLIME_EINVAL  # in two roles


@pytest.mark.parametrize("D, rows, taken", [(128, 2 ** 28 - 16, True), (128, 2 ** 28 - 15, False),
                                            (64, 2 ** 29 - 32, True), (64, 2 ** 29 - 31, False), (8, 2 ** 30 - 1, True)])
def test_norm_rows_are_within_a_launch(D, rows, taken):
    """Refused before any pointer is used; calls that are taken stop at the missing tensors."""
    lib = _lib.load()
    one = ctypes.c_float()
    p = ctypes.c_void_p(ctypes.addressof(one))
    cfg = _lib.NormConfig(B=1, N=rows, Hq=1, Hkv=1, D=D, dtype=_lib.SLIME_BF16, axes=1, eps=1e-6, positions=p, pos_row=1,
                          freqs=p)
    h = ctypes.byref(_lib.Heads(None if taken else p, 0, 0, 0))
    assert lib.slime_ca_qk_norm_rotate(ctypes.byref(cfg), h, h, p, p, h, h, None) == _lib.SLIME_EINVAL
    assert (b"NULL" if taken else b"exceed one launch") in lib.slime_ca_last_error()

"""Outputs that lie in the memory of an input are told apart from those that lie beside it (CPU only).

``tests/overlap_check.cpp`` compares ``slime_amd/csrc/overlap.hpp`` with a list of all bytes; here
the module's answers for torch's views.
"""
import os
import subprocess

import pytest
import torch

from slime_amd import attention

SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "overlap_check.cpp")


def _run(tmp_path, *defines):
    exe = str(tmp_path / "overlap_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", *defines, "-o", exe, SRC], check=True)
    return subprocess.run([exe], capture_output=True, text=True, timeout=120)


def test_against_a_list_of_all_bytes(tmp_path):
    r = _run(tmp_path)
    assert r.returncode == 0 and r.stdout == "OK\n", r.stdout


def test_a_planted_mistake_is_reported(tmp_path):
    r = _run(tmp_path, "-DPLANT_OVERLAP")
    assert r.returncode == 1 and "errors" in r.stdout, r.stdout


def _views():
    """(output, input, whether it may be the input itself, whether they overlap), by name."""
    x = torch.zeros(2, 6, 12, 8, dtype=torch.bfloat16)
    q, k, v = x[:, :, :4], x[:, :, 4:8], x[:, :, 8:]
    heads = torch.zeros(2, 4, 6, 8, dtype=torch.bfloat16)
    cache = torch.zeros(2, 9, 4, 8, dtype=torch.bfloat16)
    flat = torch.zeros(2 * 6 * 4 * 8 + 8, dtype=torch.bfloat16)
    at = lambda i: flat[i:i + 384].view(2, 6, 4, 8)  # noqa: E731
    return {
        "another tensor": (torch.zeros_like(q), q, False, False),
        "a part of the same product": (q, k, False, False),
        "the next part of it": (k, v, False, False),
        "the input itself": (q, q, True, False),
        "the input itself, where it may not be": (k, k, False, True),
        "heads that cross": (x[:, :, 3:7], q, True, True),
        "rows that cross": (cache[:, 1:7], cache[:, :6], True, True),
        "a row past the others": (cache[:, 8:9], cache[:, :8], False, False),
        "one of the rows": (cache[:, 7:8], cache[:, :8], False, True),
        "other batch entries": (x[:1, :, :4], x[1:, :, :4], True, False),
        "an element on": (at(1), at(0), True, True),
        "its last element": (flat[383:391].view(1, 1, 1, 8), at(0), False, True),
        "just behind it": (flat[384:].view(1, 1, 1, 8), at(0), False, False),
        "the same memory in another order": (heads.transpose(1, 2), heads.view(2, 6, 4, 8), True, True),
        "a broadcast input": (cache[:, :1], cache[:1, :1].expand(2, 9, 4, 8), False, True),
        "beside a broadcast input": (cache[:, 1:2], cache[:1, :1].expand(2, 9, 4, 8), False, False),
        "no elements": (x[:, :0], x, False, False),
        "a mask in bytes": (torch.zeros(4, dtype=torch.bfloat16), torch.zeros(2, 9, dtype=torch.bool), False, False),
        "bytes of its own": (flat[:8], flat.view(torch.uint8)[15:16], False, True),
        "bytes past its own": (flat[:8], flat.view(torch.uint8)[16:17], False, False),
    }


@pytest.mark.parametrize("name", _views())
def test_views(name):
    out, x, may_be, want = _views()[name]
    assert attention.load().overlaps(out, x, may_be) is want


def test_the_check_names_the_input(monkeypatch):
    q, k = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 8)
    monkeypatch.setattr(attention, "_check", lambda *a: None)  # of CUDA tensors
    attention._check_output(q, "out", q, "q", dict(q=q, k=k, alive=None))
    with pytest.raises(ValueError, match="out lies in the memory of k"):
        attention._check_output(k, "out", q, "q", dict(q=q, k=k))

"""CPU checks of the build: the library is for any C host, and needs no torch."""
import importlib.util
import os
import types

import pytest

from slime_amd import build


@pytest.fixture
def made(monkeypatch, tmp_path):
    """What a build with the compilers left out makes, in order."""
    out = []
    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    monkeypatch.setattr(build, "_compile", lambda src: src)
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: types.SimpleNamespace(returncode=0, stderr=""))
    monkeypatch.setattr(build.os, "replace", lambda tmp, to: out.append(to))
    return out


def test_all_of_it_with_torch(made):
    build.build()
    assert sorted(made) == sorted([build.LIB, build.PROBE_LIB, build.BINDING])
    assert made.index(build.LIB) < made.index(build.BINDING)


def test_the_library_without_torch(made, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    build.build(verbose=True)
    assert made == [build.LIB, build.PROBE_LIB]
    assert "no torch" in capsys.readouterr().out


def test_the_library_with_a_torch_that_knows_no_gpu(made, monkeypatch, tmp_path):
    os.makedirs(tmp_path / "torch" / "lib")
    spec = types.SimpleNamespace(submodule_search_locations=[str(tmp_path / "torch")])
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *a: spec)
    build.build()
    assert made == [build.LIB, build.PROBE_LIB]

"""CPU checks of the module behind the attention calls: it is loaded only with the torch that it was
built for."""
import pytest
import torch

from slime_amd import attention


def test_it_loads_with_its_own_torch(monkeypatch):
    monkeypatch.setattr(attention, "_native", None)
    assert attention.load().torch_version == str(torch.__version__)


def test_another_torch_is_refused(monkeypatch):
    monkeypatch.setattr(attention, "_native", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0+elsewhere")
    with pytest.raises(ImportError, match="1.0.0.elsewhere.*slime_amd.build"):
        attention.load()
    assert attention._native is None


def test_a_module_that_is_not_there_is_named(monkeypatch, tmp_path):
    monkeypatch.setattr(attention, "_native", None)
    monkeypatch.setattr(attention, "BINDING_PATH", str(tmp_path / "_binding.so"))
    with pytest.raises(ImportError, match="slime_amd.build"):
        attention.load()

"""The compiled calls are loaded only if they were built for the torch, the Python and the sources that are here."""
import pytest

from verified_metal_kernels_b200 import build
from verified_metal_kernels_b200.kernels import _common


@pytest.fixture
def unloaded(monkeypatch):
    build.build()
    build.build_calls()
    monkeypatch.setattr(_common, "_calls", None)


def test_loaded_where_the_stamp_agrees(unloaded):
    assert build.calls_fresh() and _common.calls() is _common.calls()


def test_not_loaded_for_another_torch(unloaded, monkeypatch):
    import torch
    monkeypatch.setattr(torch, "__version__", "1.0")
    with pytest.raises(RuntimeError, match="built for another torch"):
        _common.calls()


def test_not_loaded_without_a_stamp(unloaded, monkeypatch, tmp_path):
    lib = tmp_path / "_vmk_torch.so"
    lib.write_bytes(b"")
    monkeypatch.setattr(build, "CALLS_LIB", str(lib))
    assert not build.calls_fresh()
    with pytest.raises(RuntimeError, match="build it with"):
        _common.calls()
    lib.with_name("_vmk_torch.so.stamp").write_text("0" * 64 + "\n")
    assert not build.calls_fresh()

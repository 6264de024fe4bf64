"""The CPython module behind paged: used only where it was built from what is here."""
import pytest

from thor_megakernels_b200 import _lib, build, paged


def test_the_module_carries_what_it_was_built_from():
    build.build_binding()
    assert build.binding_tag().encode() in build.BINDING.read_bytes()


@pytest.mark.parametrize("what", ["source", "version", "missing"])
def test_a_module_of_another_build_is_built_anew_or_refused(monkeypatch, tmp_path, what):
    there = tmp_path / "_paged_binding.so"
    if what != "missing":
        there.write_bytes(build.BINDING.read_bytes() if build.BINDING.exists() else b"")
    monkeypatch.setattr(build, "BINDING", there)
    if what == "source":   # newer than the module or not: contents count, not times
        source = tmp_path / "paged_binding.cpp"
        source.write_bytes(build.BINDING_SOURCE.read_bytes() + b"\n// another\n")
        monkeypatch.setattr(build, "BINDING_SOURCE", source)
    if what == "version":
        import torch

        monkeypatch.setattr(torch, "__version__", "0.0.1")
    calls = []

    class Failed:
        returncode, stdout, stderr = 1, "", "no compiler"

    monkeypatch.setattr(build.subprocess, "run", lambda *a, **k: calls.append(a) or Failed)
    monkeypatch.setattr(build, "find_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    with pytest.raises(RuntimeError, match="no compiler"):
        paged._binding.__wrapped__()
    assert calls


def test_struct_sizes_are_compared_with_the_library():
    module = paged._binding()
    lib = _lib.load()
    sizes = [lib.mk_abi_sizeof(which) for which in (4, 5, 6, 7)]
    addresses = [1, 1, 1]
    for i in range(4):
        wrong = list(sizes)
        wrong[i] += 8
        with pytest.raises(RuntimeError, match="structs"):
            module.init(*addresses, *wrong)
    with pytest.raises(TypeError):
        module.init(*addresses)

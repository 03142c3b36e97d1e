"""build.py on the host: the kernel library without torch, and when the
Python binding is built again."""

import sys

import pytest

from gpu_optimizer_b200 import build as b


@pytest.fixture
def built(tmp_path, monkeypatch):
    """A binding that is newer than its sources; counts its compilations."""
    b.build()
    monkeypatch.setattr(b, "BINDING", tmp_path / "_ops.so")
    runs = []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def compile_(cmd, **kw):
        runs.append(cmd)
        (tmp_path / "_ops.so.tmp").write_bytes(b"")
        return Done()

    monkeypatch.setattr(b.subprocess, "run", compile_)
    b.build_binding()
    assert len(runs) == 1
    return runs


def test_binding_is_built_once(built):
    b.build_binding()
    assert len(built) == 1


@pytest.mark.parametrize("what", ["torch", "python"])
def test_binding_is_built_again_for_another_torch_or_python(built, monkeypatch, what):
    """The binding is compiled against both: an old one would fail at import,
    or worse."""
    import sysconfig

    import torch

    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9")
    else:
        include = sysconfig.get_paths()["include"]
        monkeypatch.setattr(sysconfig, "get_paths", lambda *a: {"include": include + ".9"})
    b.build_binding()
    assert len(built) == 2
    b.build_binding()
    assert len(built) == 2


def test_library_is_built_without_torch(built, monkeypatch, capsys):
    """libgpo.so does not need torch; the binding, which does, is left out
    with a word."""
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises ImportError
    b.BINDING.unlink()
    assert b.build() == b.LIB
    assert "torch" in capsys.readouterr().err
    assert len(built) == 1 and not b.BINDING.exists()


def test_binding_of_another_abi_is_refused(monkeypatch):
    from gpu_optimizer_b200 import _lib, attention_ops
    from gpu_optimizer_b200.runner import KernelBuildError

    class Old:
        ABI_VERSION = _lib.ABI_VERSION + 1

        @staticmethod
        def set_refused(cls):
            pass

    monkeypatch.setattr(attention_ops, "_ops", None)
    monkeypatch.setattr(attention_ops.importlib, "import_module", lambda name: Old)
    with pytest.raises(KernelBuildError, match="built for ABI"):
        attention_ops._native()

"""When the training extension is built anew (no GPU, and nothing is compiled)."""
import os

from bioemu2_b200 import build as B


def test_an_extension_for_another_torch_or_python_is_stale(tmp_path, monkeypatch):
    binding, known = tmp_path / "_training.so", tmp_path / "_training.so.for"
    monkeypatch.setattr(B, "BINDING_PATH", str(binding))
    monkeypatch.setattr(B, "BINDING_FOR", str(known))
    assert B.binding_is_stale()
    binding.write_bytes(b"")
    later = os.path.getmtime(B.BINDING_SRC) + 1e6
    os.utime(binding, (later, later))
    assert B.binding_is_stale()  # of unknown origin
    known.write_text(B.binding_for())
    assert not B.binding_is_stale()
    here = B.binding_for
    for other in (here() + "0", here().replace("cpython-3", "cpython-2"), ""):
        monkeypatch.setattr(B, "binding_for", lambda: other)
        assert B.binding_is_stale()
    monkeypatch.setattr(B, "binding_for", here)
    os.utime(binding, (0, 0))
    assert B.binding_is_stale()


def test_what_an_extension_is_for_names_torch_and_python():
    import sysconfig

    import torch

    assert torch.version.git_version in B.binding_for() and sysconfig.get_config_var("SOABI") in B.binding_for()


def test_a_built_extension_says_what_it_is_for(monkeypatch, tmp_path):
    commands = []
    monkeypatch.setattr(B, "_run", lambda cmd, verbose: commands.append(cmd))
    monkeypatch.setattr(B, "BINDING_FOR", str(tmp_path / "for"))
    B.build_binding()
    assert (tmp_path / "for").read_text() == B.binding_for()
    import torch

    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}" in commands[0]


def test_the_two_compilers_run_side_by_side(monkeypatch):
    """Each waits for the other to have started; a failure of either is the build's."""
    import threading

    import pytest

    meet = threading.Barrier(2, timeout=20)
    monkeypatch.setattr(B, "build_library", lambda verbose: meet.wait())
    monkeypatch.setattr(B, "build_binding", lambda verbose: meet.wait())
    assert B.build(force=True) == B.LIB_PATH

    def fails(verbose):
        raise RuntimeError("no compiler")

    monkeypatch.setattr(B, "build_library", lambda verbose: None)
    monkeypatch.setattr(B, "build_binding", fails)
    with pytest.raises(RuntimeError, match="no compiler"):
        B.build(force=True)

"""What the build does where host compilers are missing (nothing here compiles)."""
import os

import pytest
import torch

from sdmchat_amd import build


def test_host_compiler(monkeypatch, tmp_path):
    monkeypatch.setenv("CXX", "ccache g++-12")
    assert build.host_compiler() == ["ccache", "g++-12"]
    monkeypatch.setenv("CXX", "")
    (tmp_path / "g++").write_text("")
    (tmp_path / "g++").chmod(0o755)
    monkeypatch.setenv("PATH", str(tmp_path))
    assert build.host_compiler() == [str(tmp_path / "g++")]
    (tmp_path / "g++").unlink()
    monkeypatch.setenv("ROCM_PATH", str(tmp_path))
    assert build.host_compiler() == ["clang++"]
    clang = tmp_path / "lib" / "llvm" / "bin" / "clang++"
    clang.parent.mkdir(parents=True)
    clang.write_text("")
    assert build.host_compiler() == [str(clang)]
    monkeypatch.delenv("CXX")
    assert build.host_compiler() == [str(clang)]


def test_a_missing_compiler_is_reported(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "LISTS", str(tmp_path / "_lists.so"))
    monkeypatch.setenv("CXX", str(tmp_path / "none"))
    src, err = build._compile_lists(False)
    assert src.endswith("lists.cpp") and "none" in err and not os.path.exists(build.LISTS)


def test_the_library_is_linked_without_the_extension(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "sources", lambda: [])
    monkeypatch.setattr(build, "_compile_lists", lambda verbose: ("lists.cpp", "no compiler\n"))

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def run(cmd, **kw):   # the link: its last argument is its output
        open(cmd[-1], "w").close()
        return Done
    monkeypatch.setattr(build.subprocess, "run", run)
    with pytest.raises(RuntimeError, match="lists.cpp"):
        build.build()
    assert os.path.exists(build.LIB)
    monkeypatch.setattr(build, "_compile_lists", lambda verbose: ("lists.cpp", None))
    assert build.build() == build.LIB


def test_another_torch_makes_the_extension_stale(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "LISTS", str(tmp_path / "_lists.so"))
    monkeypatch.setattr(build, "LISTS_TORCH", str(tmp_path / "_lists.torch"))
    assert build._lists_stale(0.0)
    (tmp_path / "_lists.so").write_text("")
    assert build._lists_stale(0.0)   # compiled for a torch that is not known
    (tmp_path / "_lists.torch").write_text(torch.__version__)
    assert not build._lists_stale(0.0)
    assert build._lists_stale(os.path.getmtime(build.LISTS) + 1)
    (tmp_path / "_lists.torch").write_text("1.0")
    assert build._lists_stale(0.0)

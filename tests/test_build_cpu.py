"""build.py without what only the extension module needs: the library is for hosts that have hipcc and
nothing else.  The compilers here are scripts that write what they are asked for."""
import builtins
import os
import stat

import pytest

from test_lds_reads_cpu import hipbuild


@pytest.fixture
def made(monkeypatch, tmp_path):
    """A build into an empty folder by a hipcc that writes its -o file: (library, extension) paths."""
    cc = tmp_path / "hipcc"
    cc.write_text('#!/bin/sh\nwhile [ "$1" != "-o" ]; do shift; done\necho made > "$2"\n')
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(cc))
    monkeypatch.setattr(hipbuild, "HERE", str(tmp_path))
    monkeypatch.setattr(hipbuild, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(hipbuild, "HOST_PATH", str(tmp_path / "host.so"))
    monkeypatch.setenv("CXX", str(cc))
    return tmp_path / "lib.so", tmp_path / "host.so"


def test_builds_both(made):
    assert hipbuild.build(verbose=False) == str(made[0])
    assert made[0].exists() and made[1].exists()


@pytest.mark.parametrize("cxx", ["/bin/false", "/nowhere/g++"])
def test_library_is_linked_where_the_extension_does_not_build(made, monkeypatch, cxx):
    monkeypatch.setenv("CXX", cxx)
    with pytest.raises(RuntimeError, match="paged_host"):
        hipbuild.build(verbose=False)
    assert made[0].exists() and not made[1].exists()


def test_library_alone_where_there_is_no_torch(made, monkeypatch, capsys):
    real = builtins.__import__

    def without_torch(name, *a, **kw):
        if name.partition(".")[0] == "torch":
            raise ModuleNotFoundError(f"No module named '{name}'", name=name)
        return real(name, *a, **kw)
    monkeypatch.setattr(builtins, "__import__", without_torch)
    assert hipbuild.build() == str(made[0])
    assert made[0].exists() and not made[1].exists()
    assert "_paged_host" in capsys.readouterr().out


def test_a_library_that_does_not_compile_fails(made, monkeypatch):
    monkeypatch.setenv("HIPCC", "/bin/false")
    with pytest.raises(RuntimeError, match="hipcc failed"):
        hipbuild.build(verbose=False)
    assert not os.path.exists(made[0])

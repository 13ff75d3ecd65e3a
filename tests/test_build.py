"""The build of the in-tree libraries, with compilers that are faked (CPU only)."""
import pytest

import usagi_b200.build as build


@pytest.fixture
def compilers(tmp_path, monkeypatch):
    """Empty output paths and a _run that records the compilers it is given; those in `broken` fail."""
    for name in ("LIB_PATH", "STAMP_PATH", "BINDING_PATH", "BINDING_STAMP_PATH"):
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    ran, broken = [], set()

    def run(cmd, verbose):
        which = "nvcc" if "nvcc" in cmd[0] else "g++"
        ran.append(which)
        if which in broken:
            raise RuntimeError(f"{which} failed (1): Python.h: No such file or directory")
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").write(which)
        return ""

    monkeypatch.setattr(build, "_run", run)
    return ran, broken


def test_builds_both_once(compilers):
    ran, _ = compilers
    build.build()
    assert sorted(ran) == ["g++", "nvcc"]
    assert build.LIB_PATH.read_text() == "nvcc" and build.BINDING_PATH.read_text() == "g++"
    build.build()
    assert len(ran) == 2


def test_the_library_needs_no_binding(compilers, capsys):
    """Without headers for the binding the kernel library is built all the same: the prefill and the C ABI
    need no more.  A binding of other sources does not stay beside it."""
    ran, broken = compilers
    broken.add("g++")
    build.BINDING_PATH.write_text("of older sources")
    assert build.build() == build.LIB_PATH
    assert build.LIB_PATH.read_text() == "nvcc" and not build.needs_build()
    assert not build.BINDING_PATH.exists()
    assert "Python.h" in capsys.readouterr().err
    with pytest.raises(RuntimeError, match="Python.h"):
        build.build_binding()
    broken.clear()
    build.build()
    assert build.BINDING_PATH.read_text() == "g++" and ran.count("nvcc") == 1


def test_a_library_that_does_not_compile_is_an_error(compilers):
    _, broken = compilers
    broken.add("nvcc")
    with pytest.raises(RuntimeError):
        build.build()

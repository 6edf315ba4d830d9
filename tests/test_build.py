"""What build.py builds, and when: the library for any host, the Python binding of the per-step operators where Python's headers are."""
import os
import sysconfig

import pytest

import __graft_entry__ as graft


@pytest.fixture
def build(monkeypatch, tmp_path):
    """The module over a folder of its own with a library and a binding that are up to date; commands are recorded instead of run."""
    b = graft._load_build_module()
    b.ran, b.LIB, b.CALLS = [], str(tmp_path / "lib.so"), str(tmp_path / "_calls.so")
    for path in (b.LIB, b.CALLS):
        open(path, "w").close()

    def run(cmd, **kw):
        b.ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("R", (), {"returncode": 0, "stdout": "", "stderr": ""})
    monkeypatch.setattr(b.subprocess, "run", run)
    return b


def test_the_binding_belongs_to_one_python(pkg):
    b = graft._load_build_module()
    assert os.path.basename(b.CALLS) == "_calls" + sysconfig.get_config_var("EXT_SUFFIX") == os.path.basename(pkg.CALLS_PATH)
    assert os.path.exists(b.CALLS) and not b.needs_build()


def test_another_pythons_binding_is_not_taken_for_this_ones(build, monkeypatch, tmp_path):
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.cpython-399-x86_64-linux-gnu.so"))
    assert build.needs_build()
    assert build.build() == build.LIB
    assert len(build.ran) == 1 and build.ran[0][0] == build.nvcc_path() and os.path.exists(build.CALLS)      # the library was there


def test_the_library_is_built_without_pythons_headers(build, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(build, "PYTHON_INCLUDE", str(tmp_path))
    os.remove(build.CALLS)
    assert not build.needs_build()
    assert build.build() == build.LIB and build.ran == []
    os.remove(build.LIB)
    assert build.needs_build() and build.build() == build.LIB
    assert {c[0] for c in build.ran} == {build.nvcc_path()} and len(build.ran) == len(build.SOURCES) + 1
    assert "Python.h" in capsys.readouterr().err and not os.path.exists(build.CALLS)


def test_operators_say_that_their_binding_is_missing(pkg, monkeypatch, tmp_path):
    monkeypatch.setattr(pkg, "_calls_module", None)
    monkeypatch.setattr(pkg, "CALLS_PATH", str(tmp_path / "_calls.so"))
    with pytest.raises(RuntimeError, match="Python.h"):
        pkg.ops.gemv_w4_grouped(1 << 20, 1 << 20, 1 << 20, 64, 256, 64)

"""The build of the optional direct binding, and the library without it."""
import os
import shutil
import subprocess
import sys
import sysconfig

import pytest

from system1_omni_b200 import build as B


@pytest.fixture
def package(tmp_path, monkeypatch):
    """build.py over a folder with nothing but the binding's source."""
    pkg = tmp_path / "pkg"
    (pkg / "binding").mkdir(parents=True)
    (tmp_path / "include").mkdir()
    shutil.copy(os.path.join(B.PKG, "binding", "fastcall.cpp"), pkg / "binding")
    shutil.copy(os.path.join(B.ROOT, "include", "s1_executor.h"), tmp_path / "include")
    monkeypatch.setattr(B, "PKG", str(pkg))
    monkeypatch.setattr(B, "ROOT", str(tmp_path))
    return pkg


def extensions(pkg):
    return sorted(p.name for p in pkg.glob("_fastcall*"))


def test_the_build_goes_on_without_python_headers(package, monkeypatch, tmp_path, capfd):
    tagged = "_fastcall" + sysconfig.get_config_var("EXT_SUFFIX")
    old = package / tagged                                       # of an earlier source
    old.write_bytes(b"")
    os.utime(old, (1, 1))
    paths = dict(sysconfig.get_paths(), include=str(tmp_path / "nothing"))
    monkeypatch.setattr(B.sysconfig, "get_paths", lambda *a, **k: paths)
    assert B.build_fastcall() is None
    assert extensions(package) == []                             # what does not match the source is not left behind
    assert "ctypes" in capfd.readouterr().err


def test_the_binding_is_built_for_its_interpreter(package):
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        pytest.skip("no Python headers")
    (package / "_fastcall.so").write_bytes(b"")                  # an untagged one of an earlier build
    out = B.build_fastcall()
    assert extensions(package) == ["_fastcall" + sysconfig.get_config_var("EXT_SUFFIX")]
    assert os.path.basename(out) == extensions(package)[0]
    when = os.path.getmtime(out)
    assert B.build_fastcall() == out and os.path.getmtime(out) == when


def test_the_library_loads_without_the_binding(cs1):
    code = ("import sys; sys.modules['system1_omni_b200._fastcall'] = None\n"
            "from system1_omni_b200 import lib as L\n"
            "f = L.load().s1_gdn_step\n"
            "assert type(f).__name__ != 'Bound' and f(*[16] * 6, 4, 4, 2, 1.0, 16, 4, 65536, None, 16, 16, 0, None) == 0\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

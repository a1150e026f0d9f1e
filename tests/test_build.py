"""What a build asks for, and what the built Python extension loads."""
import os
import shutil
import subprocess
import sys
import sysconfig

from deltazip_amd import _lib, build


def test_the_library_asks_for_hipcc_alone(monkeypatch):
    """No C++ compiler, no headers of Python's or torch's: those are the extension's."""
    lines = []

    def run(cmd, **kw):
        lines.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    assert build.build_library() == build.LIB
    assert len(lines) == len(build.SOURCES) + 1 and all(os.path.basename(cmd[0]) == "hipcc" for cmd in lines)
    assert not [w for cmd in lines for w in cmd if "torch" in w or "python" in w.lower() or "dz_host" in w]


def test_the_extension_is_this_interpreters(dzlib):
    """Its name carries the interpreter's tag: another does not import it."""
    tag = sysconfig.get_config_var("EXT_SUFFIX")
    assert tag != ".so" and build.HOST.endswith(tag) and _lib.host().__file__ == build.HOST


def test_a_copied_tree_loads_its_own_library(dzlib, tmp_path):
    for path in (build.LIB, build.HOST):
        shutil.copy(path, tmp_path)
    code = ("import sys, torch; sys.path.insert(0, sys.argv[1]); import _host; "
            "print(*sorted({l.split()[-1] for l in open('/proc/self/maps') if 'libdz_amd' in l}))")
    got = subprocess.run([sys.executable, "-c", code, str(tmp_path)], capture_output=True, text=True, cwd=tmp_path, timeout=300)
    assert got.returncode == 0, got.stderr
    assert got.stdout.split() == [str(tmp_path.resolve() / os.path.basename(build.LIB))]

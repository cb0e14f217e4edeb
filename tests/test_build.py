"""plnlp_amd/build.py's choice of what to compile, in a copy of its tree with a compiler that only writes down what it is asked for
(no device, no hipcc)."""
import importlib.util
import os
import shutil
import stat
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """(the copy's build module, the compiler calls so far)"""
    pkg = tmp_path / "plnlp_amd"
    shutil.copytree(os.path.join(ROOT, "plnlp_amd", "csrc"), pkg / "csrc")
    shutil.copy(os.path.join(ROOT, "plnlp_amd", "build.py"), pkg / "build.py")
    (tmp_path / "include").mkdir()
    shutil.copy(os.path.join(ROOT, "include", "plnlp_hip.h"), tmp_path / "include")
    log, hipcc = tmp_path / "log", tmp_path / "hipcc"
    hipcc.write_text(f'#!/bin/sh\necho "$@" >> {log}\nwhile [ "$1" != -o ]; do shift; done\n: > "$2"\n')
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(hipcc))
    old = time.time() - 1000
    for folder, _, files in os.walk(tmp_path):
        for f in files:
            os.utime(os.path.join(folder, f), (old, old))
    spec = importlib.util.spec_from_file_location("build_of_a_copy", pkg / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module, lambda: log.read_text().splitlines() if log.exists() else []


def later(path):
    os.utime(path, (time.time() + 100, time.time() + 100))


def test_what_is_compiled_again(tree):
    build, calls = tree
    build.build()
    whole = len(calls())
    assert whole > len(build.SOURCES) and not build.needs_build()       # every unit and the link
    build.build()
    assert len(calls()) == whole                                        # nothing changed
    later(os.path.join(build.CSRC, "lookup.hip"))
    assert build.needs_build()
    build.build()
    assert len(calls()) == whole + 2                                    # that unit and the link


def test_changed_flags_compile_every_unit_again(tree):
    """the flags stand in build.py: objects made with the old ones are not linked beside new ones"""
    build, calls = tree
    build.build()
    whole = len(calls())
    later(build.__file__)
    assert build.needs_build()
    build.build()
    assert len(calls()) == 2 * whole

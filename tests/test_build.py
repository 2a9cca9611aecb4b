"""The extension's build: what a changed file, changed flags or an interrupted
build make it compile again. A script takes the compiler's place."""

import os
import shutil
import stat
import subprocess

import pytest

import build_hip

COMPILER = """#!/bin/sh
# writes the file after -o; fails for a name that holds $FAIL
out=
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then out=$2; fi
  shift
done
case "$out" in *"${FAIL:-no such name}"*) exit 1;; esac
echo "$(basename "$out")" >> "$LOG"
echo built > "$out"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A copy of the sources, with files that are an hour old."""
    src = tmp_path / "hip"
    shutil.copytree(build_hip.SRC_DIR, src)
    for f in src.iterdir():
        os.utime(f, (f.stat().st_mtime - 3600,) * 2)
    hipcc = tmp_path / "hipcc"
    hipcc.write_text(COMPILER)
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IEXEC)
    log = tmp_path / "log"
    for name, value in (("SRC_DIR", src), ("BUILD_DIR", tmp_path / "build"),
                        ("OUT_SO", tmp_path / "ops.so")):
        monkeypatch.setattr(build_hip, name, str(value))
    monkeypatch.setenv("HIPCC", str(hipcc))
    monkeypatch.setenv("LOG", str(log))

    def build(**kw):
        log.write_text("")
        build_hip.build(verbose=False, **kw)
        return set(log.read_text().split())

    build.src = src
    assert len(build()) == len(build_hip.SOURCES) + 1
    for f in (tmp_path / "build").glob("*.o"):
        os.utime(f, (f.stat().st_mtime - 60,) * 2)
    os.utime(build_hip.OUT_SO, (os.stat(build_hip.OUT_SO).st_mtime - 30,) * 2)
    return build


def touch(path):
    path.write_text(path.read_text() + "\n")


def test_nothing_changed(tree):
    assert tree() == set()
    assert len(tree(force=True)) == len(build_hip.SOURCES) + 1


def test_one_source(tree):
    touch(tree.src / "distill.hip")
    assert tree() == {"distill.o", "ops.so"}


def test_header_of_a_header(tree):
    """group_norm.hip includes group_norm.h through group_norm_device.h alone."""
    touch(tree.src / "group_norm.h")
    assert tree() == {"group_norm.o", "group_norm_slab.o", "small_batch.o", "ops.so"}
    assert tree() == set()


def test_header_of_all(tree):
    touch(tree.src / "common.h")
    assert {"group_norm.o", "group_norm_slab.o", "distill.o", "bn_act.o", "ops.so"} <= tree()


def test_an_interrupted_build_with_other_flags(tree, monkeypatch):
    """Some objects have the new flags when it ends: going back compiles them
    again, too."""
    monkeypatch.setattr(build_hip, "ARCH", "other")
    monkeypatch.setenv("FAIL", "small_batch.o")
    with pytest.raises(subprocess.CalledProcessError):
        tree()
    monkeypatch.setattr(build_hip, "ARCH", "gfx950")
    monkeypatch.delenv("FAIL")
    assert len(tree()) == len(build_hip.SOURCES) + 1


def test_an_interrupted_link(tree, monkeypatch):
    touch(tree.src / "distill.hip")
    monkeypatch.setenv("FAIL", "ops.so")
    with pytest.raises(subprocess.CalledProcessError):
        tree()
    monkeypatch.delenv("FAIL")
    assert tree() == {"ops.so"}

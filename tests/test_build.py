"""What ``ravel_lm_b200.build`` compiles and links, with a stand-in for nvcc that writes its arguments."""
from __future__ import annotations

import os
import stat

import pytest

FAKE = """#!/bin/sh
out=; for a in "$@"; do [ "$prev" = -o ] && out=$a; prev=$a; done
echo "$@" > "$out"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    import ravel_lm_b200.build as b
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(FAKE)
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    src = tmp_path / "csrc"
    src.mkdir()
    (src / "common.cuh").write_text("// shared\n")
    (src / "a.cu").write_text('#include "common.cuh"\n')
    (src / "b.cu").write_text("// alone\n")
    for name, value in (("CSRC", src), ("LIB", tmp_path / "lib.so"), ("OBJ", tmp_path / "_build"),
                        ("nvcc_path", lambda: str(nvcc)), ("build_host", lambda **kw: None)):
        monkeypatch.setattr(b, name, value)
    return b, src


def age(*paths):
    """Make files older than what is built next."""
    for p in paths:
        os.utime(p, (p.stat().st_mtime - 10, p.stat().st_mtime - 10))


def test_only_stale_units_are_compiled(tree):
    b, src = tree
    age(*src.iterdir())
    b.build()
    a, other = b.obj_path(src / "a.cu"), b.obj_path(src / "b.cu")
    assert a.exists() and other.exists() and b.LIB.exists() and not b.needs_build()
    before = other.stat().st_mtime_ns
    age(a, other, b.LIB)
    before = other.stat().st_mtime_ns
    (src / "common.cuh").write_text("// changed\n")
    assert b.needs_build()
    b.build()
    assert other.stat().st_mtime_ns == before and a.stat().st_mtime_ns > before


def test_extra_flags_do_not_outlive_their_build(tree):
    """A library built with extra flags (a sweep's) is rebuilt whole by the next plain build, and no unit of it is
    linked beside plain ones after an edit of another."""
    b, src = tree
    age(*src.iterdir())
    b.build()
    objs = [b.obj_path(src / "a.cu"), b.obj_path(src / "b.cu")]
    b.build(extra_flags=["-DSWEEP=1"])
    assert all("-DSWEEP=1" in o.read_text() for o in objs)
    b.build()
    assert not any("-DSWEEP=1" in o.read_text() for o in objs)
    b.build(extra_flags=["-DSWEEP=1"])
    age(*objs, b.LIB)
    (src / "b.cu").write_text("// edited\n")
    b.build()
    assert not any("-DSWEEP=1" in o.read_text() for o in objs)

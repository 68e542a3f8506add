"""When a translation unit is compiled again: its source, a header that it includes, or its command line has changed."""
import os

import pytest

from custereomatching_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two units of one source and a header, with a compiler that only writes the object."""
    (tmp_path / "a.h").write_text("\n")
    (tmp_path / "a.hip").write_text('#include "a.h"\n')
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\necho made >> "$2"\n')
    cc.chmod(0o755)
    lib = tmp_path / "lib"
    for name, value in (("CSRC", str(tmp_path)), ("LIBDIR", str(lib)), ("LIB", str(lib / "out.so")), ("HIPCC", str(cc)),
                        ("UNITS", [("a1", "a.hip", ["-DX=1"]), ("a2", "a.hip", ["-DX=2"])]), ("MFMA", ["a2"]),
                        ("HAZARD_CHECKED", ()), ("WAIT_CHECKED", ())):
        monkeypatch.setattr(build, name, value)
    build.build()
    return tmp_path


def times(tree):
    return [(tree / "lib" / n).read_text().count("made") for n in ("a1.o", "a2.o", "out.so")]


def later(path):
    t = os.path.getmtime(path) + 10
    os.utime(path, (t, t))


def test_nothing_changed(tree):
    build.build()
    assert times(tree) == [1, 1, 1]


def test_header_changed(tree):
    later(tree / "a.h")
    build.build()
    assert times(tree) == [2, 2, 2]


def test_flags_of_all_or_of_one_unit_changed(tree, monkeypatch):
    monkeypatch.setattr(build, "MFMA_VGPR", ["-other"])
    build.build()
    assert times(tree) == [1, 2, 2]
    monkeypatch.setattr(build, "CFLAGS", [*build.CFLAGS, "-more"])
    build.build()
    assert times(tree) == [2, 3, 3]
    build.build()
    assert times(tree) == [2, 3, 3]


def test_object_without_a_record_of_its_command(tree):
    os.remove(tree / "lib" / "a1.cmd")
    build.build()
    assert times(tree) == [2, 1, 2]

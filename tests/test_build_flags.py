"""Compiler flags belong to a library's identity: another set compiles every object again and gives another stamp.  The compiler is a script
that writes its command line into its output."""
import os
import stat

import pytest

from nmrf_amd import build

FAKE = """#!/usr/bin/env python3
import os, sys
out = sys.argv[sys.argv.index("-o") + 1]
if os.path.exists(os.path.join(os.path.dirname(os.path.realpath(sys.argv[0])), "fail")) and out.endswith("b.o"):
    sys.exit(1)
open(out, "w").write(" ".join(sys.argv[1:]))
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    src = tmp_path / "csrc"
    src.mkdir()
    for name in ("a.hip", "b.hip", "build_stamp.hip", "common.h"):
        (src / name).write_text("// " + name)
    fake = tmp_path / "hipcc"
    fake.write_text(FAKE)
    fake.chmod(fake.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(fake))
    for name, value in (("CSRC", src), ("LIBDIR", tmp_path / "lib"), ("LIB", tmp_path / "lib" / "lib.so"), ("OBJDIR", tmp_path / "obj")):
        monkeypatch.setattr(build, name, str(value))
    monkeypatch.setattr(build, "_deps_mtime", lambda: 0.0)
    monkeypatch.setattr(build, "FLAGS", ["-O3", "-first"])

    def run():
        """The objects a build compiles."""
        for f in (tmp_path / "obj").glob("*.o"):
            os.utime(f, (2e9, 2e9))                                 # (newer than any source)
        was = {f.name: f.stat().st_mtime_ns for f in (tmp_path / "obj").glob("*.o")}
        build.build_library(verbose=False)
        return {f.name for f in (tmp_path / "obj").glob("*.o") if f.stat().st_mtime_ns != was.get(f.name)}
    return tmp_path, run


def test_other_flags_compile_everything_again(tree, monkeypatch):
    root, run = tree
    first = build.source_stamp()
    assert run() == {"a.o", "b.o", "build_stamp.o"} and run() == set()
    monkeypatch.setattr(build, "FLAGS", ["-O3", "-second"])
    assert build.source_stamp() != first
    assert run() == {"a.o", "b.o", "build_stamp.o"} and run() == set()
    assert all("-second" in f.read_text() for f in (root / "obj").glob("*.o"))


def test_a_build_cut_short_begins_again(tree, monkeypatch):
    root, run = tree
    run()
    monkeypatch.setattr(build, "FLAGS", ["-O3", "-second"])
    (root / "fail").write_text("")
    with pytest.raises(RuntimeError, match="hipcc failed"):
        run()
    (root / "fail").unlink()
    monkeypatch.setattr(build, "FLAGS", ["-O3", "-first"])          # back to the first flags: a.o may be of the second ones
    assert run() == {"a.o", "b.o", "build_stamp.o"}
    assert all("-first" in f.read_text() for f in (root / "obj").glob("*.o"))


def test_tools_compile_with_the_products_flags():
    """What the tools compare with the product is compiled with its flags: every hipcc line that takes a source."""
    tools = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tools")
    seen = 0
    for name in sorted(os.listdir(tools)):
        if not name.endswith((".sh", ".py")):
            continue
        with open(os.path.join(tools, name)) as f:
            for line in f:
                if "bin/hipcc" in line and (".hip" in line.replace("libnmrf_hip", "") or "src]" in line):
                    seen += 1
                    assert "$FLAGS" in line or "*FLAGS" in line, (name, line)
    assert seen >= 6

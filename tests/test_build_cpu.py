"""The in-tree library against the sources beside it (no compiler is run)."""
import os

import pytest

from dynamicpdb_amd import build_ext


@pytest.fixture
def tree(tmp_path, monkeypatch):
    (tmp_path / "a.hip").write_text('#include "a.h"\n')
    (tmp_path / "a.h").write_text("// 1\n")
    monkeypatch.setattr(build_ext, "CSRC", str(tmp_path))
    monkeypatch.setattr(build_ext, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build_ext, "STAMP", str(tmp_path / ".build_stamp"))
    return tmp_path


def test_a_library_of_other_sources_is_refused(tree, monkeypatch):
    build_ext.require_current()                      # nothing built: nothing to refuse
    (tree / "lib.so").write_text("")
    build_ext.require_current()                      # no stamp: taken as it is
    (tree / ".build_stamp").write_text(build_ext._digest())
    build_ext.require_current()
    for f in ("a.hip", "a.h"):
        before = (tree / f).read_text()
        (tree / f).write_text(before + "// 2\n")
        with pytest.raises(RuntimeError, match="rebuild"):
            build_ext.require_current()
        (tree / f).write_text(before)
        build_ext.require_current()
    monkeypatch.setattr(build_ext, "FLAGS", build_ext.FLAGS + ["-g"])
    with pytest.raises(RuntimeError, match="rebuild"):
        build_ext.require_current()


def test_benchmark_and_smoke_ask():
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
    for f in ("bench.py", "__graft_entry__.py"):
        with open(os.path.join(root, f)) as fh:
            assert "build_ext.require_current()" in fh.read()


def test_a_build_that_fails_leaves_no_stamp(tree, monkeypatch):
    """an object and a library whose compile is cut short do not look finished to the next build"""
    (tree / "lib.so").write_text("")
    (tree / ".build_stamp").write_text("x")
    (tree / "build").mkdir()
    (tree / "build" / "a.o").write_text("")
    (tree / "build" / "a.o.stamp").write_text(build_ext._digest(["a.hip"]))
    monkeypatch.setattr(build_ext, "HIPCC", "/bin/false")
    with pytest.raises(RuntimeError):
        build_ext.build(force=True)
    assert not (tree / "build" / "a.o.stamp").exists()
    (tree / "build" / "a.o.stamp").write_text(build_ext._digest(["a.hip"]))
    with pytest.raises(RuntimeError, match="link"):
        build_ext.build()                            # the object is taken, the link fails
    assert not (tree / ".build_stamp").exists()

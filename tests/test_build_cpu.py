"""The in-tree build: what makes an object or the library out of date."""
import os

import pytest

from visual_odometry_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two small sources, a header and a compiler that writes down its command lines."""
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "a.hip").write_text("a")
    (csrc / "b.hip").write_text("b")
    header = tmp_path / "h.h"
    header.write_text("h")
    monkeypatch.setattr(build, "CSRC", str(csrc))
    monkeypatch.setattr(build, "headers", lambda: [str(header)])
    monkeypatch.setattr(build, "OBJDIR", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "LIBDIR", str(tmp_path / "lib"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib" / "lib.so"))
    monkeypatch.setattr(build, "CFLAGS", ["-O3"])
    monkeypatch.setattr(build, "hipcc", lambda: "hipcc")
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")

        class Result:
            returncode, stdout, stderr = 0, "", ""
        return Result
    monkeypatch.setattr(build.subprocess, "run", run)

    def builds(**kw):
        """Sources compiled and links made by one call."""
        del ran[:]
        build.build_library(**kw)
        return sorted(os.path.basename(c[c.index("-c") + 1]) for c in ran if "-c" in c), sum("-shared" in c for c in ran)
    builds.csrc, builds.header = csrc, header
    return builds


def later(path):
    t = os.path.getmtime(path) + 10
    os.utime(path, (t, t))


def test_an_unchanged_tree_is_not_built_again(tree):
    assert tree() == (["a.hip", "b.hip"], 1)
    assert tree() == ([], 0)


def test_a_changed_source_or_header_is_compiled(tree):
    tree()
    later(tree.csrc / "a.hip")
    assert tree() == (["a.hip"], 1)
    later(tree.header)
    assert tree()[0] in (["a.hip", "b.hip"],)


def test_changed_flags_compile_everything(tree, monkeypatch):
    tree()
    monkeypatch.setattr(build, "CFLAGS", ["-O3", "-Xclang", "-target-feature"])
    assert tree() == (["a.hip", "b.hip"], 1)
    assert tree() == ([], 0)
    monkeypatch.setattr(build, "hipcc", lambda: "/another/hipcc")
    assert tree() == (["a.hip", "b.hip"], 1)


def test_objects_of_unknown_flags_are_compiled(tree):
    """A tree built before command lines were written down: objects and library are newer than everything, and alone."""
    tree()
    for d in (build.OBJDIR, build.LIBDIR):
        for f in os.listdir(d):
            if not f.endswith((".o", ".so")):
                os.remove(os.path.join(d, f))
    assert tree() == (["a.hip", "b.hip"], 1)


def test_a_forced_build_compiles_everything(tree):
    tree()
    assert tree(force=True) == (["a.hip", "b.hip"], 1)


def test_a_source_taken_away_is_linked_out(tree):
    tree()
    os.remove(tree.csrc / "b.hip")
    assert tree() == ([], 1)

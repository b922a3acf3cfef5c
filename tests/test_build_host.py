"""The build's reuse of objects: compiled anew when a source is newer or the flags are others; the compiler is a stand-in that writes its arguments."""
import os
import time

import pytest


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from semiuhpe_amd import build as B
    csrc = tmp_path / "pkg" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "suhpe.h").write_text("")
    for name in ("a.hip", "b.hip"):
        (csrc / name).write_text(name)
    (csrc / "c.h").write_text("")
    past = time.time() - 100
    for f in [tmp_path / "include" / "suhpe.h", *csrc.iterdir()]:
        os.utime(f, (past, past))
    monkeypatch.setattr(B, "HERE", str(tmp_path / "pkg"))
    monkeypatch.setattr(B, "CSRC", str(csrc))
    monkeypatch.setattr(B, "LIB", str(csrc / "lib.so"))
    monkeypatch.setattr(B, "SOURCES", ["a.hip", "b.hip"])
    monkeypatch.setattr(B, "_hipcc", lambda: "hipcc")
    ran = []

    def run(cmd):
        if "-c" in cmd:
            ran.append(os.path.basename(cmd[cmd.index("-c") + 1]))
            if ran[-1] in fail:
                raise RuntimeError("compile error")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(" ".join(cmd))
    fail = []
    monkeypatch.setattr(B.subprocess, "check_call", run)
    return B, csrc, ran, fail


def test_objects_of_other_flags_are_not_linked(tree, monkeypatch):
    B, csrc, ran, _ = tree
    B.build(verbose=False)
    assert sorted(ran) == ["a.hip", "b.hip"]
    ran.clear()
    B.build(verbose=False)
    assert ran == []
    monkeypatch.setattr(B, "FLAGS", B.FLAGS[:-4])
    B.build(verbose=False)
    assert sorted(ran) == ["a.hip", "b.hip"]
    ran.clear()
    (csrc / "build" / "flags.txt").unlink()                 # objects of a tree that kept no record
    B.build(verbose=False)
    assert sorted(ran) == ["a.hip", "b.hip"]
    ran.clear()
    (csrc / "b.hip").write_text("newer")
    os.utime(csrc / "b.hip", (time.time() + 5, time.time() + 5))
    B.build(verbose=False)
    assert ran == ["b.hip"]


def test_a_build_that_failed_half_way_is_taken_up(tree, monkeypatch):
    B, csrc, ran, fail = tree
    B.build(verbose=False)
    monkeypatch.setattr(B, "FLAGS", B.FLAGS + ["-DX"])
    fail.append("b.hip")
    with pytest.raises(RuntimeError):
        B.build(verbose=False)
    ran.clear()
    fail.clear()
    B.build(verbose=False)
    assert sorted(ran) == ["a.hip", "b.hip"]                # the old b.o is not linked beside the new a.o

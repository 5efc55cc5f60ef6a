"""The incremental build of the kernel library, with a compiler that only notes what it is asked for."""
import os
import subprocess

import pytest

from distributed_tensorflow_amd.ops import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two sources and a header; -> (folder, list of the files made by each call of the compiler)."""
    made, fail = [], set()
    for n in ("one.hip", "two.hip", "common.h"):
        (tmp_path / n).write_text("// " + n)
        os.utime(tmp_path / n, (1, 1))
    for name, at in (("CSRC", tmp_path), ("OBJ", tmp_path / "obj"), ("LIB", tmp_path / "lib.so")):
        monkeypatch.setattr(B, name, str(at))
    monkeypatch.setattr(B, "FLAGS", ["-O3"])
    monkeypatch.setattr(B, "EXTRA_FLAGS", {})

    def compiler(cmd, **kw):
        out = os.path.basename(cmd[cmd.index("-o") + 1])
        made.append(out)
        if out in fail:
            return subprocess.CompletedProcess(cmd, 1, "", "failed")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(" ".join(cmd))
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B.subprocess, "run", compiler)

    def build(**kw):
        del made[:]
        B.build(verbose=False, **kw)
        return sorted(made)

    build.fail, build.made = fail, made
    return tmp_path, build


def test_what_did_not_change_is_not_built(tree):
    _, build = tree
    assert build() == ["lib.so", "one.o", "two.o"]
    assert build() == [] and build(force=True) == ["lib.so", "one.o", "two.o"] and build() == []


def test_other_flags_build_again(tree, monkeypatch):
    at, build = tree
    build()
    monkeypatch.setattr(B, "FLAGS", ["-O3", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"])
    assert build() == ["lib.so", "one.o", "two.o"]
    for o in ("one.o", "two.o"):
        assert "-packed-fp32-ops" in (at / "obj" / o).read_text()
    monkeypatch.setattr(B, "EXTRA_FLAGS", {"two.hip": ["-fno-honor-nans"]})
    assert build() == ["lib.so", "two.o"]
    monkeypatch.setattr(B, "HIPCC", "another-compiler")
    assert build() == ["lib.so", "one.o", "two.o"] and build() == []


def test_objects_of_unknown_flags_are_built_again(tree):
    """A tree that was built before commands were recorded."""
    at, build = tree
    build()
    for f in os.listdir(at / "obj"):
        if f.endswith(".cmd"):
            os.remove(at / "obj" / f)
    assert build() == ["lib.so", "one.o", "two.o"]


def test_sources_headers_and_temporary_files(tree):
    at, build = tree
    build()
    os.utime(at / "one.hip", None)
    for o in ("one.o", "two.o"):
        os.utime(at / "obj" / o, (2, 2))
    os.utime(at / "one.hip", (3, 3))
    assert build() == ["lib.so", "one.o"]
    assert build(save_temps=True, force=True) == ["lib.so", "one.o", "two.o"] and build() == []
    (at / "three.hip").write_text("")
    os.utime(at / "three.hip", (1, 1))
    assert build() == ["lib.so", "three.o"]
    os.remove(at / "three.hip")
    assert build() == ["lib.so"]                                # (its code leaves the library)
    os.utime(at / "common.h", None)
    for o in ("one.o", "two.o"):
        os.utime(at / "obj" / o, (2, 2))
    assert build() == ["lib.so", "one.o", "two.o"]


def test_a_failed_build_is_taken_up_again(tree):
    at, build = tree
    build()
    build.fail.add("lib.so")
    with pytest.raises(RuntimeError, match="link failed"):
        build(force=True)
    build.fail.clear()
    assert build() == ["lib.so"]
    build.fail.add("two.o")
    with pytest.raises(RuntimeError, match="two.hip"):
        build(force=True)
    (at / "obj" / "two.o").write_text("half a file")            # newer than its source
    build.fail.clear()
    assert "two.o" in build()

"""When an object of the kernel library is built again.  A stand-in for the compiler writes its own arguments into the file it is asked for."""
import os
import stat
import sys

import pytest

from internevo_amd import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    (tmp_path / "csrc").mkdir()
    for name in ("one.hip", "two.hip"):
        (tmp_path / "csrc" / name).write_text("// " + name)
    (tmp_path / "csrc" / "common.h").write_text("")
    compiler = tmp_path / "hipcc"
    compiler.write_text(f"#!{sys.executable}\nimport sys\na = sys.argv\nopen(a[a.index('-o') + 1], 'w').write(' '.join(a[1:]))\nopen({str(tmp_path / 'calls')!r}, 'a').write(a[-3] + '\\n')\n")
    compiler.chmod(compiler.stat().st_mode | stat.S_IXUSR)
    for name, value in (("CSRC", tmp_path / "csrc"), ("OBJ", tmp_path / "csrc" / "build"), ("LIB", tmp_path / "csrc" / "lib.so")):
        monkeypatch.setattr(B, name, str(value))
    monkeypatch.setattr(B, "_hipcc", lambda: str(compiler))
    monkeypatch.setattr(B, "_headers_mtime", lambda: 0.0)
    past = 1_000_000_000
    for name in ("one.hip", "two.hip"):
        os.utime(tmp_path / "csrc" / name, (past, past))

    def built():
        """names of the sources that a call compiles"""
        (tmp_path / "calls").write_text("")
        B.build(verbose=False)
        return sorted(os.path.basename(c) for c in (tmp_path / "calls").read_text().split() if c.endswith(".hip"))

    return tmp_path, built


def test_unchanged_sources_are_compiled_once(tree):
    _, built = tree
    assert built() == ["one.hip", "two.hip"] and built() == []


def test_other_flags_compile_everything_again(tree, monkeypatch):
    _, built = tree
    built()
    monkeypatch.setattr(B, "FLAGS", [*B.FLAGS, "-DOTHER"])
    assert built() == ["one.hip", "two.hip"] and built() == []
    assert all("-DOTHER" in open(os.path.join(B.OBJ, o)).read() for o in ("one.o", "two.o"))


def test_other_flags_of_one_source_compile_that_one(tree, monkeypatch):
    _, built = tree
    built()
    monkeypatch.setattr(B, "EXTRA_FLAGS", {"two.hip": ["-DOTHER"]})
    assert built() == ["two.hip"] and built() == []


def test_an_object_of_unknown_flags_is_compiled_again(tree):
    tmp_path, built = tree
    built()
    obj = tmp_path / "csrc" / "build" / "one.o"
    for f in (tmp_path / "csrc" / "build").iterdir():
        if f.name.startswith("one.") and f != obj:
            f.unlink()
    assert obj.exists() and built() == ["one.hip"]


def test_a_changed_source_is_compiled_again(tree):
    tmp_path, built = tree
    built()
    os.utime(tmp_path / "csrc" / "one.hip", (4_000_000_000, 4_000_000_000))
    assert built() == ["one.hip"]


def test_packed_fp32_arithmetic_is_off_for_every_source():
    at = B.FLAGS.index("-packed-fp32-ops")
    assert B.FLAGS[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]


def test_two_programs_build_one_after_the_other(tree):
    """The second waits and finds everything up to date, where it used to remove objects that the first was linking."""
    import multiprocessing
    import time

    tmp_path, _ = tree
    real, start = B._compile, multiprocessing.get_context("fork")

    def slow(src, force):
        time.sleep(0.3)
        return real(src, force)

    B._compile = slow
    try:
        (tmp_path / "calls").write_text("")
        ps = [start.Process(target=B.build, kwargs=dict(verbose=False)) for _ in range(2)]
        [p.start() for p in ps]
        [p.join(60) for p in ps]
    finally:
        B._compile = real
    assert [p.exitcode for p in ps] == [0, 0]
    assert sorted(os.path.basename(c) for c in (tmp_path / "calls").read_text().split() if c.endswith(".hip")) == ["one.hip", "two.hip"]

"""The in-tree build (similaripy_amd/_build.py) with a stand-in for the compiler that writes its command into what it makes."""
from __future__ import annotations

import os
import sys

import pytest

from similaripy_amd import _build


@pytest.fixture
def project(tmp_path, monkeypatch):
    """Two units, one header of each, a compiler that copies its own command into the output file."""
    cc = tmp_path / "cc.py"
    cc.write_text("#!%s\nimport sys\nargs = sys.argv[1:]\nout = args[args.index('-o') + 1]\n"
                  "text = ' '.join(a for a in args if a.startswith('-D') or a.startswith('-f'))\n"
                  "ins = [open(a).read() for a in args if a.endswith('.o') and a != out]\n"
                  "open(out, 'w').write('|'.join(ins) if ins else text)\n" % sys.executable)
    cc.chmod(0o755)
    units = {}
    for name in ("a", "b"):
        src, header = tmp_path / (name + ".hip"), tmp_path / (name + ".hpp")
        src.write_text("")
        header.write_text("")
        units[src] = [header]
    lib = tmp_path / "lib"
    for name, value in (("UNITS", units), ("SOURCES", list(units)), ("HEADERS", [h for hs in units.values() for h in hs]), ("LIB_DIR", lib),
                        ("LIB_PATH", lib / "libx.so"), ("HIPCC_FLAGS", ["-fone"])):
        monkeypatch.setattr(_build, name, value)
    monkeypatch.setenv("HIPCC", str(cc))
    monkeypatch.delenv("SIMILARIPY_AMD_HIPCC_EXTRA", raising=False)
    return tmp_path


def age(path, seconds):
    t = path.stat().st_mtime - seconds
    os.utime(path, (t, t))


def built(project):
    _build.build()
    return (project / "lib" / "libx.so").read_text()


def make_old(project):
    """Everything there was made some time ago, in its order."""
    for p in sorted(project.rglob("*"), key=lambda p: p.stat().st_mtime):
        if p.is_file():
            age(p, 100)


def test_a_build_after_other_flags_takes_nothing_from_it(project, monkeypatch):
    assert built(project) == "-fone|-fone"
    monkeypatch.setenv("SIMILARIPY_AMD_HIPCC_EXTRA", "-DX=1")
    assert _build.is_stale() and built(project) == "-fone -DX=1|-fone -DX=1"
    assert not _build.is_stale()
    make_old(project)
    monkeypatch.delenv("SIMILARIPY_AMD_HIPCC_EXTRA")
    (project / "b.hpp").write_text("changed")
    assert _build.is_stale() and built(project) == "-fone|-fone"                   # (not: unit a still with -DX=1)
    make_old(project)
    monkeypatch.setattr(_build, "HIPCC_FLAGS", ["-ftwo"])
    assert _build.is_stale() and built(project) == "-ftwo|-ftwo"


def test_only_what_changed_is_compiled(project, monkeypatch):
    built(project)
    make_old(project)
    before = {p.name: p.stat().st_mtime for p in (project / "lib").glob("*.o")}
    assert not _build.is_stale() and built(project) == "-fone|-fone"
    (project / "b.hpp").write_text("changed")
    assert _build.is_stale() and built(project) == "-fone|-fone" and not _build.is_stale()
    after = {p.name: p.stat().st_mtime for p in (project / "lib").glob("*.o")}
    assert after["a.o"] == before["a.o"] and after["b.o"] > before["b.o"]


def test_a_library_without_its_objects_is_used_as_it_is(project):
    """A copy of the tree may hold the library alone: it is not stale, and a later build compiles all of it."""
    built(project)
    for p in (project / "lib").glob("*.o*"):
        p.unlink()
    assert not _build.is_stale()
    (project / "a.hpp").write_text("changed")
    assert built(project) == "-fone|-fone"


def test_an_object_of_unknown_flags_is_compiled_again(project):
    built(project)
    (project / "lib" / "a.o").write_text("-fold")
    for p in (project / "lib").glob("*.cmd"):
        p.unlink()
    make_old(project)
    assert not _build.is_stale()                        # (the library alone says nothing of its flags: its time counts)
    (project / "b.hpp").write_text("changed")
    assert built(project) == "-fone|-fone"

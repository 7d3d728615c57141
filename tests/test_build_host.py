"""The build: the product's library does not depend on what only tests and records need, and a failed
build leaves the library of the last good one alone.  A stand-in compiler, no GPU."""

import os
import stat
import sys

import pytest

import __graft_entry__ as entry
from kfold_amd import build

# writes its -o file; fails for sources that hold FAIL, and at assembly listings where NO_LISTING is set
COMPILER = """#!/bin/sh
out=; listing=; bad=
while [ $# -gt 0 ]; do
    case "$1" in
        -o) out=$2; shift;;
        -S) listing=1;;
        *.hip) grep -q FAIL "$1" && bad=1;;
    esac
    shift
done
[ -n "$bad" ] && { echo "cannot compile" >&2; exit 1; }
[ -n "$listing" ] && { [ -n "$NO_LISTING" ] && exit 3; exit 0; }
echo new > "$out"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    cc = tmp_path / "cc"
    cc.write_text(COMPILER)
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "a.hip").write_text("one\n")
    (csrc / "b.hip").write_text("two\n")
    for name, value in (("HIPCC", str(cc)), ("CSRC", csrc), ("LIB", tmp_path / "lib.so"), ("ISA_JSON", tmp_path / "isa.json"),
                        ("RESOURCES_JSON", tmp_path / "res.json")):
        monkeypatch.setattr(build, name, value)
    return tmp_path


def test_a_build_writes_library_and_records(tree):
    assert build.build().read_text() == "new\n"
    assert build.ISA_JSON.read_text() == "{}\n" and build.RESOURCES_JSON.exists()


def test_library_without_listings(tree, monkeypatch, capsys):
    """Assembly listings that cannot be made cost the records, not the library; records of an older
    build do not stay."""
    monkeypatch.setenv("NO_LISTING", "1")
    build.ISA_JSON.write_text("old")
    build.RESOURCES_JSON.write_text("old")
    assert build.build().read_text() == "new\n"
    assert not build.ISA_JSON.exists() and not build.RESOURCES_JSON.exists()
    assert "records" in capsys.readouterr().err


def test_failed_source_is_named_and_the_old_library_stays(tree):
    (build.CSRC / "b.hip").write_text("FAIL\n")
    build.LIB.write_text("old\n")
    with pytest.raises(RuntimeError, match="(?s)b.hip.*exit status 1.*cannot compile"):
        build.build()
    assert build.LIB.read_text() == "old\n"


@pytest.mark.parametrize("missing", [False, True])
def test_entry_builds_without_the_host_model(tree, monkeypatch, capsys, missing):
    """A host model that does not compile, or a tree without the tests, leaves build() with its library."""
    lib = build.ROOT / "libkfold_hip.so"
    monkeypatch.setattr(build, "build", lambda verbose=False: lib)
    if missing:
        monkeypatch.setitem(sys.modules, "tests.hostsim", None)
    else:
        from tests.hostsim import build as host

        def refuse(force=False):
            raise RuntimeError("host build failed for x")
        monkeypatch.setattr(host, "build", refuse)
    entry.build()
    err = capsys.readouterr().err
    assert "host model" in err and ("host build failed for x" in err or missing)
    assert os.path.exists(lib)

"""The build compiles what its sources or its command lines ask for (a stand-in for the compiler writes down how it was called)."""
import os
import stat

import pytest

from iggt_official_amd import build_ext as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    log = tmp_path / "log"
    cc = tmp_path / "cc"
    cc.write_text(f'#!/bin/sh\necho "$@" >> {log}\nfor a in "$@"; do [ "$last" = -o ] && : > "$a"; last="$a"; done\n')
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    src = tmp_path / "csrc"
    src.mkdir()
    for name in ("a.hip", "b.hip", "attention_v3.hip"):
        (src / name).write_text("")
    for name, value in dict(CSRC=str(src), LIB_DIR=str(tmp_path / "lib"), LIB=str(tmp_path / "lib" / "x.so"), HIPCC=str(cc), FLAGS=["-O3"], PER_FILE_FLAGS={}).items():
        monkeypatch.setattr(B, name, value)

    def calls(**kw):
        log.write_text("")
        B.build(verbose=False, **kw)
        return [os.path.basename(line.split(" -o ")[1].split()[0]) for line in log.read_text().splitlines()]

    return src, calls, monkeypatch


def test_a_change_of_flags_compiles_again(tree):
    src, calls, patch = tree
    every = ["a.o", "attention_v3.o", "b.o", "x.so"]
    assert sorted(calls()) == every and calls() == []
    patch.setattr(B, "FLAGS", ["-O3", "-DNEW"])
    assert sorted(calls()) == every and calls() == []
    patch.setattr(B, "PER_FILE_FLAGS", {"b.hip": ["-g"]})
    assert calls() == ["b.o", "x.so"] and calls() == []
    assert sorted(calls(force=True)) == every


def test_a_source_that_is_gone_leaves_the_library(tree):
    src, calls, _ = tree
    calls()
    (src / "a.hip").unlink()
    assert calls() == ["x.so"] and calls() == []


def test_a_failed_compilation_is_tried_again(tree):
    src, calls, patch = tree
    good = B.HIPCC
    patch.setattr(B, "HIPCC", "/bin/false")
    with pytest.raises(RuntimeError):
        calls()
    patch.setattr(B, "HIPCC", good)
    assert len(calls()) == 4

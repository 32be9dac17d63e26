"""Which objects build.build() compiles again (a stand-in for the compiler notes its calls)."""
from __future__ import annotations

import os
import stat

import pytest


@pytest.fixture()
def tree(tmp_path, monkeypatch):
    from multimodalstudio_amd import build as b
    csrc, include, objects = tmp_path / "csrc", tmp_path / "include", tmp_path / "build"
    for d in (csrc, include):
        d.mkdir()
    (csrc / "one.hip").write_text("1")
    (csrc / "two.hip").write_text("2")
    (include / "api.h").write_text("0")
    log = tmp_path / "log"
    cc = tmp_path / "cc"
    cc.write_text(f'#!/bin/sh\nfor a; do last="$a"; [ "$prev" = -o ] && out="$a"; prev="$a"; done\n'
                  f'echo "$out" >> {log}\n[ -e {tmp_path}/broken ] && exit 1\ntouch "$out"\n')
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for name, value in (("CSRC", csrc), ("INCLUDE", include), ("BUILD", objects), ("LIB", tmp_path / "lib.so"),
                        ("HIPCC", str(cc)), ("CFLAGS", ["-O3"])):
        monkeypatch.setattr(b, name, value)

    def run():
        log.write_text("")
        b.build()
        return sorted(os.path.basename(x) for x in log.read_text().split())
    return b, tmp_path, run


def _later(path):
    t = path.stat().st_mtime + 100
    os.utime(path, (t, t))


def test_what_is_compiled_again(tree):
    b, root, run = tree
    assert run() == ["lib.so", "one.o", "two.o"] and run() == []
    for o in root.glob("build/*.o"):
        _later(o)
    _later(root / "lib.so")
    _later(root / "csrc" / "one.hip")
    _later(root / "csrc" / "one.hip")
    assert "one.o" in run() and "two.o" not in run()


def test_another_flag_or_compiler_compiles_all(tree, monkeypatch):
    b, root, run = tree
    run()
    monkeypatch.setattr(b, "CFLAGS", ["-O3", "-DOTHER"])
    assert [x for x in run() if x.endswith(".o")] == ["one.o", "two.o"] and run() == []
    other = root / "cc2"
    other.write_text((root / "cc").read_text())
    other.chmod((root / "cc").stat().st_mode)
    monkeypatch.setattr(b, "HIPCC", str(other))
    assert [x for x in run() if x.endswith(".o")] == ["one.o", "two.o"]


def test_a_failed_compile_is_not_taken_for_done(tree, monkeypatch):
    b, root, run = tree
    run()
    monkeypatch.setattr(b, "CFLAGS", ["-O2"])
    (root / "broken").write_text("")
    with pytest.raises(RuntimeError, match="hipcc failed"):
        run()
    (root / "broken").unlink()
    monkeypatch.setattr(b, "CFLAGS", ["-O3"])
    assert [x for x in run() if x.endswith(".o")] == ["one.o", "two.o"]

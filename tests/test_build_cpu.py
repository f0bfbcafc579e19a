"""What a build takes over from an earlier one: objects of the same sources, made with the same compiler and flags, and no others."""
import os

import pytest

from tts_amd import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two sources and a compiler that writes down what it is asked for."""
    (tmp_path / "csrc").mkdir()
    for name in ("one.hip", "two.cpp"):
        (tmp_path / "csrc" / name).write_text("// nothing\n")
    log = tmp_path / "log"
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ $# -gt 1 ]; do [ "$1" = -o ] && out=$2; shift; done\n[ -e %s ] && exit 1\necho x > $out\n' % (log, tmp_path / "broken"))
    cc.chmod(0o755)
    monkeypatch.setattr(build, "HIPCC", str(cc))
    monkeypatch.setattr(build, "CSRC", str(tmp_path / "csrc"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))

    def run():
        if log.exists():
            log.unlink()
        build.build_lib()
        lines = log.read_text().splitlines() if log.exists() else []
        return sum(" -c " in line for line in lines), sum("-shared" in line for line in lines)

    return tmp_path, run


def test_objects_of_other_flags_are_made_again(tree, monkeypatch):
    tmp, run = tree
    assert run() == (2, 1)
    assert run() == (0, 0)
    flags = list(build.FLAGS)
    monkeypatch.setattr(build, "FLAGS", flags + ["-DX=1"])
    assert run() == (2, 1)
    assert run() == (0, 0)
    monkeypatch.setattr(build, "FLAGS", flags)
    assert run() == (2, 1)
    other = tmp / "cc2"
    other.write_text((tmp / "cc").read_text())
    other.chmod(0o755)
    monkeypatch.setattr(build, "HIPCC", str(other))
    assert run() == (2, 1)
    later = os.path.getmtime(tmp / "obj" / "one.o") + 10
    os.utime(tmp / "csrc" / "one.hip", (later, later))
    assert run()[0] == 1


def test_a_build_that_failed_leaves_nothing_to_take_over(tree, monkeypatch):
    """New flags, a compiler that stops: the next build makes everything, whatever objects lie there."""
    tmp, run = tree
    assert run() == (2, 1)
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-DX=1"])
    (tmp / "broken").write_text("")
    with pytest.raises(RuntimeError):
        run()
    (tmp / "broken").unlink()
    assert run() == (2, 1)


def test_objects_from_before_there_was_a_record_are_made_again(tree):
    tmp, run = tree
    run()
    for name in os.listdir(tmp / "obj"):
        if not name.endswith(".o"):
            os.remove(tmp / "obj" / name)
    assert run() == (2, 1)

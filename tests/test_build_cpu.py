"""Two processes that build the library at once (the ranks of a job that
starts on a fresh checkout) each put a whole file in place.  A script stands
for the compiler."""
import os
import shutil
import threading
from pathlib import Path

import pytest

from hbfsim_b200 import build


@pytest.fixture
def fake(tmp_path, monkeypatch):
    compiler = tmp_path / "compiler"
    compiler.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\nprintf made > "$2"\n')
    compiler.chmod(0o755)
    package = tmp_path / "package"
    package.mkdir()
    monkeypatch.setattr(build, "NVCC", str(compiler))
    monkeypatch.setattr(build, "LIB", package / "libhbfsim_b200.so")
    return package


def test_builds_at_once_do_not_share_a_file(fake, monkeypatch):
    both = threading.Barrier(2, timeout=30)
    copy, targets, errors = shutil.copyfile, [], []

    def copy_and_wait(src, dst, **more):
        copy(src, dst, **more)
        targets.append(os.fspath(dst))
        both.wait()  # the other one has written its file as well

    def run():
        try:
            build.build(force=True)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    monkeypatch.setattr(shutil, "copyfile", copy_and_wait)
    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors
    assert len(set(targets)) == 2
    assert os.listdir(fake) == ["libhbfsim_b200.so"]
    assert build.LIB.read_text() == "made" and os.access(build.LIB, os.X_OK)


def test_a_failed_copy_leaves_the_old_library(fake, monkeypatch):
    build.LIB.write_text("old")

    def fails(src, dst, **more):
        Path(dst).write_text("half")
        raise OSError("no space")

    monkeypatch.setattr(shutil, "copyfile", fails)
    with pytest.raises(OSError):
        build.build(force=True)
    assert os.listdir(fake) == ["libhbfsim_b200.so"] and build.LIB.read_text() == "old"

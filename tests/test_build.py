"""Builds that several callers ask for at once, with a compiler that only writes down what it is asked for."""
import os
import stat
import threading

import pytest

import warpdecode_b200 as wd

COMPILER = """#!/usr/bin/env python3
import os, sys, time
out = sys.argv[sys.argv.index("-o") + 1]
if os.environ.get("FAKE_FAILS") and out.endswith(os.environ["FAKE_FAILS"]):
    sys.exit("no")
with open(os.environ["FAKE_LOG"], "a") as f:
    f.write(os.path.basename(out) + "\\n")
fd = os.open(out, os.O_CREAT | os.O_EXCL | os.O_WRONLY)      # another one that writes the same file is a failure
os.write(fd, b"half ")
time.sleep(0.2)
os.write(fd, b"whole")
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    src = tmp_path / "csrc"
    src.mkdir()
    files = [str(src / n) for n in ("one.cu", "two.cu")]
    for f in files:
        open(f, "w").write("// nothing")
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(COMPILER)
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    log = tmp_path / "log"
    for name, value in (("HERE", str(tmp_path)), ("LIB_PATH", str(tmp_path / "lib.so")), ("SOURCES", files), ("UNITS", {"one": files[:1], "two": files[1:]})):
        monkeypatch.setattr(wd, name, value)
    monkeypatch.setenv("NVCC", str(nvcc))
    monkeypatch.setenv("FAKE_LOG", str(log))
    return tmp_path


def test_callers_at_once_build_once(tree):
    failed = []

    def call():
        try:
            wd.build()
            assert (tree / "lib.so").read_bytes() == b"half whole"
        except BaseException as e:
            failed.append(e)

    callers = [threading.Thread(target=call) for _ in range(4)]
    for t in callers:
        t.start()
    for t in callers:
        t.join()
    assert not failed, failed
    assert sorted(x.replace(".new", "") for x in (tree / "log").read_text().split()) == ["lib.so", "one.o", "two.o"]


def test_only_what_is_older_than_its_source_is_built_again(tree):
    wd.build()
    later = os.path.getmtime(tree / "lib.so") + 5
    os.utime(tree / "csrc" / "two.cu", (later, later))
    (tree / "log").write_text("")
    wd.build()
    assert sorted(x.replace(".new", "") for x in (tree / "log").read_text().split()) == ["lib.so", "two.o"]


def test_a_failure_leaves_no_half_of_an_object(tree, monkeypatch):
    monkeypatch.setenv("FAKE_FAILS", "two.o.new")
    with pytest.raises(RuntimeError):
        wd.build()
    assert not (tree / "lib.so").exists() and not (tree / "build" / "two.o").exists()
    monkeypatch.delenv("FAKE_FAILS")
    wd.build()
    assert (tree / "lib.so").read_bytes() == b"half whole"

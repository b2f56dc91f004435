"""The library's build keeps an object only if it was compiled from the present sources with the present flags, also
after a build that failed or was cut off (the compiler replaced by a script)."""
import importlib.util
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COMPILER = """#!/bin/sh
# writes its arguments as the output; "broken" sources fail after half of it
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then out=$2; fi
  all="$all $1"
  last=$1
  shift
done
case "$all" in *" -c "*)
  if grep -q broken "$last"; then echo half > "$out"; exit 1; fi;;
esac
echo "$all" > "$out"
"""


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(ROOT, "mlu-ops_b200", "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(COMPILER)
    nvcc.chmod(0o755)
    monkeypatch.setenv("NVCC", str(nvcc))
    monkeypatch.delenv("MLUOP_B200_NVCC_FLAGS", raising=False)
    for name in ("a.cu", "b.cu"):
        (tmp_path / name).write_text("fine")
    (tmp_path / "h.h").write_text("")
    monkeypatch.setattr(m, "CSRC", str(tmp_path))
    monkeypatch.setattr(m, "LIB_DIR", str(tmp_path / "lib"))
    monkeypatch.setattr(m, "OBJ_DIR", str(tmp_path / "lib" / "obj"))
    monkeypatch.setattr(m, "LIB", str(tmp_path / "lib" / "x.so"))
    monkeypatch.setattr(m, "sources", lambda: [str(tmp_path / "a.cu"), str(tmp_path / "b.cu")])
    monkeypatch.setattr(m, "headers", lambda: [str(tmp_path / "h.h")])
    m.tmp = tmp_path
    return m


def objects(m):
    return {n: open(os.path.join(m.OBJ_DIR, n)).read() for n in ("a.cu.o", "b.cu.o")}


def age(m):
    """Everything that is there becomes a minute older, so that what is written next is newer."""
    for folder, _, names in os.walk(str(m.tmp)):
        for n in names:
            t = os.path.getmtime(os.path.join(folder, n)) - 60
            os.utime(os.path.join(folder, n), (t, t))


def test_a_failed_build_with_other_flags_leaves_nothing_behind(build, monkeypatch):
    build.build(force=True)
    age(build)
    (build.tmp / "b.cu").write_text("broken")
    monkeypatch.setenv("MLUOP_B200_NVCC_FLAGS", "-DEXPERIMENT")
    with pytest.raises(subprocess.CalledProcessError):
        build.build()
    age(build)
    (build.tmp / "b.cu").write_text("fine")
    monkeypatch.delenv("MLUOP_B200_NVCC_FLAGS")
    build.build()
    assert not any("EXPERIMENT" in text or text == "half\n" for text in objects(build).values())
    assert all(n in open(build.LIB).read() for n in objects(build))


def test_half_an_object_is_not_kept(build):
    build.build(force=True)
    age(build)
    (build.tmp / "b.cu").write_text("broken")
    with pytest.raises(subprocess.CalledProcessError):
        build.build()
    assert objects(build)["b.cu.o"] != "half\n"


def test_objects_are_kept_and_rebuilt_as_needed(build):
    build.build(force=True)
    age(build)
    (build.tmp / "b.cu").write_text("fine too")
    stamp = os.path.getmtime(os.path.join(build.OBJ_DIR, "a.cu.o"))
    build.build()
    assert os.path.getmtime(os.path.join(build.OBJ_DIR, "a.cu.o")) == stamp
    assert os.path.getmtime(os.path.join(build.OBJ_DIR, "b.cu.o")) > stamp
    assert build.up_to_date()
    assert sorted(os.listdir(build.OBJ_DIR)) == ["a.cu.o", "b.cu.o", "flags.txt"]

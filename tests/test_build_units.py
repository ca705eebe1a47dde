"""When an object is compiled anew, with a stand-in for nvcc."""
import importlib.util
import os
import shutil

import pytest

from conftest import entry

STAND_IN = """#!/bin/sh
while [ $# -gt 0 ]; do
  case "$1" in -o) out="$2"; shift;; -MF) list="$2"; shift;; *.cu) unit="$1";; esac
  shift
done
echo "$unit" >> "$CALLS"
echo new > "$out"
printf '%s: %s \\\\\\n %s/a.cuh\\n' "$out" "$unit" "$(dirname "$unit")" > "$list"
"""


@pytest.fixture()
def tree(tmp_path, monkeypatch):
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(STAND_IN)
    nvcc.chmod(0o755)
    monkeypatch.setenv("NVCC", str(nvcc))
    monkeypatch.setenv("CALLS", str(tmp_path / "calls"))
    first = tmp_path / "first"
    (first / "csrc").mkdir(parents=True)
    shutil.copy(entry.PKG_DIR / "build.py", first / "build.py")
    for name in ("a.cu", "a.cuh"):
        (first / "csrc" / name).write_text("")
        os.utime(first / "csrc" / name, (1e9, 1e9))

    def compile_in(place):
        spec = importlib.util.spec_from_file_location("build_of_" + place.name, place / "build.py")
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        before = (tmp_path / "calls").read_text().count("\n") if (tmp_path / "calls").exists() else 0
        m._compile(m.units()[0], False, False)
        return (tmp_path / "calls").read_text().count("\n") - before
    return first, compile_in


def test_what_is_newer_is_compiled_and_nothing_else(tree):
    first, compile_in = tree
    assert compile_in(first) == 1 and compile_in(first) == 0
    os.utime(first / "csrc" / "a.cuh", (4e9, 4e9))
    assert compile_in(first) == 1


def test_objects_of_a_copied_tree_are_not_the_copys(tree, tmp_path):
    first, compile_in = tree
    assert compile_in(first) == 1
    copy = tmp_path / "copy"
    shutil.copytree(first, copy)                                     # the list beside the object names the files of the first tree
    os.utime(copy / "csrc" / "a.cuh", (4e9, 4e9))
    assert compile_in(copy) == 1
    link = tmp_path / "link"
    link.symlink_to(first)                                           # the same tree under another name is the same tree
    assert compile_in(link) == 0

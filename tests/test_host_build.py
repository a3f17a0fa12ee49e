"""What the incremental build takes for up to date, with a compiler that only records its calls."""
import importlib.util
import os
import stat
import time

import pytest

from conftest import ROOT

COMPILER = """#!/bin/sh
case "$*" in *--version*) echo "$VERSION_OF_FAKE"; exit 0;; esac
while [ $# -gt 0 ]; do
    case "$1" in -o) out="$2"; shift;; -c) src="$2"; shift;; esac
    shift
done
echo partial > "$out"
[ -n "$src" ] && [ "$(basename "$src")" = "$FAIL_OF_FAKE" ] && exit 1
echo "$(basename "${src:-link}")" >> "$LOG_OF_FAKE"
"""


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build module over two sources of each kind in a directory of their own; ``build.calls()`` compiles and tells what
    was compiled or linked."""
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(ROOT, "torchsplinekan_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    fake = tmp_path / "compiler"
    fake.write_text(COMPILER)
    fake.chmod(fake.stat().st_mode | stat.S_IXUSR)
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for name in ("a.cu", "b.cu", "c.cpp", "d.cpp"):
        (csrc / name).write_text("// " + name)
    lib = tmp_path / "lib"
    for name, value in dict(PKG=str(tmp_path), CSRC=str(csrc), LIB_DIR=str(lib), LIB_PATH=str(lib / "lib.so"), SOURCES=["a.cu", "b.cu"],
                            HEADERS=[], EXT_SOURCES=["c.cpp", "d.cpp"], EXT_HEADERS=[]).items():
        monkeypatch.setattr(mod, name, value)
    monkeypatch.setattr(mod.shutil, "which", lambda name, path=None: str(fake))
    monkeypatch.setenv("LOG_OF_FAKE", str(tmp_path / "log"))
    monkeypatch.setenv("VERSION_OF_FAKE", "1")
    monkeypatch.setenv("FAIL_OF_FAKE", "")

    def calls():
        (tmp_path / "log").write_text("")
        if hasattr(mod, "_version"):
            mod._version.cache_clear()
        mod.build_library()
        mod.build_extension()
        return sorted((tmp_path / "log").read_text().split())

    mod.calls, mod.csrc = calls, csrc
    return mod


def age(build, *changed):
    """Everything built so far was built a while ago, from older sources; ``changed`` were edited since."""
    now = time.time()
    for top in (build.PKG, os.path.join(build.PKG, "build"), build.LIB_DIR):
        for name in os.listdir(top):
            if name.endswith((".o", ".so")):
                os.utime(os.path.join(top, name), (now - 100, now - 100))
    for name in os.listdir(build.csrc):
        at = now - (50 if name in changed else 200)
        os.utime(build.csrc / name, (at, at))


EXTENSION = ["c.cpp", "d.cpp", "link"]
ALL = sorted(["a.cu", "b.cu", "link"] + EXTENSION)


def test_one_changed_source_is_compiled_alone(build):
    assert build.calls() == ALL
    age(build)
    assert build.calls() == []
    age(build, "a.cu")
    assert build.calls() == ["a.cu", "link", "link"]          # the extension is linked against the library
    age(build, "d.cpp")
    assert build.calls() == ["d.cpp", "link"]


def test_other_flags_make_every_object_out_of_date(build, monkeypatch):
    build.calls()
    age(build, "a.cu")
    monkeypatch.setattr(build, "NVCC_FLAGS", build.NVCC_FLAGS + ["-DOTHER"])
    assert build.calls() == ["a.cu", "b.cu", "link", "link"]
    age(build)
    assert build.calls() == []


def test_another_compiler_or_torch_makes_every_object_out_of_date(build, monkeypatch):
    build.calls()
    age(build, "a.cu", "c.cpp")
    monkeypatch.setenv("VERSION_OF_FAKE", "2")
    assert build.calls() == ALL
    age(build, "c.cpp")
    monkeypatch.setattr("importlib.metadata.version", lambda name: "another")
    assert build.calls() == EXTENSION
    age(build)
    monkeypatch.setattr("importlib.metadata.version", lambda name: "a third")
    assert build.calls() == EXTENSION                         # nothing was edited, the headers are others
    age(build)
    assert build.calls() == []


@pytest.mark.parametrize("name", ["a.cu", "c.cpp"])
def test_a_compilation_that_fails_leaves_no_object(build, monkeypatch, name):
    build.calls()
    age(build, name)
    monkeypatch.setenv("FAIL_OF_FAKE", name)
    for _ in range(2):
        with pytest.raises(RuntimeError, match=name):
            build.calls()
    monkeypatch.setenv("FAIL_OF_FAKE", "")
    assert name in build.calls()

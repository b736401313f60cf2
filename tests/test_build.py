"""What the in-tree build compiles again: objects whose source, headers or command line are not those they were made from."""
import os

import pytest

from kubeoperator_amd.ops import _build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source folder of two kernels and the bindings; compilers that only write their output file. Returns a function that builds
    and names what was compiled."""
    src = tmp_path / "csrc"
    src.mkdir()
    for f in ("one.hip", "two.hip", "bindings.cpp", "common.h"):
        (src / f).write_text("//")
        os.utime(src / f, (1, 1))
    monkeypatch.setattr(_build, "CSRC", str(src))
    monkeypatch.setattr(_build, "BUILD_DIR", str(tmp_path / "objects"))
    monkeypatch.setattr(_build, "SO_PATH", str(tmp_path / "_C.so"))
    monkeypatch.setattr(_build, "_hipcc", lambda: "hipcc")
    ran = []

    def run(cmd):
        out = cmd[cmd.index("-o") + 1]
        ran.append(os.path.basename(out))
        if "-DFAILS" in cmd:
            raise RuntimeError("build command failed")
        with open(out, "w") as f:
            f.write(" ".join(cmd))

    monkeypatch.setattr(_build, "_run", run)

    def build():
        ran.clear()
        _build.build()
        return sorted(ran)

    build.src = src
    return build


ALL = ["_C.so.tmp", "bindings.cpp.o", "one.hip.o", "two.hip.o"]


def test_nothing_changed_nothing_compiled(tree):
    assert tree() == ALL
    assert tree() == []


def test_other_flags_compile_again(tree, monkeypatch):
    """An object made with other flags is not kept, however new it is: packed fp32 instructions are switched off by one."""
    tree()
    monkeypatch.setattr(_build, "BASE_HIPFLAGS", [])
    assert tree() == ["_C.so.tmp", "one.hip.o", "two.hip.o"]
    assert tree() == []
    monkeypatch.setitem(_build.FILE_FLAGS, "two.hip", ["-fno-slp-vectorize"])
    assert tree() == ["_C.so.tmp", "two.hip.o"]
    monkeypatch.setattr(_build, "ARCH", "gfx942")
    assert tree() == ["_C.so.tmp", "one.hip.o", "two.hip.o"]
    monkeypatch.setenv("KOP_EXT_NAME", "_Cother")
    assert tree() == ["_C.so.tmp", "bindings.cpp.o"]


def test_objects_of_unknown_flags_and_newer_sources_compile_again(tree):
    tree()
    for f in os.listdir(_build.BUILD_DIR):  # as a build that kept no record left them
        if not f.endswith(".o"):
            os.remove(os.path.join(_build.BUILD_DIR, f))
    assert tree() == ALL
    os.utime(tree.src / "one.hip")
    os.utime(tree.src / "one.hip", (2e9, 2e9))
    assert tree() == ["_C.so.tmp", "one.hip.o"]


def test_a_failed_compilation_is_tried_again(tree, monkeypatch):
    tree()
    monkeypatch.setitem(_build.FILE_FLAGS, "one.hip", ["-DFAILS"])
    for _ in range(2):
        with pytest.raises(RuntimeError):
            tree()
    monkeypatch.setitem(_build.FILE_FLAGS, "one.hip", [])
    assert tree() == []  # the object is still the one that these flags made

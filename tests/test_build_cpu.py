"""The build: objects and libraries are there whole or not at all."""
import os
import stat

import pytest

from paraconv2d_b200 import build


@pytest.fixture
def place(tmp_path, monkeypatch):
    """A tree of its own with one kernel source and a stand-in for the compiler."""
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "a.cu").write_text("// a kernel\n")
    monkeypatch.setattr(build, "CSRC", str(tmp_path / "csrc"))
    monkeypatch.setattr(build, "INCLUDE", str(tmp_path / "include"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path / "objects"))
    monkeypatch.setattr(build, "KERNEL_LIB", str(tmp_path / "lib.so"))

    def compiler(script):
        path = tmp_path / "compiler"
        path.write_text("#!/bin/sh\nwhile [ $# -gt 0 ]; do [ \"$1\" = -o ] && out=$2; [ \"$1\" = -c ] && src=$2; shift; done\n"
                        + script)
        path.chmod(path.stat().st_mode | stat.S_IXUSR)
        monkeypatch.setattr(build, "NVCC", str(path))

    return tmp_path, compiler


def test_an_interrupted_compiler_leaves_no_object(place):
    path, compiler = place
    compiler('echo half > "$out"; exit 1\n')
    with pytest.raises(RuntimeError):
        build.build_kernel_lib()
    assert os.listdir(path / "objects") == [] and not (path / "lib.so").exists()
    compiler('echo whole > "$out"\n')
    build.build_kernel_lib()
    assert os.listdir(path / "objects") == ["a.cu.o"] and (path / "objects" / "a.cu.o").read_text() == "whole\n"


def test_an_object_keeps_its_name_until_the_next_one_is_whole(place):
    """While a second build compiles, a first one may link what is there."""
    path, compiler = place
    compiler('echo first > "$out"\n')
    build.build_kernel_lib()
    obj = path / "objects" / "a.cu.o"
    compiler(f'echo second > "$out"; [ -z "$src" ] || cat {obj} > {path}/seen\n')
    build.build_kernel_lib(force=True)
    assert (path / "seen").read_text() == "first\n" and obj.read_text() == "second\n"


def test_objects_newer_than_their_sources_are_kept(place):
    path, compiler = place
    compiler('echo first > "$out"\n')
    build.build_kernel_lib()
    (path / "lib.so").unlink()
    compiler('[ -z "$src" ] || exit 1; echo linked > "$out"\n')
    build.build_kernel_lib()
    assert (path / "objects" / "a.cu.o").read_text() == "first\n"

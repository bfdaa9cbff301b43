"""When the library's objects are compiled anew: a source, a header or the recipe itself (its flags) is newer, and always when asked to"""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def recipe(tmp_path, monkeypatch):
    """the build module on a tree of two sources, with a compiler that only leaves its output file"""
    spec = importlib.util.spec_from_file_location("recipe", os.path.join(ROOT, "nonauto-lm_amd", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    csrc, lib = tmp_path / "csrc", tmp_path / "lib"
    csrc.mkdir(), lib.mkdir()
    for name in ("a.hip", "b.hip", "common.hpp"):
        (csrc / name).write_text("")
    own = tmp_path / "build.py"
    own.write_text("")
    for name, value in (("CSRC", csrc), ("LIBDIR", lib), ("LIB", lib / "lib.so"), ("__file__", own), ("RECIPE", own)):
        monkeypatch.setattr(module, name, str(value), raising=False)
    monkeypatch.setattr(module, "SOURCES", ["a.hip", "b.hip"])
    made = []

    def compiler(cmd):
        made.append(os.path.basename(cmd[cmd.index("-o") + 1]))
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(module.subprocess, "check_call", compiler)

    def touch(name, at):
        os.utime(tmp_path / name, (at, at))

    for name in ("csrc/a.hip", "csrc/b.hip", "csrc/common.hpp", "build.py"):
        touch(name, 1000)
    module.build(verbose=False)
    assert sorted(made) == ["a.o", "b.o", "lib.so"]
    for name in ("lib/a.o", "lib/b.o", "lib/lib.so"):
        touch(name, 2000)
    del made[:]
    return module, made, touch


@pytest.mark.parametrize("newer,want", [(None, []), ("csrc/a.hip", ["a.o", "lib.so"]), ("csrc/common.hpp", ["a.o", "b.o", "lib.so"]),
                                        ("build.py", ["a.o", "b.o", "lib.so"])])
def test_what_is_compiled_anew(recipe, newer, want):
    module, made, touch = recipe
    if newer:
        touch(newer, 3000)
    module.build(verbose=False)
    assert sorted(made) == want


def test_forced(recipe):
    module, made, _ = recipe
    module.build(force=True, verbose=False)
    assert sorted(made) == ["a.o", "b.o", "lib.so"]


def test_the_entry_compiles_every_time(monkeypatch):
    sys.path.insert(0, ROOT)
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **k: calls.append(cmd))
    entry.build()
    assert len(calls) == 1 and calls[0][1].endswith("build.py") and "--force" in calls[0]

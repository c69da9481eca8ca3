"""The build recipe without a compiler: what is compiled again, and when."""
import os
import re

import pytest


@pytest.fixture
def recipe(tmp_path, monkeypatch):
    """situation3d_amd.build over a folder of its own; run() -> the sources it compiled, and whether it linked."""
    from situation3d_amd import build
    monkeypatch.setattr(build, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    calls = []

    def compiler(cmd):
        calls.append(cmd)
        if build.fail in cmd:
            raise RuntimeError("compiler")
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass

    monkeypatch.setattr(build.subprocess, "check_call", compiler)
    monkeypatch.setattr(build, "fail", None, raising=False)

    def run(**kw):
        calls.clear()
        build.build(**kw)
        return sorted(os.path.basename(c[c.index("-c") + 1]) for c in calls if "-c" in c), any("-shared" in c for c in calls)

    build_run = run
    build_run.module = build
    return build_run


def test_objects_of_other_flags_are_compiled_again(recipe, monkeypatch):
    build = recipe.module
    everything = sorted(build.SOURCES)
    assert recipe() == (everything, True)
    assert recipe() == ([], False)
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-DOTHER"])
    assert recipe() == (everything, True)
    assert recipe() == ([], False)
    monkeypatch.setenv("HIPCC", os.path.abspath(__file__))                # another compiler
    assert recipe() == (everything, True)


def test_an_interrupted_build_leaves_no_mixture(recipe, monkeypatch):
    build = recipe.module
    assert recipe()[1]
    flags = build.FLAGS
    monkeypatch.setattr(build, "FLAGS", flags + ["-DOTHER"])
    monkeypatch.setattr(build, "fail", os.path.join(build.CSRC, build.SOURCES[0]))
    with pytest.raises(RuntimeError):
        recipe()
    monkeypatch.setattr(build, "FLAGS", flags)
    monkeypatch.setattr(build, "fail", None)
    assert recipe() == (sorted(build.SOURCES), True)


def test_objects_without_a_record_are_compiled_again(recipe):
    build = recipe.module
    assert recipe()[1]
    os.remove(os.path.join(build.OBJ, "command"))
    assert recipe() == (sorted(build.SOURCES), True)


def _included(path, seen):
    for name in re.findall(r'^#include "([^"]+)"', open(path).read(), re.M):
        for folder in (os.path.dirname(path), os.path.join(os.path.dirname(path), "..", "..", "include")):
            at = os.path.normpath(os.path.join(folder, name))
            if os.path.exists(at) and at not in seen:
                seen.add(at)
                _included(at, seen)
    return seen


def test_every_included_header_makes_its_sources_stale(recipe, monkeypatch):
    """... wherever a source stands in the list."""
    build = recipe.module
    monkeypatch.setattr(build, "SOURCES", build.SOURCES[::-1])
    assert recipe()[1]
    headers = {src: _included(os.path.join(build.CSRC, src), set()) for src in build.SOURCES}
    before = {os.path.join(build.OBJ, f): os.path.getmtime(os.path.join(build.OBJ, f)) for f in os.listdir(build.OBJ)}
    mtime = os.path.getmtime
    for header in sorted(set().union(*headers.values())):
        # objects as old as they were, the header newer than they are
        monkeypatch.setattr(build.os.path, "getmtime", lambda p: before.get(p, 0.0) if not os.path.normpath(p) == header else 1e18)
        compiled, linked = recipe()
        monkeypatch.setattr(build.os.path, "getmtime", mtime)
        assert linked and {s for s in headers if header in headers[s]} <= set(compiled), header


def test_the_entry_point_compiles_every_time(monkeypatch):
    import __graft_entry__
    from oracle import pointnet2_ref
    from situation3d_amd import build
    forced = []
    monkeypatch.setattr(build, "build", lambda force=False, verbose=False: forced.append(force) or build.LIB)
    monkeypatch.setattr(pointnet2_ref, "build", lambda force=False: None)
    monkeypatch.setattr(build.os.path, "exists", lambda p: True)
    __graft_entry__.build()
    assert forced == [True]

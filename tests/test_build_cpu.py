"""What the build runs, without running it: with torch and without, and under another Python."""

import importlib.util
import os
import types

import pytest

from dragon_b200 import build


@pytest.fixture
def commands(tmp_path, monkeypatch):
    """The commands of a build into an empty folder; each leaves its output behind, newer than what was there."""
    ran, clock = [], [2_000_000_000]
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path / "build"))

    def run(cmd):
        ran.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        clock[0] += 1
        os.utime(out, (clock[0], clock[0]))
        return ""

    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build.concurrent.futures, "ThreadPoolExecutor", Serial)
    return ran


class Serial(object):
    def __init__(self, max_workers):
        pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        pass

    map = staticmethod(map)


def outputs(ran):
    return sorted(os.path.basename(c[c.index("-o") + 1]) for c in ran)


def test_without_torch_the_other_libraries_are_built(commands, monkeypatch, capsys):
    find_spec = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find_spec(name, *a))
    assert build.build().endswith("libdgn.so")
    assert {"libdgn.so", "libdragon_collective.so", "dgn_norm.o"} <= set(outputs(commands))
    assert not any("dgn_torch" in word or word.startswith("-ltorch") for c in commands for word in c)
    assert "dgn_torch.so" in capsys.readouterr().out


def test_the_extension_follows_the_versions_it_was_built_for(commands, monkeypatch):
    build.build()
    assert {"libdgn.so", "dgn_torch.o", "dgn_torch.so"} <= set(outputs(commands))
    del commands[:]
    build.build()
    assert commands == []
    stamp = os.path.join(build.OBJ, "dgn_torch.versions")
    monkeypatch.setattr(build, "sys", types.SimpleNamespace(version="another Python"))
    write = build._newer

    def newer(target, deps):  # the stamp was written just now, after objects that the fixture dates into the future
        if stamp in deps and "another Python" in open(stamp).read():
            os.utime(stamp, (2_100_000_000, 2_100_000_000))
        return write(target, deps)

    monkeypatch.setattr(build, "_newer", newer)
    build.build()
    assert "dgn_torch.o" in outputs(commands) and "libdgn.so" not in outputs(commands)

"""The extension builder's choice of what to compile again, with compilers that
only write down what they were asked for."""
import os
import subprocess

import pytest

from cpd_amd.ops import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Three sources and a compiler; ``tree.compiled`` are the sources of the
    last build, ``tree.breaks`` the one whose compiler is killed half way."""
    class Tree:
        compiled, breaks = [], None

        def build(self, **kw):
            self.compiled = []
            return build.build_hip(verbose=False, **kw)

        def touch(self, name):
            path = tmp_path / "csrc" / name
            at = os.path.getmtime(tmp_path / "_cpd_hip.so") + 2
            os.utime(path, (at, at))

    t = Tree()
    (tmp_path / "csrc").mkdir()
    for name in ("a.hip", "b.hip", "hip_bindings.cpp"):
        (tmp_path / "csrc" / name).write_text("\n")
    old = os.path.getmtime(build.__file__)
    for name in ("a.hip", "b.hip", "hip_bindings.cpp"):
        os.utime(tmp_path / "csrc" / name, (old, old))

    def run(cmd, verbose):
        out = cmd[cmd.index("-o") + 1]
        if "-c" not in cmd:
            open(out, "w").write("linked")
            return
        src = cmd[cmd.index("-c") + 1]
        t.compiled.append(os.path.basename(src))
        with open(cmd[cmd.index("-MF") + 1], "w") as f:
            f.write(f"{out}: {src}\n")
        open(out, "w").write("half")
        if os.path.basename(src) == t.breaks:
            raise subprocess.CalledProcessError(-9, cmd)
        open(out, "w").write("whole")

    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "CSRC", str(tmp_path / "csrc"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path / "_obj"))
    monkeypatch.setattr(build, "_torch_paths", lambda: ([], [], "1"))
    monkeypatch.setattr(build, "_run", run)
    return t


def test_only_what_changed(tree):
    tree.build()
    assert sorted(tree.compiled) == ["a.hip", "b.hip", "hip_bindings.cpp"]
    tree.build()
    assert tree.compiled == []
    tree.touch("b.hip")
    tree.build()
    assert tree.compiled == ["b.hip"]
    tree.build(force=True)
    assert len(tree.compiled) == 3


def test_another_architecture_makes_every_object(tree, monkeypatch):
    """Objects of two architectures are never linked together."""
    tree.build()
    monkeypatch.setattr(build, "GFX_ARCH", "gfx942")
    tree.touch("a.hip")
    tree.build()
    assert len(tree.compiled) == 3


def test_a_killed_compiler_is_run_again(tree):
    """What it left, newer than its source, is not linked."""
    tree.breaks = "a.hip"
    with pytest.raises(subprocess.CalledProcessError):
        tree.build()
    tree.breaks = None
    tree.build()
    assert "a.hip" in tree.compiled


def test_no_workers_asked_for(tree, monkeypatch):
    monkeypatch.setenv("MAX_JOBS", "0")
    tree.build()
    assert len(tree.compiled) == 3

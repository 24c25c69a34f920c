"""The incremental build: what is made again, and when (the compilers are stood in for)."""
import os
import types

import pytest

from distributed_pytorch_amd import build as B


@pytest.fixture()
def tree(tmp_path, monkeypatch):
    """A package of one source for each module; -> (build(), {name of what was made: how often})."""
    pkg = tmp_path / "pkg"
    for path in ("kernels/a.hip", "kernels/b.hip", "transformer/bind.cpp"):
        f = pkg / "csrc" / path
        f.parent.mkdir(parents=True, exist_ok=True)
        f.write_text('#include "../common.h"\n' if path.endswith("a.hip") else "")
    (pkg / "csrc" / "common.h").write_text("")
    made, fail = [], []

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        made.append(os.path.basename(out).split(".cpython")[0])
        if any(f in out for f in fail):
            return types.SimpleNamespace(returncode=1, stderr="no")
        with open(out, "w"):
            pass
        return types.SimpleNamespace(returncode=0, stderr="")

    monkeypatch.setattr(B, "HERE", str(pkg))
    monkeypatch.setattr(B, "CSRC", str(pkg / "csrc"))
    monkeypatch.setattr(B.subprocess, "run", run)
    monkeypatch.delenv("DPA_BUILD_DEFS", raising=False)

    def go(**kw):
        del made[:]
        B.build(**kw)
        return sorted(made)

    go.fail, go.made, go.pkg = fail, made, pkg
    return go


EVERYTHING = ["_C", "_T", "kernels_a.hip.o", "kernels_b.hip.o", "transformer_bind.cpp.o"]


def test_made_once_and_again_where_a_source_or_header_is_newer(tree):
    assert tree() == EVERYTHING and tree() == [] and tree(force=True) == EVERYTHING

    def age(files, t):
        for f in files:
            os.utime(f, (t, t))

    for name, again in (("common.h", ["_C", "kernels_a.hip.o"]), ("kernels/b.hip", ["_C", "kernels_b.hip.o"])):
        age((tree.pkg / "csrc").rglob("*.*"), 1000)
        age((tree.pkg.parent / "build" / "obj").iterdir(), 2000)
        age(tree.pkg.glob("_*"), 3000)
        assert tree() == []
        age([tree.pkg / "csrc" / name], 4000)
        assert tree() == again


def test_made_again_by_another_command(tree, monkeypatch):
    """Flags alone (a target feature switched off) make every object that they are for again."""
    tree()
    monkeypatch.setattr(B, "NO_PACKED_FP32", [])
    assert tree() == ["_C", "kernels_a.hip.o", "kernels_b.hip.o"] and tree() == []
    monkeypatch.setenv("DPA_BUILD_DEFS", "-DX=1")
    assert tree() == ["_C", "kernels_a.hip.o", "kernels_b.hip.o"] and tree() == []


def test_a_link_that_failed_is_made_again(tree):
    """... and not left at the library of the objects before."""
    tree()
    tree.fail.append("_C")
    with pytest.raises(RuntimeError, match="link failed"):
        tree(force=True)
    del tree.fail[:]
    assert "_C" in tree()

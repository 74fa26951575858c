"""The build's order and conditions, with the compilers replaced by a recorder."""
import subprocess
import sys
from pathlib import Path

import pytest

from pilm_b200 import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A copy of the source tree's names; runs: what was compiled, in order."""
    for d in ("csrc", "include"):
        (tmp_path / d).mkdir()
    for s in b.SOURCES + ["args.cpp"]:
        (tmp_path / "csrc" / s).write_text("")
    for name, path in dict(HERE=tmp_path, CSRC=tmp_path / "csrc", INCLUDE=tmp_path / "include",
                           LIB=tmp_path / "libpilm_cuda.so", ARGS=tmp_path / "_args.so",
                           ARGS_STAMP=tmp_path / "_build" / "args.stamp").items():
        monkeypatch.setattr(b, name, path)
    runs = []

    def run(cmd, check):
        out = Path(cmd[cmd.index("-o") + 1])
        runs.append(out.name)
        if out.name in run.fail:
            raise subprocess.CalledProcessError(1, cmd)
        out.write_text("")
    run.fail = set()
    monkeypatch.setattr(b.subprocess, "run", run)
    monkeypatch.setattr(b, "nvcc", lambda: "nvcc")
    return runs, run


def test_the_library_is_built_first_and_both_only_once(tree):
    runs, _ = tree
    assert b.build() == b.LIB and b.LIB.exists() and b.ARGS.exists()
    assert runs[-2:] == ["libpilm_cuda.so.tmp", "_args.so.tmp"] and len(runs) == len(b.SOURCES) + 2
    b.build()
    assert len(runs) == len(b.SOURCES) + 2
    b.build(force=True)
    assert len(runs) == 2 * (len(b.SOURCES) + 2)


@pytest.mark.parametrize("lack", ["torch", "Python.h", "compiler"])
def test_nvcc_alone_builds_the_library(tree, monkeypatch, lack, tmp_path):
    runs, _ = tree
    if lack == "torch":
        monkeypatch.setattr(b.util, "find_spec", lambda name: None)
    elif lack == "Python.h":
        monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "none")})
    else:
        monkeypatch.setenv("CXX", "no-such-compiler")
    with pytest.warns(UserWarning, match="_args.so was not built"):
        assert b.build() == b.LIB
    assert b.LIB.exists() and not b.ARGS.exists() and "_args.so.tmp" not in runs


def test_an_extension_that_does_not_compile_is_named_and_the_library_stands(tree):
    runs, run = tree
    run.fail.add("_args.so.tmp")
    with pytest.raises(RuntimeError, match="_args.so, the Python entry"):
        b.build()
    assert b.LIB.exists() and not b.ARGS.exists()


def test_another_torch_rebuilds_the_extension_alone(tree, monkeypatch):
    runs, _ = tree
    b.build()
    del runs[:]
    monkeypatch.setattr(b.metadata, "version", lambda name: "0.0+other")
    b.build()
    assert runs == ["_args.so.tmp"]
    b.build()
    assert runs == ["_args.so.tmp"]


def test_the_extension_loads_in_a_process_that_has_not_imported_torch():
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", "from pilm_b200 import bindings; print(bindings.args().__name__)"], cwd=root,
                       capture_output=True, text=True, timeout=300)
    assert r.stdout.strip() == "pilm_b200._args", r.stderr


def test_an_extension_that_does_not_load_says_why(monkeypatch):
    from pilm_b200 import bindings
    monkeypatch.setattr(bindings, "_args", None)
    monkeypatch.setitem(sys.modules, "pilm_b200._args", None)
    monkeypatch.delattr(sys.modules["pilm_b200"], "_args", raising=False)
    with pytest.raises(RuntimeError, match="python -m pilm_b200.build.*: .*_args"):
        bindings.args()

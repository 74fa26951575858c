"""bench.py's cache flags: used by the run that they are given to, or refused."""
import sys

import pytest

import bench


def run(monkeypatch, *argv):
    """What main() would run: the flags reach one of these and nothing is printed for another workload."""
    ran = []
    for name in ("run_prefill", "run_sweep", "run_config", "run_reference", "run_ours"):
        monkeypatch.setattr(bench, name, lambda args, *a, name=name: ran.append((name, args)) or None)
    monkeypatch.setattr(sys, "argv", ["bench.py", *argv])
    bench.main()
    return ran


@pytest.mark.parametrize("argv,what", [
    (["--sweep", "all", "--kv", "e4m3"], "--sweep"),
    (["--config", "2", "--kv", "e4m3"], "--config"),
    (["--impl", "reference", "--kv", "e4m3"], "--impl reference"),
    (["--window", "64"], "--kv e4m3"), (["--sinks", "4"], "--kv e4m3"), (["--prefill", "64", "--window", "8"], "--kv e4m3"),
    (["--kv", "e4m3", "--sinks", "4"], "--window"),
    (["--kv", "e4m3", "--window", "-1"], "negative"), (["--kv", "e4m3", "--window", "8", "--sinks", "-1"], "negative"),
])
def test_flags_that_a_run_would_not_use_are_refused(monkeypatch, capsys, argv, what):
    with pytest.raises(SystemExit) as e:
        run(monkeypatch, *argv)
    assert e.value.code == 2 and what in capsys.readouterr().err


@pytest.mark.parametrize("argv,name", [
    ([], "run_ours"), (["--kv", "e4m3"], "run_ours"), (["--kv", "e4m3", "--window", "64", "--sinks", "4"], "run_ours"),
    (["--prefill", "64"], "run_prefill"), (["--prefill", "64", "--kv", "e4m3", "--window", "8"], "run_prefill"),
    (["--impl", "reference"], "run_reference"), (["--sweep", "all"], "run_sweep"), (["--config", "2"], "run_config"),
])
def test_runs_that_take_their_flags(monkeypatch, capsys, argv, name):
    assert [n for n, _ in run(monkeypatch, *argv)] == [name]


def test_lines_name_the_cache():
    from argparse import Namespace
    assert bench.kv_config(Namespace(kv="bf16", window=0, sinks=0)) == {}
    assert bench.kv_config(Namespace(kv="e4m3", window=8, sinks=1)) == {"kv_cache": "e4m3", "window": 8, "sinks": 1}

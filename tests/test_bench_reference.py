"""CPU: the bench where the reference's CPU path is neither built nor buildable:
its reference arm says so in one line and ends well, and the other arm's line
carries the reason in that leg's place instead of failing."""
import argparse
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def bench(monkeypatch):
    import bench
    from oracle import oracle as O
    monkeypatch.setattr(O, "ref_available", lambda: False)
    monkeypatch.setattr(O, "build", lambda: None)
    return bench


def test_reference_arm_is_unavailable_in_one_line(bench, capsys):
    bench.run_reference(argparse.Namespace(workload="decode_b64_zipf", steps=2, warmup=1))
    out = capsys.readouterr().out.splitlines()
    assert len(out) == 1
    line = json.loads(out[0])
    assert line["impl"] == "reference" and "sources" in line["unavailable"]


def test_missing_reference_is_told_apart_from_other_errors(bench):
    with pytest.raises(bench.NoReference):
        bench.cpu_reference("decode_b1", steps=1, warmup=0)


def test_the_command_prints_one_json_line_on_stdout():
    from oracle import oracle as O
    if O.ref_available() or os.path.exists(os.path.join(ROOT, "..", "reference", "quant.c")):
        pytest.skip("the reference is here: its arm would be timed")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--impl", "reference", "--gpus", "1", "--steps", "2", "--warmup", "1"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert len(r.stdout.splitlines()) == 1 and "unavailable" in json.loads(r.stdout)

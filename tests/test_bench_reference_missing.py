"""bench.py's reference arm where the reference was not built (CPU only): it says so in one line, and does not give
the timing of the restatement of the reference's code as the reference's own."""
import argparse
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_reference_arm_without_the_reference(monkeypatch, capsys):
    sys.path.insert(0, ROOT)
    import bench
    from oracle import oracle as orc
    monkeypatch.setenv("RANK", "0")
    monkeypatch.setattr(orc, "ref_lib", lambda: None)

    def timed(*_):
        raise AssertionError("nothing is to be timed")
    monkeypatch.setattr(bench, "cpu_timed_steps", timed)
    assert bench.run_reference_arm(argparse.Namespace(gpus=1, steps=2, warmup=0, gather="p2p")) == 0
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 1
    d = json.loads(lines[0])
    assert d["impl"] == "reference" and d["unavailable"] and "value" not in d

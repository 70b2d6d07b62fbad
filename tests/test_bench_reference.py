"""The benchmark where the reference's package is absent: its line still
comes, with the reason in place of the CPU baselines."""

from __future__ import annotations

import json

import pytest


@pytest.fixture
def bench(monkeypatch, tmp_path):
    import bench
    from oracle import reference_runs

    monkeypatch.setattr(reference_runs, "REF_DIR", tmp_path)
    return bench


def test_cpu_baselines_give_the_reason(bench):
    append, config1 = {"value": 1.0}, {"value": 2.0}
    cpu = bench.cpu_baselines(None, append, config1, 0)  # the state is not looked at
    assert "oracle/_ref" in cpu["unavailable"]
    assert append == {"value": 1.0} and config1 == {"value": 2.0}
    json.dumps(cpu)


def test_reference_arm_gives_the_reason(bench, capsys):
    assert bench.main(["--impl", "reference", "--steps", "1", "--warmup", "3"]) == 0
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and "oracle/_ref" in line["unavailable"]

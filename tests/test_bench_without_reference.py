"""bench.py where the reference's CPU library is not built: the reference arm says so and ends well, and
our own arm has no CPU baseline instead of an error."""
import json

import pytest

import bench
from oracle import oracle as orc


@pytest.fixture
def no_reference(monkeypatch, tmp_path):
    monkeypatch.setattr(orc, "REF_SO", str(tmp_path / "libref_litemind.so"))


@pytest.mark.parametrize("workload", ["decode", "prefill", "ffn", "load"])
def test_reference_arm_is_unavailable(no_reference, capsys, workload):
    assert bench.main(["--impl", "reference", "--workload", workload, "--steps", "1", "--warmup", "0"]) == 0
    lines = [line for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    assert len(lines) == 1
    d = json.loads(lines[0])
    assert d["impl"] == "reference" and d["unavailable"] and "\n" not in d["unavailable"]


def test_own_arm_asks_before_it_measures_the_reference(no_reference):
    assert "oracle/_ref" in bench.reference_missing()

"""bench.py where the reference library is not built: both arms still print their line."""

import json
import sys

import numpy as np
import pytest

import bench
from oracle import cpu


@pytest.fixture
def no_reference(monkeypatch, tmp_path):
    monkeypatch.setattr(cpu, "REFERENCE_SO", str(tmp_path / "libovvs_ref.so"))


@pytest.mark.parametrize("config", ["c1", "c3", "c4", "ivf", "gemm"])
def test_reference_arm_says_that_it_is_unavailable(config, no_reference, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--config", config])
    monkeypatch.delenv("RANK", raising=False)
    assert bench.main() == 0
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and "libovvs_ref.so" in line["unavailable"]
    assert "\n" not in line["unavailable"]
    monkeypatch.setenv("RANK", "1")  # one line from all ranks together
    assert bench.main() == 0
    assert capsys.readouterr().out == ""


@pytest.mark.parametrize("metric,k,dtype", [("l2", 10, "f32"), ("inner_product", 7, "f16"),
                                            ("l2", 650, "f32")])
def test_own_arm_is_checked_against_the_restatement(metric, k, dtype, no_reference, monkeypatch):
    """Without the reference there is no baseline, but the results are still checked: right ones
    pass, a wrong one does not."""
    monkeypatch.setattr(bench, "CHUNK", 700)
    monkeypatch.setattr(bench, "_reference_sizes", lambda cfg, seconds: (2, 9))
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2300, 16)).astype(np.float16 if dtype == "f16" else np.float32)
    x[1500] = x[20]  # equal distances on both sides of a shard boundary
    q = rng.standard_normal((12, 16)).astype(np.float32)
    q[3] = x[20]
    cfg = dict(n=x.shape[0], dim=16, nq=12, k=k, metric=metric, dtype=dtype)
    nb, ds = (a.reshape(12, k) for a in
              cpu.Oracle().brute_search(x.astype(np.float32), q, k, metric))
    got = bench._search_baseline(cfg, x, q, nb, ds, 12.0)
    assert got["cpu_baseline"]["value"] is None
    assert "libovvs_ref.so" in got["cpu_baseline"]["unavailable"]
    assert got["parity"]["ok"] and got["parity"]["id_mismatch"] == 0
    assert "restatement" in got["parity"]["against"]
    far = ds.copy()
    far[2, 0] += np.abs(far[2, 0]) * np.float32(0.01) + 1  # no tie with what it should be
    assert not bench._search_baseline(cfg, x, q, nb, far, 12.0)["parity"]["ok"]

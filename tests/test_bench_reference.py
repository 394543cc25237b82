"""bench.py's reference arm where the reference is not built: one line that says
it is unavailable, and no figure of this repository's own restatement."""
import argparse
import json
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("rank", [0, 1])
def test_unavailable_without_the_reference(rank, tmp_path, monkeypatch, capsys):
    monkeypatch.syspath_prepend(str(ROOT))
    import bench
    from oracle import oracle as O

    monkeypatch.setattr(O, "REF_SO", tmp_path / "none.so")
    monkeypatch.setattr(O, "_ref", None)
    monkeypatch.setattr(O, "mul_mat", lambda *a, **k: pytest.fail("the restatement was timed"))
    monkeypatch.setenv("RANK", str(rank))
    args = argparse.Namespace(gpus=1, steps=1, warmup=3, workload="qwen3-4b-layer", mode=None)
    bench.run_reference(args, bench.WORKLOADS["qwen3-4b-layer"])
    out = capsys.readouterr().out.splitlines()
    assert len(out) == (1 if rank == 0 else 0)
    if rank == 0:
        d = json.loads(out[0])
        assert d["impl"] == "reference" and "not built" in d["unavailable"] and set(d) == {"impl", "unavailable"}

"""Where the reference's sources are not at hand, oracle/_ref is not built: a
test that compares with it is skipped, not failed, so that those behind it run."""
import subprocess
import sys
from pathlib import Path

import pytest

from oracle import oracle as O

ROOT = Path(__file__).resolve().parents[1]


def test_a_comparison_with_the_reference_is_skipped(tmp_path):
    (tmp_path / "test_one.py").write_text(f"""
import sys
from pathlib import Path
sys.path.insert(0, {str(ROOT)!r})
from oracle import oracle as O
O.REF_SO, O._ref = Path({str(tmp_path / "none.so")!r}), None
def test_first():
    O.ref()
def test_second():
    pass
""")
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-rs", "-p", "no:cacheprovider", "test_one.py"],
                       cwd=tmp_path, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "1 passed, 1 skipped" in r.stdout, r.stdout + r.stderr
    assert "needs the reference sources" in r.stdout


def test_it_is_an_error_elsewhere(tmp_path, monkeypatch):
    monkeypatch.setattr(O, "REF_SO", tmp_path / "none.so")
    monkeypatch.setattr(O, "_ref", None)
    with pytest.raises(RuntimeError, match="needs the reference sources"):
        O.ref()

"""The serving example end to end: shared prompt, paged MX cache, drafts and their verification."""
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "rust-fp4-blackwell_b200" / "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_drafts_do_not_change_greedy_answers(fmt):
    import serve_mxkv
    plain, drafted, n0, n1 = serve_mxkv.main(["--requests", "5", "--prompt", "70", "--tokens", "48", "--draft", "3",
                                              "--format", fmt])
    assert n1 <= n0 and all(len(t) == 48 for t in plain + drafted)
    # both see the same cache; sums in another order can turn a near tie of the argmax, after which a request differs
    alike = sum(p == d for p, d in zip(plain, drafted))
    assert alike >= 4

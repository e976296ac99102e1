"""A product always has a status word: the weights' own where the caller gives none."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_the_weights_word_is_passed(monkeypatch):
    from dsgx10_b200 import linear
    w = linear.LinearW(64, 512, torch.zeros(8 * 2368, dtype=torch.uint8, device="cuda"))
    x = torch.zeros(2, 512, dtype=torch.bfloat16, device="cuda")
    linear.linear_decode(w, x)
    assert w.status.dtype == torch.int32 and int(w.status) == 0
    calls, mine = [], torch.zeros(1, dtype=torch.int32, device="cuda")
    monkeypatch.setattr(linear, "_fn", lambda *a: calls.append(a) or 0)   # (no launch: what the call would be given)
    linear.linear_decode(w, x)
    linear.linear_decode(w, x, status=mine)
    assert [c[-2] for c in calls] == [w.status.data_ptr(), mine.data_ptr()]

"""What the Python calls of the 8-bit cache and of sampling hand to the library, without a GPU:
the tensors are on the CPU, the library is a record of its calls."""
import pytest

import gcu

torch = pytest.importorskip("torch")


class Calls:
    """A library that launches nothing: every call is noted and succeeds."""

    def __init__(self, work=0):
        self.made, self.work = [], work

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_work"):
                return self.work
            self.made.append((name, args))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    calls = Calls()
    gcu._torch()
    monkeypatch.setattr(gcu, "lib", lambda: calls)
    monkeypatch.setattr(gcu, "_device", lambda what, index: -1)
    monkeypatch.setattr(gcu, "_on", lambda stream, dev: 0)
    return calls


def sample(logits):
    m = logits.shape[0]
    gcu.dev_sample(torch.zeros(m, dtype=torch.int32), logits, torch.zeros(m))


def test_logits_rows_that_are_one_row(library):
    """A stride of 0 is not the library's 0, which stands for rows one behind the other."""
    one = torch.zeros((1, 40))
    sample(one)
    sample(one.expand(3, -1).contiguous())
    assert len(library.made) == 2
    for rows in (one.expand(3, -1), torch.zeros(60).as_strided((3, 40), (8, 1))):
        with pytest.raises(gcu.GcuError, match="rows of 40 logits"):
            sample(rows)
    assert len(library.made) == 2


def prefill(xo, ntok, nh=2, hd=64):
    kv = gcu.KvCacheI8.empty(1, 1, 16, hd, device="cpu")
    gcu.dev_attention_prefill_i8(xo, torch.zeros((nh, ntok, hd)), kv, 0)


def test_prefill_rows_that_are_one_row(library):
    """As above for the rows that prefill attention writes."""
    prefill(torch.zeros((3, 128)), 3)
    prefill(torch.zeros((3, 160))[:, :128], 3)
    prefill(torch.zeros((1, 128)).expand(1, -1), 1)
    assert [args[1] for _, args in library.made] == [128, 160, 0]
    for xo in (torch.zeros((1, 128)).expand(3, -1), torch.zeros(300).as_strided((3, 128), (64, 1))):
        with pytest.raises(gcu.GcuError, match="rows"):
            prefill(xo, 3)
    assert len(library.made) == 3

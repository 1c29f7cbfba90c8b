"""Refusals of the torch wrappers of the 4-bit and expert operators, on tensors that say they are on a GPU and hold nothing, with a
library that only notes its calls: what is refused never gets that far."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ozaki_blackwell_b200 import experts, mx4

pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer")   # empty tensors have none


@pytest.fixture
def gpu(monkeypatch):
    """gpu(*shape): a tensor on a GPU that is not there; gpu.calls: the library's calls so far, as their arguments."""
    calls = []
    for module in (mx4, experts):
        monkeypatch.setattr(module, "_call", lambda index, entry, *args: calls.append(args))

    def make(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda:0")

    make.calls = calls
    with FakeTensorMode():
        yield make


def _routing(gpu, tokens=4, top=2, rows=8):
    return experts.Routing(gpu(4, dtype=torch.int32), gpu(tokens, top, dtype=torch.int32), gpu(rows, dtype=torch.int32), 1)


def test_combine_needs_a_row_for_each_of_the_routing(gpu):
    r = _routing(gpu)
    for rows in (1, 7):
        with pytest.raises(ValueError, match="8 rows"):
            experts.combine(gpu(rows, 16), r)
    assert not gpu.calls
    for rows in (8, 9):     # more do no harm
        assert experts.combine(gpu(rows, 16), r).shape == (4, 16)
    assert len(gpu.calls) == 2


def test_status_is_the_library_s(monkeypatch):
    """mx4.status: nothing where all went well, the library's error where a wait expired or segments were refused."""
    from ozaki_blackwell_b200 import OzakiError
    codes = iter([0, 10004, 10001])
    monkeypatch.setattr(mx4, "_lib", type("Library", (), {"ozb_status": staticmethod(lambda: next(codes))}))
    assert mx4.status() is None
    for code in (10004, 10001):
        with pytest.raises(OzakiError) as e:
            mx4.status()
        assert e.value.code == code

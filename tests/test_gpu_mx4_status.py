"""What a product could not tell its caller at once reaches Python by mx4.status."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_status_after_refused_segments():
    from ozaki_blackwell_b200 import OzakiError, mx4
    a = mx4.quantize(torch.randn(8, 128, device="cuda"))
    mx4.segment_matmul(a, a, torch.tensor([0, 64, 128], dtype=torch.int32, device="cuda"))
    assert mx4.status() is None
    mx4.segment_matmul(a, a, torch.tensor([0, 65, 128], dtype=torch.int32, device="cuda"))
    with pytest.raises(OzakiError) as e:
        mx4.status(a.codes.device)
    assert e.value.code == 10001
    assert mx4.status(0) is None

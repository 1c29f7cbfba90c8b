"""The gradient of the weighted sum over the widest rows that it takes: columns are counted in 32 bits, which a step past the last piece
must not leave."""
import pytest
import torch

pytestmark = pytest.mark.gpu
WIDEST = 2 ** 31 - 1024   # elements of a row


@pytest.mark.parametrize("h", [WIDEST, WIDEST - 256])
def test_widest_rows(h):
    from ozaki_blackwell_b200 import experts as ex
    guard = 4096
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = torch.Generator(device="cuda").manual_seed(h)
    part = torch.randint(-4, 5, (1 << 20,), generator=g, device="cuda").bfloat16()   # small whole numbers: every product is exact
    dy, z = torch.empty(1, h, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, h, dtype=torch.bfloat16, device="cuda")
    for c in range(0, h, 1 << 20):
        dy[0, c: c + (1 << 20)] = part[: min(1 << 20, h - c)]
    z[0, -300:] = 1.0
    z[0, :300] = 2.0
    ids = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    r = ex.sort(ids, 1)
    from ozaki_blackwell_b200._lib import lib
    dz, dw = torch.full((h + guard,), 9.0, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 1, device="cuda")
    weights = torch.full((1, 1), 0.5, device="cuda")
    assert lib.ozb_expert_combine_grad(1, 1, h, dy.data_ptr(), 1, h, z.data_ptr(), h, 1, r.rows.data_ptr(), r.slots.data_ptr(), weights.data_ptr(), dz.data_ptr(), h,
                                       dw.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    assert bool((dz[h:] == 9).all())
    for c in range(0, h, 1 << 28):
        n = min(1 << 28, h - c)
        assert torch.equal(dz[c: c + n], 0.5 * dy[0, c: c + n])
    assert dw.item() == dy[0, -300:].double().sum().item() + 2 * dy[0, :300].double().sum().item()

"""Products of 4-bit operands whose every partial sum is a number of FP32: the result is the exact one, bit for bit, in whatever order and
form it is summed.

Values are codes times 2^0 .. 2^(far - 1), so multiples of 1/2 up to 6 2^(far - 1); products are multiples of 1/4 up to 36 4^(far - 1), and K
of them stay below 2^22 with `far` chosen as below: 24 bits hold every sum. The oracle is a product in 64 bits; BF16 and FP16 round it
once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TABLE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _far(k):
    return next(far for far in (3, 2, 1) if k * 36 * 4 ** (far - 1) < 2 ** 22)


def _operand(k, seed, *shape):
    """A random Mx4 of vectors [*shape] of k values, and the values in 64 bits. Bytes behind the last block's scale are random too."""
    from ozaki_blackwell_b200.mx4 import Mx4
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = -(-k // 32)
    c = torch.randint(0, 16, (*shape, 32 * blocks), generator=g, device="cuda", dtype=torch.uint8)
    c[..., k:] = 0
    s = torch.randint(0, 256, (*shape, -(-blocks // 16) * 16), generator=g, device="cuda", dtype=torch.uint8)
    s[..., :blocks] = 127 + s[..., :blocks] % _far(k)
    values = torch.tensor(TABLE, dtype=torch.float64, device="cuda")[c.int()]
    values *= torch.exp2(s[..., :blocks].double() - 127).repeat_interleave(32, -1)
    return Mx4(c[..., 0::2] | c[..., 1::2] << 4, s, k), values[..., :k]


def _same(y, exact):
    return torch.equal(y, exact.float().to(y.dtype))


def _status():
    from ozaki_blackwell_b200._lib import lib
    assert lib.ozb_status() == 0


@pytest.mark.parametrize("m,n,k", [(600, 10000, 5000), (2053, 4097, 7168), (513, 8192, 65), (4100, 4100, 1090)])
def test_pairs_of_ctas(m, n, k):
    """Two CTAs share a tile and each turns scales for both tensor cores; every slot of scales is used again and again, each time with
    others, so that a stale one shows."""
    from ozaki_blackwell_b200 import mx4
    (x, xv), (w, wv) = _operand(k, m, m), _operand(k, n, n)
    exact = xv @ wv.t()
    for dtype in TYPES:
        assert _same(mx4.matmul(x, w, dtype), exact)
    want = mx4.matmul(x, w)
    for _ in range(20):
        assert torch.equal(mx4.matmul(x, w), want)
    _status()

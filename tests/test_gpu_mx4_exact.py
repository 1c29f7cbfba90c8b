"""Products of 4-bit operands whose every partial sum is a number of FP32: the result is the exact one, bit for bit, in whatever order and
form it is summed.

Values are codes times 2^0 .. 2^(far - 1), so multiples of 1/2 up to 6 2^(far - 1); products are multiples of 1/4 up to 36 4^(far - 1), and K
of them stay below 2^22 with `far` chosen as below: 24 bits hold every sum. The oracle is a product in 64 bits; BF16 and FP16 round it
once."""
import pytest
import torch

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TABLE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _far(k):
    return next(far for far in (3, 2, 1) if k * 36 * 4 ** (far - 1) < 2 ** 22)


def _operand(k, seed, *shape, device="cuda"):
    """A random Mx4 of vectors [*shape] of k values, and the values in 64 bits. Bytes behind the last block's scale are random too."""
    from ozaki_blackwell_b200.mx4 import Mx4
    g = torch.Generator(device=device).manual_seed(seed)
    blocks = -(-k // 32)
    c = torch.randint(0, 16, (*shape, 32 * blocks), generator=g, device=device, dtype=torch.uint8)
    c[..., k:] = 0
    s = torch.randint(0, 256, (*shape, -(-blocks // 16) * 16), generator=g, device=device, dtype=torch.uint8)
    s[..., :blocks] = 127 + s[..., :blocks] % _far(k)
    values = torch.tensor(TABLE, dtype=torch.float64, device=device)[c.int()]
    values *= (1 << (s[..., :blocks].int() - 127)).double().repeat_interleave(32, -1)
    return Mx4(c[..., 0::2] | c[..., 1::2] << 4, s, k), values[..., :k]


def _same(y, exact):
    return torch.equal(y, exact.float().to(y.dtype))


def _status():
    from ozaki_blackwell_b200._lib import lib
    assert lib.ozb_status() == 0


@pytest.mark.parametrize("m,n,k", [(3, 64, 16384), (4, 100, 16400), (17, 130, 20000), (40, 50, 700)])
def test_the_comparison_sees_small_mistakes(m, n, k):
    """On the host: partial sums of a split k rounded to BF16, a block left out, one code or one scale taken for another."""
    (x, xv), (w, wv) = _operand(k, m, m, device="cpu"), _operand(k, n, n, device="cpu")
    exact, far = xv @ wv.t(), _far(k)
    assert k * 36 * 4 ** (far - 1) < 2 ** 22 and torch.equal(exact.float().double(), exact)
    assert _same((xv.float() @ wv.float().t()), exact)         # any order of summation in FP32
    parts = [xv[:, a: a + k // 4] @ wv[:, a: a + k // 4].t() for a in range(0, k, k // 4)]
    assert not _same(sum(p.bfloat16().float() for p in parts), exact)
    assert not _same((xv[:, : k // 32 * 32 - 32] @ wv[:, : k // 32 * 32 - 32].t()).float(), exact)
    for change in (0.5, 2.0):
        wrong = xv.clone()
        wrong[m - 1, 32: 64] *= change
        assert not _same((wrong @ wv.t()).float(), exact)
    wrong = xv.clone()
    wrong[0, k - 1] += 0.5
    assert not _same((wrong @ wv.t()).float(), exact)


@gpu
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


# columns of 16, 32, 64 and 128 tokens; a long k split over clusters of two and four; tokens as lanes
@gpu
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 18432, 1090), (16, 130, 33), (30, 5000, 1090), (60, 20000, 700), (100, 20000, 700), (128, 19000, 2085), (3, 64, 16384),
                                   (4, 100, 16400), (17, 130, 20000), (30, 6000, 7937), (5, 6000, 9000), (140, 9500, 1090), (250, 4000, 5000)])
def test_dense(m, n, k):
    from ozaki_blackwell_b200 import mx4
    (x, xv), (w, wv) = _operand(k, m + 1, m), _operand(k, n + 1, n)
    exact = xv @ wv.t()
    for dtype in TYPES:
        assert _same(mx4.matmul(x, w, dtype), exact)
    _status()


def _grouped(r, n, k, offsets, types=TYPES):
    from ozaki_blackwell_b200 import mx4
    groups = len(offsets) - 1
    (x, xv), (w, wv) = _operand(k, r, r), _operand(k, n, groups, n)
    for dtype in types:
        out = torch.full((r, n), 7.0, dtype=dtype, device="cuda")
        mx4.grouped_matmul(x, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), dtype, out=out)
        for g in range(groups):
            lo, hi = offsets[g], offsets[g + 1]
            assert _same(out[lo:hi], xv[lo:hi] @ wv[g].t()), (dtype, g)
        assert bool((out[: offsets[0]] == 7).all()) and bool((out[offsets[-1]:] == 7).all())
    _status()


# a long k with few tokens to a group (split over clusters, 16 and 32 columns), segments empty, skewed, apart from the ends
@gpu
@pytest.mark.parametrize("k", [7937, 8192, 16400])
@pytest.mark.parametrize("r,offsets", [(40, [0, 0, 37, 40, 40]), (40, [3, 13, 23, 23, 36]), (100, [0, 1, 1, 99, 100]), (90, [0, 30, 60, 89, 90]), (5, [0, 0, 0, 0, 5]), (7, [0, 0, 0, 0, 0])])
def test_rows_of_groups_over_a_long_k(r, offsets, k):
    _grouped(r, 300, k, offsets, TYPES[:2])


# more than 48 tiles to a CTA (beyond what is worked out ahead), k of several stages: weights as lanes, tokens as lanes, pairs
@gpu
@pytest.mark.parametrize("r,n,k,groups", [(1600, 57000, 200, 16), (2400, 57600, 1090, 8), (1100, 113700, 1090, 2)])
def test_rows_of_groups_in_many_tiles(r, n, k, groups):
    each = r // groups
    _grouped(r, n, k, [0] + [g * each + (g * 37 % 50 - 25) for g in range(1, groups)] + [r - 3], TYPES[:1])


@gpu
@pytest.mark.parametrize("r,n,k,groups", [(900, 700, 1090, 30), (2400, 1500, 1090, 8), (1300, 7300, 1090, 2), (500, 130, 96, 1024)])
def test_rows_of_groups(r, n, k, groups):
    cuts = torch.sort(torch.randint(0, r + 1, (groups - 1,), generator=torch.Generator().manual_seed(r))).values.tolist()
    _grouped(r, n, k, [0] + cuts + [r])


@gpu
@pytest.mark.parametrize("m,n,groups,far", [(20, 300, 9, 30), (140, 1500, 8, 12), (300, 700, 40, 3), (1100, 3100, 3, 20), (1100, 3100, 64, 2)])
def test_segments(m, n, groups, far):
    from ozaki_blackwell_b200 import mx4
    lengths = torch.randint(0, far, (groups,), generator=torch.Generator().manual_seed(m)) * 64
    offsets = [0] + lengths.cumsum(0).tolist()
    k = offsets[-1] + 41
    (a, av), (b, bv) = _operand(k, m, m), _operand(k, n, n)
    for dtype in TYPES[: 3 if groups < 64 else 1]:
        y = mx4.segment_matmul(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), dtype)
        for g in range(groups):
            assert _same(y[g], av[:, offsets[g]: offsets[g + 1]] @ bv[:, offsets[g]: offsets[g + 1]].t()), (dtype, g)
    _status()


@gpu
@pytest.mark.parametrize("tokens,top,experts,n,k", [(3, 2, 5, 96, 8200), (3, 2, 5, 8200, 96), (20, 4, 6, 8000, 8000), (700, 2, 2, 700, 1090), (1500, 1, 7, 400, 2000)])
def test_the_layer_and_its_gradients(tokens, top, experts, n, k):
    """Operands that are codes already: a block of them is held exactly whatever its largest. With factors that are the same power of two
    for all slots dz is too, by rows and by columns."""
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    g = torch.Generator(device="cuda").manual_seed(tokens)
    codes = lambda *shape: torch.tensor(TABLE, device="cuda")[torch.randint(0, 16, shape, generator=g, device="cuda")]  # noqa: E731
    x, dy, w = codes(tokens, k), codes(tokens, n), codes(experts, n, k)
    ids = torch.randint(-1, experts, (tokens, top), generator=g, device="cuda")
    weights = torch.full((tokens, top), 2.0, device="cuda")
    y, z, r = ex.matmul(x, mx4.quantize(w), ids, weights, keep=True)
    assert torch.equal(y, ex.matmul(x, mx4.quantize(w), ids, weights))
    dx, _, dw = ex.matmul_grad(dy, x, z, mx4.quantize(w, dim=-2), r, weights)
    want_y, want_dx = torch.zeros(tokens, n, dtype=torch.float64, device="cuda"), torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
    for e in range(experts):
        chosen = (ids == e).double()                    # a token may choose an expert more than once
        times = chosen.sum(1, keepdim=True)
        want_y += 2 * times * (x.double() @ w[e].double().t())
        want_dx += 2 * times * (dy.double() @ w[e].double())
        assert _same(dw[e], (2 * times * dy.double()).t() @ x.double())
    assert _same(y, want_y) and _same(dx, want_dx)
    _status()


# pairs with fewer weights than a CTA's half of a tile; rows of Y with a pitch, whose last columns end inside 16 bytes: tokens as lanes, pairs, few tokens
@gpu
@pytest.mark.parametrize("m,n,k,pitch", [(20000, 50, 700, 50), (20000, 97, 90, 104), (300, 9601, 300, 9608), (150, 9503, 300, 9504), (1100, 3001, 1090, 3016), (40, 1001, 300, 1008)])
def test_results_with_a_pitch(m, n, k, pitch):
    from ozaki_blackwell_b200 import mx4
    (x, xv), (w, wv) = _operand(k, m, m), _operand(k, n, n)
    exact = xv @ wv.t()
    for dtype in TYPES:
        out = torch.full((m + 2, pitch), 5.0, dtype=dtype, device="cuda")
        mx4.matmul(x, w, dtype, out=out[1: m + 1, :n])
        assert _same(out[1: m + 1, :n], exact)
        assert bool((out[0] == 5).all()) and bool((out[m + 1] == 5).all()) and bool((out[:, n:] == 5).all())
    _status()


@gpu
@pytest.mark.parametrize("m,n,pitch,gap", [(140, 1501, 1504, 0), (140, 1501, 1504, 3), (1100, 3001, 3008, 2), (20, 301, 304, 1)])
def test_segments_with_a_pitch(m, n, pitch, gap):
    from ozaki_blackwell_b200 import mx4
    offsets = [0, 64, 64, 320, 384, 640, 704, 768, 790]
    (a, av), (b, bv) = _operand(790, m, m), _operand(790, n, n)
    for dtype in TYPES:
        out = torch.full((8, m + gap, pitch), 5.0, dtype=dtype, device="cuda")
        mx4.segment_matmul(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), dtype, out=out[:, :m, :n])
        for g in range(8):
            assert _same(out[g, :m, :n], av[:, offsets[g]: offsets[g + 1]] @ bv[:, offsets[g]: offsets[g + 1]].t())
        assert bool((out[:, m:] == 5).all()) and bool((out[:, :, n:] == 5).all())
    _status()

"""The microscaled 4-bit format on the GPU: rounding to it and back bit for bit against the definition in 64 bits, and its products.

Tolerance of a product: the sum of K products, each exact in FP32, is accumulated in FP32. Each of at most K additions is off by at
most one unit in the last place of a partial sum, which sum |a b| bounds (the instruction may cut where it could round: 2^-23, not
2^-24): |y - exact| <= K 2^-23 sum |a b|, plus half a unit of the output type, finfo(type).eps / 2 |exact|."""
import ctypes

import pytest
import torch

import mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _mx4():
    from ozaki_blackwell_b200 import mx4
    return mx4


def _status():
    from ozaki_blackwell_b200._lib import lib
    assert lib.ozb_status() == 0


def _random(n, k, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, k, generator=g) * torch.exp2((spread * torch.randn(n, -(-k // 32), generator=g)).round()).repeat_interleave(32, 1)[:, :k]


def _packed(n, k, seed, spread=3.0):
    return _mx4().quantize(_random(n, k, seed, spread).cuda())


def _check_product(y, x, w, dtype):
    """y against the exact product of float64 matrices x and w."""
    exact, size = x @ w.t(), x.abs() @ w.abs().t()
    bound = x.shape[1] * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * exact.abs() + torch.finfo(dtype).smallest_normal
    off = (y.cpu().double() - exact).abs()
    assert bool((off <= bound).all()), f"{(off / bound).max()} of the bound at {tuple(y.shape)} x {x.shape[1]}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rule", ["floor", "ceil"])
@pytest.mark.parametrize("dim", [-1, -2])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (2, 31), (3, 33), (33, 3), (65, 257), (130, 515), (7, 1024), (259, 66), (64, 256)])
def test_quantize_is_the_definition(dtype, rule, dim, shape):
    mx4 = _mx4()
    x = _random(*shape, seed=shape[0] * 1000 + shape[1]).to(dtype)
    # values on and next to the borders between codes, and a block's largest on both sides of 6
    x.view(-1)[: min(x.numel(), 9)] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -2.5], dtype=dtype)[: min(x.numel(), 9)]
    q = mx4.quantize(x.cuda(), dim, rule)
    codes, scales = ref.unpack(q)
    want = ref.quantize(x if dim == -1 else x.t(), rule)
    assert torch.equal(scales, want[1]) and torch.equal(codes, want[0])
    assert torch.equal(mx4.dequantize(q).cpu().double(), ref.values(*want, q.length))


@pytest.mark.parametrize("dim", [-1, -2])
def test_quantize_edges(dim):
    mx4 = _mx4()
    inf, nan, tiny, big = float("inf"), float("nan"), 2.0 ** -149, 3.4028234663852886e38
    x = torch.zeros(14, 64)
    for i, v in enumerate([0.0, -0.0, tiny, 3 * tiny, 2.0 ** -126, 1.75 * 2.0 ** -125, 2.0 ** -125, 2.0 ** -124, big, -big, inf, -inf, nan, 1.5]):
        x[i, 5] = v
        x[i, 40] = -v / 3
    x = x if dim == -1 else x.t().contiguous()
    for rule in ("floor", "ceil"):
        q = mx4.quantize(x.cuda(), dim, rule)
        codes, scales = ref.unpack(q)
        want = ref.quantize(x if dim == -1 else x.t(), rule)
        assert torch.equal(scales, want[1]) and torch.equal(codes, want[0])
        back, values = mx4.dequantize(q).cpu(), ref.values(*want, 64).float()   # 4 * 2^126, nearest to the largest number, is an infinity
        assert torch.equal(torch.isnan(back), torch.isnan(values)) and torch.equal(back.nan_to_num(), values.nan_to_num())
        assert bool(torch.isnan(back[10:13]).all()) and not bool(torch.isnan(back[:10]).any()) and bool(torch.isfinite(back[13]).all())


@pytest.mark.parametrize("dim", [-1, -2])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strides_and_offsets(dim, dtype):
    """Rows with a pitch, and starts that are not aligned for wide loads, take the same values."""
    mx4 = _mx4()
    big = _random(40, 700, 5).to(dtype).cuda()
    for view in (big[3:30, 1:600], big[:, 8:520], big[5:6, 3:99], big[::2, 2:98]):
        got, want = mx4.quantize(view, dim), mx4.quantize(view.contiguous(), dim)
        for a, b in zip(ref.unpack(got), ref.unpack(want)):
            assert torch.equal(a, b)


def test_quantize_stack_is_each_matrix():
    mx4 = _mx4()
    x = _random(3 * 50, 100, 6).reshape(3, 50, 100).cuda()
    for dim in (-1, -2):
        q = mx4.quantize(x, dim, "ceil")
        for i in range(3):
            one = mx4.quantize(x[i], dim, "ceil")
            for a, b in zip(ref.unpack(mx4.Mx4(q.codes[i], q.scales[i], q.length)), ref.unpack(one)):
                assert torch.equal(a, b)


def test_nothing_is_written_behind_the_blocks():
    from ozaki_blackwell_b200._lib import lib
    x = _random(5, 40, 7).cuda()
    for by_rows, nvec, length in ((1, 5, 40), (0, 40, 5)):
        codes = torch.full((nvec + 1, 64), 0xAB, dtype=torch.uint8, device="cuda")
        scales = torch.full((nvec + 1, 16), 0xCD, dtype=torch.uint8, device="cuda")
        assert lib.ozb_mx4_quantize(x.data_ptr(), 0, nvec, length, 40, by_rows, 0, None, None, 0, 0, 1, 0, codes.data_ptr(), 64, 0, scales.data_ptr(), 16, 0, None) == 0
        torch.cuda.synchronize()
        blocks = -(-length // 32)
        assert bool((codes[nvec] == 0xAB).all()) and bool((codes[:, 16 * blocks:] == 0xAB).all())
        assert bool((scales[nvec] == 0xCD).all()) and bool((scales[:, blocks:] == 0xCD).all())


@pytest.mark.parametrize("dim", [-1, -2])
@pytest.mark.parametrize("h,dtype", [(130, torch.float32), (1600, torch.bfloat16), (33, torch.float16)])
def test_quantize_of_routed_rows(dim, h, dtype):
    from ozaki_blackwell_b200 import experts
    mx4 = _mx4()
    tokens, top = 90, 3
    x = _random(tokens, h, 8).to(dtype).cuda()
    g = torch.Generator().manual_seed(h)
    r = experts.sort(torch.randint(-1, 5, (tokens, top), generator=g).cuda(), 5, 64)
    for src in (x, _random(tokens, h + 9, 8).to(dtype).cuda()[:, 3: 3 + h]):
        rows = experts.gather(src, r).cpu()
        got, want = ref.unpack(mx4.quantize(src, dim, "ceil", routing=r)), ref.quantize(rows if dim == -1 else rows.t(), "ceil")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dim", [-1, -2])
def test_quantize_takes_any_routing_without_leaving_its_arrays(dim):
    from ozaki_blackwell_b200 import experts
    mx4 = _mx4()
    x = _random(3, 64, 9).cuda()
    rows = torch.tensor([[0, 5], [-3, 2 ** 31 - 1], [-1, 1]], dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 5, 6, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    r = experts.Routing(torch.zeros(2, dtype=torch.int32, device="cuda"), rows, slots)
    want = torch.zeros(5, 64)
    want[0], want[1] = x[0].cpu(), x[2].cpu()
    got, want = ref.unpack(mx4.quantize(x, dim, routing=r)), ref.quantize(want if dim == -1 else want.t())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_dequantize_every_code_and_scale(dtype):
    mx4 = _mx4()
    codes = torch.arange(16, dtype=torch.uint8).repeat(2).repeat(256, 1)
    packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).cuda()
    scales = torch.zeros(256, 16, dtype=torch.uint8, device="cuda")
    scales[:, 0] = torch.arange(256, dtype=torch.uint8)
    got = mx4.dequantize(mx4.Mx4(packed, scales, 32), dtype).cpu()
    want = ref.values(codes, scales[:, :1], 32).to(torch.float32).to(dtype)   # exact in FP32 (or an overflow), then one rounding
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    out = torch.full((256, 40), 7.0, dtype=dtype, device="cuda")
    mx4.dequantize(mx4.Mx4(packed, scales, 31), dtype, out=out[:, 1:32])
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 32:] == 7).all()) and torch.equal(out[:, 1:32].cpu().nan_to_num(), want[:, :31].nan_to_num())


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 128, 32), (1, 2048, 4096), (2, 130, 33), (15, 127, 64), (16, 129, 65), (17, 256, 255), (31, 64, 256), (33, 300, 257),
                                   (64, 128, 2085), (65, 1, 511), (128, 400, 512), (129, 257, 1000), (300, 70, 1537), (512, 384, 96), (513, 640, 288),
                                   (700, 130, 2049), (3, 640, 16384), (150, 9500, 96), (300, 6000, 500), (129, 7200, 1100), (1100, 3070, 300), (2060, 1550, 1025),
                                   (513, 5000, 64), (40, 1024, 8192), (4, 300, 16400), (90, 500, 9000), (17, 130, 20000)])
def test_product(shape):
    m, n, k = shape
    mx4 = _mx4()
    for dtype in TYPES:
        spread = 0.0 if dtype == torch.float16 else 3.0    # sums stay below 65504
        x, w = _packed(m, k, 1, spread), _packed(n, k, 2, spread)
        _check_product(mx4.matmul(x, w, dtype), ref.of(x), ref.of(w), dtype)
    _status()


def test_product_of_far_scales():
    """Scales over the whole range of the format whose products stay within FP32, each row of X at another one."""
    mx4 = _mx4()
    m, n, k = 40, 150, 200
    x, w = _packed(m, k, 3, 0.0), _packed(n, k, 4, 0.0)
    far = (torch.arange(m) % 20 - 10) * 12
    x.scales.copy_((x.scales.cpu().int() + far[:, None]).clamp(0, 254).to(torch.uint8))
    _check_product(mx4.matmul(x, w, torch.float32), ref.of(x), ref.of(w), torch.float32)


def test_product_with_blocks_that_are_not_numbers():
    mx4 = _mx4()
    m, n, k = 20, 200, 320
    x, w = _packed(m, k, 5), _packed(n, k, 6)
    x.scales[3, 9], w.scales[100, 0] = 255, 255
    y = mx4.matmul(x, w, torch.float32).cpu()
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[3], bad[:, 100] = True, True
    assert torch.equal(torch.isnan(y), bad)
    # what lies behind the last block of a row is not read into the product
    x2, w2 = _packed(m, 40, 7), _packed(n, 40, 8)
    want = mx4.matmul(x2, w2, torch.float32)
    for q in (x2, w2):
        q.scales[:, 2:] = 255
    assert torch.equal(mx4.matmul(x2, w2, torch.float32), want)


def test_product_pitches_and_out():
    mx4 = _mx4()
    m, n, k = 37, 150, 300
    x, w = _packed(m, k, 9), _packed(n, k, 10)

    def spread(q):
        c = torch.full((q.codes.shape[0], 224), 0xFF, dtype=torch.uint8, device="cuda")
        s = torch.full((q.codes.shape[0], 32), 0xFF, dtype=torch.uint8, device="cuda")
        c[:, 16: 16 + q.codes.shape[1]], s[:, 16: 16 + 10] = q.codes, q.scales[:, :10]
        return mx4.Mx4(c[:, 16: 16 + q.codes.shape[1]], s[:, 16:], k)

    out = torch.full((m + 1, n + 9), 3.0, dtype=torch.bfloat16, device="cuda")
    want = mx4.matmul(x, w)
    got = mx4.matmul(spread(x), spread(w), out=out[:m, 4: 4 + n])
    assert torch.equal(got, want)
    assert bool((out[m] == 3).all()) and bool((out[:, :4] == 3).all()) and bool((out[:, 4 + n:] == 3).all())


@pytest.mark.parametrize("offsets", [[0, 5, 5, 30, 47], [0, 0, 0, 0, 0], [3, 3, 40, 41, 44], [0, 47, 47, 47, 47], [0, 16, 32, 40, 47]])
@pytest.mark.parametrize("k", [64, 700])
def test_grouped_product(offsets, k):
    mx4 = _mx4()
    r, n, groups = 47, 200, 4
    x, w = _packed(r, k, 11), [_packed(n, k, 12 + g) for g in range(groups)]
    stack = mx4.Mx4(torch.stack([q.codes for q in w]), torch.stack([q.scales for q in w]), k)
    out = torch.full((r, n), 9.0, dtype=torch.float32, device="cuda")
    mx4.grouped_matmul(x, stack, torch.tensor(offsets, dtype=torch.int32, device="cuda"), torch.float32, out=out)
    xs = ref.of(x)
    inside = torch.zeros(r, dtype=torch.bool)
    for g in range(groups):
        lo, hi = offsets[g], offsets[g + 1]
        inside[lo:hi] = True
        if hi > lo:
            _check_product(out[lo:hi], xs[lo:hi], ref.of(w[g]), torch.float32)
    assert bool((out.cpu()[~inside] == 9).all())
    _status()


@pytest.mark.parametrize("groups,r,n", [(1024, 500, 130), (3, 2000, 130), (40, 900, 130), (64, 2100, 130), (4, 1600, 3100), (5, 900, 2000), (2, 2500, 6000), (1, 300, 6000)])
def test_grouped_product_many_groups_and_wide_segments(groups, r, n):
    mx4 = _mx4()
    k = 96
    g = torch.Generator().manual_seed(groups)
    cuts = torch.sort(torch.randint(0, r + 1, (groups - 1,), generator=g)).values
    offsets = [0] + cuts.tolist() + [r]
    x = _packed(r, k, 13)
    w = mx4.quantize(_random(groups * n, k, 14).reshape(groups, n, k).cuda())
    out = torch.full((r + 2, n), 7.0, dtype=torch.bfloat16, device="cuda")
    mx4.grouped_matmul(x, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), torch.bfloat16, out=out[1: r + 1])
    assert bool((out[[0, r + 1]] == 7).all())
    xs, ws = ref.of(x), ref.of(w)
    for i in range(groups):
        if offsets[i + 1] > offsets[i]:
            _check_product(out[1 + offsets[i]: 1 + offsets[i + 1]], xs[offsets[i]: offsets[i + 1]], ws[i], torch.bfloat16)
    _status()


def test_grouped_product_takes_any_offsets_without_leaving_its_arrays():
    """Offsets out of range or out of order are cut: rows that no cut segment holds stay as they were."""
    mx4 = _mx4()
    r, n, k = 33, 140, 64
    x, w = _packed(r, k, 15), mx4.quantize(_random(3 * n, k, 16).reshape(3, n, k).cuda())
    guard = torch.full((r + 2, n), 5.0, device="cuda")
    mx4.grouped_matmul(x, w, torch.tensor([-7, 10, 4, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), torch.float32, out=guard[1: r + 1])
    xs, ws = ref.of(x), ref.of(w)
    assert bool((guard[0] == 5).all()) and bool((guard[r + 1] == 5).all())
    _check_product(guard[1:5], xs[:4], ws[0], torch.float32)      # rows 0 .. 3 are the first segment's alone
    _check_product(guard[11: r + 1], xs[10:], ws[2], torch.float32)
    _status()


@pytest.mark.parametrize("offsets", [[0, 64, 64, 320, 448], [0, 0, 0, 0, 0], [64, 128, 192, 256, 320], [0, 448, 448, 448, 448], [128, 128, 128, 128, 192]])
def test_segment_product(offsets):
    mx4 = _mx4()
    m, n, r = 150, 210, 448
    a, b = _packed(m, r, 17), _packed(n, r, 18)
    y = mx4.segment_matmul(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), torch.float32)
    av, bv = ref.of(a), ref.of(b)
    for g in range(4):
        lo, hi = offsets[g], offsets[g + 1]
        if hi == lo:
            assert bool((y[g] == 0).all())
        else:
            _check_product(y[g], av[:, lo:hi], bv[:, lo:hi], torch.float32)
    # a segment does not see what its neighbours hold, numbers or not
    a.scales[:, lo // 32: hi // 32] = 255
    y2 = mx4.segment_matmul(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), torch.float32)
    assert torch.equal(y2[:3], y[:3])
    _status()


@pytest.mark.parametrize("m,n,groups", [(200, 400, 16), (600, 1000, 16), (300, 100, 64), (40, 900, 32), (130, 400, 20)])
def test_segment_product_of_many(m, n, groups):
    mx4 = _mx4()
    g = torch.Generator().manual_seed(m)
    lengths = torch.randint(0, 12, (groups,), generator=g) * 64
    offsets = [0] + lengths.cumsum(0).tolist()
    r = max(64, offsets[-1])
    a, b = _packed(m, r, 19), _packed(n, r, 20)
    y = mx4.segment_matmul(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), torch.bfloat16)
    av, bv = ref.of(a), ref.of(b)
    for i in range(groups):
        lo, hi = offsets[i], offsets[i + 1]
        _check_product(y[i], av[:, lo:hi], bv[:, lo:hi], torch.bfloat16)
    _status()


def test_streams_and_graphs():
    """Calls on two streams at once, and a captured graph replayed on other inputs, give what single calls give."""
    mx4 = _mx4()
    xs = [_random(40, 1000, 20 + i).cuda().bfloat16() for i in range(4)]
    w = _packed(500, 1000, 30)
    want = [mx4.matmul(mx4.quantize(x), w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * 4
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = mx4.matmul(mx4.quantize(x), w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a chain over two streams, each step behind an event of the other's last, on buffers that are written again and again
    a, b = streams
    buf, out, done = xs[0].clone(), torch.empty_like(want[0]), torch.cuda.Event()
    torch.cuda.synchronize()
    for i in list(range(4)) * 8:
        with torch.cuda.stream(a):
            a.wait_event(done)
            buf.copy_(xs[i])
            q = mx4.quantize(buf)
            ready = torch.cuda.Event()
            ready.record(a)
        with torch.cuda.stream(b):
            b.wait_event(ready)
            mx4.matmul(q, w, out=out)
            keep = out.clone()
            done = torch.cuda.Event()
            done.record(b)
        b.synchronize()
        assert torch.equal(keep, want[i])
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mx4.matmul(mx4.quantize(x), w)
    for i in (2, 1, 3):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(y, want[i])


@pytest.mark.parametrize("m,n", [(8, 8), (300, 6000), (1100, 3100)])
def test_first_product_of_a_process_in_a_capture(m, n):
    import subprocess
    import sys
    code = (f"import torch; from ozaki_blackwell_b200 import mx4; x, w = torch.randn({m}, 64, device='cuda'), torch.randn({n}, 64, device='cuda'); g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n    q, p = mx4.quantize(x), mx4.quantize(w); y = mx4.matmul(q, p, torch.float32)\n"
            "g.replay(); a, b = (mx4.dequantize(t).double() for t in (q, p)); assert torch.allclose(y.double(), a @ b.t(), rtol=1e-5, atol=1e-4)")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]


def test_offsets_past_32_bits():
    """An output of more than 2^32 bytes, and codes behind them, are addressed in 64 bits."""
    mx4 = _mx4()
    m, n, k = 70000, 33000, 32
    x, w = _packed(m, k, 40), _packed(n, k, 41)
    y = mx4.matmul(x, w)
    rows = torch.tensor([0, 1, 32767, 65100, 65101, m - 1])
    _check_product(y[rows.cuda()], ref.of(mx4.Mx4(x.codes[rows.cuda()], x.scales[rows.cuda()], k)), ref.of(w), torch.bfloat16)
    big = y[:, :n - 1]
    q = mx4.quantize(big)
    one = mx4.quantize(big[m - 1:].contiguous())
    for a, b in zip(ref.unpack(mx4.Mx4(q.codes[m - 1:], q.scales[m - 1:], q.length)), ref.unpack(one)):
        assert torch.equal(a, b)


def test_refusals():
    mx4 = _mx4()
    x = torch.randn(4, 64, device="cuda")
    q = mx4.quantize(x)
    with pytest.raises(TypeError):
        mx4.quantize(x.double())
    with pytest.raises(TypeError):
        mx4.matmul(q, q, torch.float64)
    with pytest.raises(ValueError):
        mx4.quantize(x.t())
    with pytest.raises(ValueError):
        mx4.quantize(x, dim=0)
    with pytest.raises(ValueError):
        mx4.quantize(x, rule="nearest")
    with pytest.raises(ValueError):
        mx4.matmul(q, mx4.quantize(torch.randn(4, 65, device="cuda")))
    with pytest.raises(ValueError):
        mx4.matmul(mx4.Mx4(q.codes, q.scales[:3], 64), q)
    with pytest.raises(ValueError):
        mx4.matmul(mx4.Mx4(q.codes, q.scales, 65), q)
    with pytest.raises(ValueError):
        mx4.matmul(q, q, out=torch.empty(4, 4, device="cuda"))
    with pytest.raises(RuntimeError):
        mx4.matmul(mx4.Mx4(q.codes.view(-1)[8:-8].view(-1)[:32].view(1, 32), q.scales[:1], 64), q)   # codes off 16 bytes
    with pytest.raises(RuntimeError):
        mx4.matmul(q, mx4.Mx4(q.codes[:0], q.scales[:0], 64))                                          # nothing to compute
    with pytest.raises(ValueError):
        mx4.segment_matmul(q, q, torch.tensor([0, 64], device="cuda"))                                 # int64
    stack = mx4.quantize(x.reshape(2, 2, 64))
    with pytest.raises(ValueError):
        mx4.grouped_matmul(q, stack, torch.tensor([0, 4], dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        mx4.grouped_matmul(q, stack, torch.tensor([0, 2, 4], dtype=torch.int32))

"""Tokens by expert and back on the GPU: the sort against a slot-by-slot one, rows and sums against 64 bits, and the whole layer with
its gradients.

Tolerances: a sum of n terms in FP32 is off by at most n 2^-24 of the sum of their magnitudes (n - 1 roundings of partial sums and one
of each product, every one by half a unit); the output type adds finfo(type).eps / 2 of the value."""
import pytest
import torch

import mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _experts():
    from ozaki_blackwell_b200 import experts
    return experts


def _ids(tokens, top, experts, seed, drop=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, top), generator=g)
    bad = torch.tensor([-1, experts, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (tokens, top), generator=g)]
    return torch.where(torch.rand(tokens, top, generator=g) < drop, bad, ids)


@pytest.mark.parametrize("tokens,top,experts", [(1, 1, 1), (1, 8, 4), (3, 2, 1024), (33, 3, 7), (256, 8, 64), (257, 8, 64), (2048, 1, 3), (2049, 1, 1000), (3000, 7, 129), (20000, 4, 256)])
@pytest.mark.parametrize("align", [1, 7, 64])
def test_sort(tokens, top, experts, align):
    ids = _ids(tokens, top, experts, tokens + top)
    offsets, rows = ref.sort(ids, experts, align) if tokens * top * experts < 3e6 else _fast_sort(ids, experts, align)
    for dtype in (torch.int32, torch.int64):
        r = _experts().sort(ids.to(dtype).cuda(), experts, align)
        assert r.offsets.tolist() == offsets
        assert r.rows.reshape(-1).tolist() == rows
        slots = [-1] * r.slots.numel()
        for s, row in enumerate(rows):
            if row >= 0:
                slots[row] = s
        assert r.slots.tolist() == slots


def _fast_sort(ids, experts, align):
    flat = ids.reshape(-1).tolist()
    count = [0] * experts
    place = []
    for e in flat:
        if 0 <= e < experts:
            place.append(count[e])
            count[e] += 1
        else:
            place.append(-1)
    offsets = [0]
    for c in count:
        offsets.append(offsets[-1] + -(-c // align) * align)
    return offsets, [offsets[e] + p if p >= 0 else -1 for e, p in zip(flat, place)]


@pytest.mark.parametrize("slots,experts", [(256 * 1024, 40), (256 * 1024 + 1, 1024), (300000, 3), (3000001, 77)])
def test_sort_of_many(slots, experts):
    """Over 256 chunks of 1024 slots the counts go through a scan of their own."""
    ids = _ids(slots, 1, experts, slots).cuda()
    r = _experts().sort(ids, experts, 8)
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=experts + 1)
    offsets = torch.nn.functional.pad(((counts[:experts] + 7) // 8 * 8).cumsum(0), (1, 0))
    place = offsets[key[order]] + torch.arange(slots, device="cuda") - (counts.cumsum(0) - counts)[key[order]]
    rows = torch.full((slots,), -1, device="cuda").scatter(0, order, torch.where(key[order] < experts, place, -1))
    assert torch.equal(r.offsets.long(), offsets) and torch.equal(r.rows.reshape(-1).long(), rows)
    kept = rows >= 0
    want = torch.full((r.slots.numel(),), -1, device="cuda")
    want[rows[kept]] = torch.arange(slots, device="cuda")[kept]
    assert torch.equal(r.slots.long(), want)


@pytest.mark.parametrize("what", ["all dropped", "one expert", "every token the same expert twice"])
def test_sort_extremes(what):
    tokens, top, experts = 700, 4, 33
    ids = {"all dropped": torch.full((tokens, top), -1), "one expert": torch.full((tokens, top), 32),
           "every token the same expert twice": torch.tensor([5, 5, 0, 5]).repeat(tokens, 1)}[what]
    offsets, rows = ref.sort(ids, experts, 32)
    r = _experts().sort(ids.int().cuda(), experts, 32)
    assert r.offsets.tolist() == offsets and r.rows.reshape(-1).tolist() == rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top,h", [(1, 1, 1), (5, 2, 7), (19, 3, 128), (40, 8, 2050), (130, 1, 1000)])
def test_rows_there_and_back(dtype, tokens, top, h):
    ex = _experts()
    r = ex.sort(_ids(tokens, top, 6, h).cuda(), 6, 16)
    g = torch.Generator().manual_seed(h)
    wide = torch.randn(tokens, h + 24, generator=g).to(dtype).cuda()
    weights = torch.randn(tokens, top, generator=g).cuda()
    rows, slots = r.rows.cpu().long(), r.slots.cpu().long()
    for x in (wide[:, :h], wide[:, 8: 8 + h], wide[:, 3: 3 + h], wide[:, :h].contiguous()):
        y = ex.gather(x, r)
        want = torch.where(slots[:, None] >= 0, x.cpu()[slots.clamp(min=0) // top], torch.zeros((), dtype=dtype))
        assert torch.equal(y.cpu(), want)

    R = slots.numel()
    zw = torch.randn(R, h + 16, generator=g).to(dtype).cuda()
    zw[(r.slots < 0)] = float("nan")     # rows that no slot uses are not read into anything
    for z in (zw[:, :h], zw[:, 5: 5 + h]):
        zz = torch.where(rows[..., None] >= 0, z.cpu().double()[rows.clamp(min=0)], 0.0)
        for wt in (weights, None):
            w64 = weights.cpu().double() if wt is not None else torch.ones(tokens, top, dtype=torch.float64)
            exact, size = (zz * w64[..., None]).sum(1), (zz.abs() * w64.abs()[..., None]).sum(1)
            bound = (top + 1) * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * exact.abs() + torch.finfo(dtype).tiny
            assert bool(((ex.combine(z, r, wt).cpu().double() - exact).abs() <= bound).all())

            dy = wide[:, 1: 1 + h]
            dz, dw = ex.combine_grad(dy, z, r, wt)
            d = dy.cpu().double()
            f = torch.where(slots >= 0, w64.reshape(-1)[slots.clamp(min=0)], 0.0)
            want = f[:, None] * d[slots.clamp(min=0) // top]
            off = (dz.cpu().double() - want).abs()
            assert bool((off <= (torch.finfo(dtype).eps / 2 + 2.0 ** -24) * want.abs() + torch.finfo(dtype).tiny).all())
            assert bool((dz.cpu()[slots < 0] == 0).all())
            dots, mags = (zz * d[:, None]).sum(-1), (zz.abs() * d.abs()[:, None]).sum(-1)
            assert bool(((dw.cpu().double() - dots).abs() <= (h + 1) * 2.0 ** -24 * mags + 1e-37).all())
            assert bool((dw.cpu()[rows < 0] == 0).all())


def test_combine_is_linear_so_its_gradient_is_its_difference():
    ex = _experts()
    tokens, top, h = 11, 3, 40
    r = ex.sort(_ids(tokens, top, 5, 3).cuda(), 5, 4)
    z, dy = (torch.randint(-8, 9, (n, h)).float().cuda() for n in (r.slots.numel(), tokens))   # small whole numbers: every sum is exact
    weights = torch.randint(-4, 5, (tokens, top)).float().cuda()
    dz, dw = ex.combine_grad(dy, z, r, weights)
    loss = lambda z, w: (ex.combine(z, r, w) * dy).sum().item()  # noqa: E731
    base = loss(z, weights)
    for t in range(tokens):
        for j in range(top):
            w = weights.clone()
            w[t, j] += 1
            assert loss(z, w) - base == dw[t, j].item()
    for i, c in [(0, 0), (3, 7), (r.slots.numel() - 1, 39), (8, 20)]:
        zz = z.clone()
        zz[i, c] += 1
        assert loss(zz, weights) - base == dz[i, c].item()


def test_indices_out_of_range_are_none():
    ex = _experts()
    tokens, top, h = 6, 2, 72
    z, dy = torch.randn(5, h, device="cuda"), torch.randn(tokens, h, device="cuda")
    rows = torch.tensor([[0, 5], [-3, 2 ** 31 - 1], [-1, 1], [-2 ** 31, 9], [-1, 2 ** 30], [6, -1]], dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 5, 12, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    r = ex.Routing(torch.zeros(2, dtype=torch.int32, device="cuda"), rows, slots)
    y = ex.combine(z, r)
    assert torch.equal(y[0], z[0]) and torch.equal(y[2], z[1]) and bool((y[[1, 3, 4, 5]] == 0).all())
    guard = torch.full((7, h), 5.0, device="cuda")
    x = ex.gather(dy, r, out=guard[1:6])
    assert torch.equal(x[0], dy[0]) and torch.equal(x[1], dy[2]) and bool((x[2:] == 0).all()) and bool((guard[[0, 6]] == 5).all())
    dz, dw = ex.combine_grad(dy, z, r)
    assert torch.equal(dz[0], dy[0]) and torch.equal(dz[1], dy[2]) and bool((dz[2:] == 0).all())
    assert bool((dw[[0, 1, 3, 4, 5], [1, 0, 1, 0, 0]] == 0).all())


def _layer(x, w, ids, weights, z_type):
    """The layer in 64 bits on values that the 4-bit format holds: y and z by slot."""
    tokens, top = ids.shape
    y, z = torch.zeros(tokens, w.shape[1], dtype=torch.float64), torch.zeros(tokens, top, w.shape[1], dtype=torch.float64)
    for t in range(tokens):
        for j in range(top):
            e = int(ids[t, j])
            if 0 <= e < len(w):
                z[t, j] = (w[e] @ x[t]).to(z_type).double()
                y[t] += weights[t, j] * z[t, j]
    return y, z


@pytest.mark.parametrize("tokens,top,experts,n,k", [(1, 1, 1, 1, 1), (4, 4, 16, 130, 300), (70, 2, 5, 96, 64), (300, 3, 4, 200, 257)])
def test_layer_and_its_gradients(tokens, top, experts, n, k):
    """Everything together, as a program uses it. x, W, dy are such that the 4-bit format holds them exactly (every block's largest
    value is 4, the others are codes), so the layer is the plain one, its gradients are the formula's, and y's error is that of
    rounding z and y (each finfo.eps / 2) and of FP32 sums."""
    from ozaki_blackwell_b200 import mx4
    ex = _experts()
    g = torch.Generator().manual_seed(tokens)

    def exact4(*shape):
        v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0])[torch.randint(0, 7, shape, generator=g)] * torch.where(torch.rand(shape, generator=g) < 0.5, -1, 1)
        v[..., ::16] = 4.0          # a largest value in every block along a row
        v.reshape(-1, shape[-1])[::16] = 4.0   # ... and nearly always along a column; what is not held exactly is checked as rounded
        return v

    x, dy, w = exact4(tokens, k), exact4(tokens, n), exact4(experts, n, k)
    ids, weights = _ids(tokens, top, experts, 5, 0.15), torch.tensor([0.5, 1.0, 2.0])[torch.randint(0, 3, (tokens, top), generator=g)]
    for dtype in (torch.bfloat16, torch.float32):
        half = torch.finfo(dtype).eps / 2
        xg, dyg, wg = x.to(dtype).cuda(), dy.to(dtype).cuda(), w.cuda()
        wq, wt = mx4.quantize(wg), mx4.quantize(wg, dim=-2)
        y, z, r = ex.matmul(xg, wq, ids.cuda(), weights.cuda(), keep=True)
        want, zs = _layer(x.double(), w.double(), ids, weights.double(), dtype)
        size = (zs.abs() * weights.double()[..., None]).sum(1)
        bound = (2 * half + (k + top + 1) * 2.0 ** -23) * size + half * want.abs()
        assert bool(((y.cpu().double() - want).abs() <= bound).all())
        # inference keeps no padding and gives the same numbers
        assert torch.equal(ex.matmul(xg, wq, ids.cuda(), weights.cuda()), y)

        dx, dweights, dw = ex.matmul_grad(dyg, xg, z, wt, r, weights.cuda())
        slots, z64 = r.slots.cpu().long(), z.cpu().double()
        kept = slots >= 0
        of = slots.clamp(min=0) // top
        dz = torch.where(kept[:, None], weights.double().reshape(-1)[slots.clamp(min=0)][:, None] * dy.double()[of], 0.0)
        z64 = torch.where(kept[:, None], z64, 0.0)
        dots = torch.zeros(tokens * top, dtype=torch.float64)
        dots[slots[kept]] = (dy.double()[of] * z64).sum(1)[kept]
        mags = (dy.double().abs()[of] * z64.abs()).sum(1).max()
        assert bool(((dweights.cpu().double().reshape(-1) - dots).abs() <= (n + 1) * 2.0 ** -24 * mags + 1e-30).all())
        rows4 = lambda m: ref.values(*ref.quantize(m.float()), m.shape[1])  # noqa: E731
        wt64, offsets = ref.of(wt), r.offsets.tolist()
        dzr, dzc, xc = rows4(dz), rows4(dz.t()), rows4(torch.where(kept[:, None], x.double()[of], 0.0).t())
        want_dx, size_dx = torch.zeros(tokens, k, dtype=torch.float64), torch.zeros(tokens, k, dtype=torch.float64)
        for e in range(experts):
            lo, hi = offsets[e], offsets[e + 1]
            part, mag = dzr[lo:hi] @ wt64[e].t(), dzr[lo:hi].abs() @ wt64[e].abs().t()
            rows = [i for i in range(lo, hi) if kept[i]]
            want_dx.index_add_(0, of[rows], part[[i - lo for i in rows]])
            size_dx.index_add_(0, of[rows], mag[[i - lo for i in rows]])
            want_dw, size_dw = dzc[:, lo:hi] @ xc[:, lo:hi].t(), dzc[:, lo:hi].abs() @ xc[:, lo:hi].abs().t()
            off = (dw[e].cpu().double() - want_dw).abs()
            assert bool((off <= half * want_dw.abs() + (hi - lo + 1) * 2.0 ** -23 * size_dw).all())
        off = (dx.cpu().double() - want_dx).abs()
        assert bool((off <= (2 * half + (n + top + 1) * 2.0 ** -23) * size_dx).all())


def test_layer_captured_and_replayed():
    from ozaki_blackwell_b200 import mx4
    ex = _experts()
    g = torch.Generator().manual_seed(1)
    tokens, top, experts, n, k = 9, 2, 6, 200, 320
    w = torch.randn(experts, n, k, generator=g).cuda()
    wq, wt = mx4.quantize(w), mx4.quantize(w, dim=-2)
    sets = [(torch.randn(tokens, k, generator=g).cuda().bfloat16(), torch.randint(-1, experts, (tokens, top), generator=g).cuda(),
             torch.rand(tokens, top, generator=g).cuda(), torch.randn(tokens, n, generator=g).cuda().bfloat16()) for _ in range(3)]

    def step(x, ids, weights, dy):
        y, z, r = ex.matmul(x, wq, ids, weights, keep=True)
        return (y, *ex.matmul_grad(dy, x, z, wt, r, weights))

    want = [[t.clone() for t in step(*s)] for s in sets]
    held = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for i in (1, 2, 0):
        for a, b in zip(held, sets[i]):
            a.copy_(b)
        graph.replay()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


def test_refusals():
    ex = _experts()
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    r = ex.sort(ids, 3)
    x, z = torch.randn(4, 8, device="cuda"), torch.randn(8, 8, device="cuda")
    for bad in (ids.float(), ids.reshape(-1), ids.t(), ids.cpu()):
        with pytest.raises(ValueError):
            ex.sort(bad, 3)
    for experts, align in ((0, 1), (1025, 1), (3, 0), (3, 257)):
        with pytest.raises(ValueError):
            ex.sort(ids, experts, align)
    with pytest.raises(ValueError):
        ex.gather(torch.randn(5, 8, device="cuda"), r)
    with pytest.raises(TypeError):
        ex.gather(x.double(), r)
    with pytest.raises(ValueError):
        ex.combine(z, r, torch.ones(4, 2, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError):
        ex.combine_grad(x.bfloat16(), z, r)
    with pytest.raises(ValueError):
        ex.combine_grad(x, z[:7], r)
    with pytest.raises(ValueError):
        ex.gather(x, ex.Routing(r.offsets, r.rows.long(), r.slots))
    with pytest.raises(ValueError):
        ex.matmul_grad(x, x, z, None, r)      # segments that are not padded to 64


def test_gradient_refuses_offsets_of_other_experts():
    from ozaki_blackwell_b200 import mx4
    ex = _experts()
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    x, dy, w = torch.randn(4, 64, device="cuda"), torch.randn(4, 32, device="cuda"), torch.randn(3, 32, 64, device="cuda")
    wt = mx4.quantize(w, dim=-2)
    _, z, r = ex.matmul(x, mx4.quantize(w), ids, keep=True)
    for offsets in (r.offsets.long(), r.offsets[:-1], r.offsets.cpu(), r.offsets.reshape(1, -1)):
        with pytest.raises(ValueError):
            ex.matmul_grad(dy, x, z, wt, ex.Routing(offsets, r.rows, r.slots, r.align))
    assert len(ex.matmul_grad(dy, x, z, wt, r)) == 3

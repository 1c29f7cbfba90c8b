"""Calls as programs make them: captured over forked streams, replayed two at a time, on operands that are views, at the ends of the
scales' range, over more than 2^31 elements, on routings that leave experts without tokens or one with all of them."""
import pytest
import torch

import mx4_ref as ref

pytestmark = pytest.mark.gpu
TABLE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _codes(seed, *shape):
    """Values that the format holds exactly, whatever the largest of a block."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.tensor(TABLE, device="cuda")[torch.randint(0, 16, shape, generator=g, device="cuda")]


def test_capture_over_forked_streams():
    from ozaki_blackwell_b200 import mx4
    m, n, k = 70, 300, 500
    x, w = _codes(1, m, k), _codes(2, n, k)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            q = mx4.quantize(w)
        p = mx4.quantize(x)
        main.wait_stream(side)
        y = mx4.matmul(p, q, torch.float32)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            back = mx4.dequantize(mx4.quantize(y, dim=-2))
        yt = mx4.matmul(q, p, torch.float32)
        main.wait_stream(side)
    for seed in range(3, 8):
        x.copy_(_codes(seed, m, k))
        w.copy_(_codes(seed + 10, n, k))
        graph.replay()
        want = x.double() @ w.double().t()
        assert torch.equal(y, want.float()) and torch.equal(yt, y.t())
        assert torch.equal(back, mx4.dequantize(mx4.quantize(y, dim=-2)))


def test_two_graphs_at_once():
    """Each has its own maps and workspaces: replayed side by side they do not meet."""
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    tokens, top, experts, n, k = 200, 2, 6, 320, 256
    streams, graphs, held, got, want = [torch.cuda.Stream() for _ in range(2)], [], [], [], []
    w = _codes(1, experts, n, k)
    wq, wt = mx4.quantize(w), mx4.quantize(w, dim=-2)
    weights = torch.full((tokens, top), 2.0, device="cuda")
    for i in range(2):
        x, dy = _codes(10 + i, tokens, k), _codes(20 + i, tokens, n)
        ids = torch.randint(0, experts, (tokens, top), generator=torch.Generator().manual_seed(i)).cuda()
        held.append((x, dy, ids))

        def step(x=x, dy=dy, ids=ids):
            y, z, r = ex.matmul(x, wq, ids, weights, keep=True)
            return (y, *ex.matmul_grad(dy, x, z, wt, r, weights))

        want.append([t.clone() for t in step()])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(step())
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(30):
        for t in (*got[0], *got[1]):
            t.fill_(9)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("far", [40, 100, 126])
@pytest.mark.parametrize("m,n,k", [(9, 140, 200), (300, 9600, 96), (2, 70, 16384)])
def test_scales_at_opposite_ends(m, n, k, far):
    """2^far on one side and 2^-far on the other: the products are those of the codes."""
    from ozaki_blackwell_b200 import mx4
    x, w = _codes(1, m, k), _codes(2, n, k)
    p, q = mx4.quantize(x), mx4.quantize(w)
    for a, b in ((p, q), (q, p)):
        up, down = (mx4.Mx4(t.codes, (t.scales.int() + d).clamp(0, 254).to(torch.uint8), t.length) for t, d in ((a, far), (b, -far)))
        # a block whose scale is cut at the lowest or highest stands for other values: take them as they are
        want = (mx4.dequantize(mx4.Mx4(up.codes, (up.scales.int() - far).to(torch.uint8), k)).double()
                @ mx4.dequantize(mx4.Mx4(down.codes, (down.scales.int() + far).to(torch.uint8), k)).double().t())
        assert torch.equal(mx4.matmul(up, down, torch.float32), want.float())


def test_operands_that_are_views():
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    tokens, top, experts, n, k = 33, 2, 4, 70, 96
    x, w = _codes(1, tokens, k + 40)[:, 5: 5 + k], _codes(2, experts, n, k)
    ids = torch.randint(0, experts, (tokens, top), generator=torch.Generator().manual_seed(1)).cuda()
    wide = mx4.quantize(_codes(3, experts + 2, n + 9, k))
    part = mx4.Mx4(wide.codes[1: 1 + experts, 4: 4 + n], wide.scales[1: 1 + experts, 4: 4 + n], k)
    whole = mx4.Mx4(part.codes.contiguous(), part.scales.contiguous(), k)
    assert torch.equal(ex.matmul(x, part, ids), ex.matmul(x.contiguous(), whole, ids))
    # a matrix's columns and a single row of it; every second matrix of a stack
    got, want = mx4.quantize(w[::2], dim=-2), mx4.quantize(w[::2].contiguous(), dim=-2)
    assert all(torch.equal(a, b) for a, b in zip(ref.unpack(got), ref.unpack(want)))   # the scales' bytes behind the last block are nobody's
    one = x[7: 8]
    assert torch.equal(mx4.matmul(mx4.quantize(one), mx4.quantize(w[0]), torch.float32), (one.double() @ w[0].double().t()).float())
    # one matrix for all planes: read again and again
    many = w[:1].expand(3, n, k)
    q = mx4.quantize(many)
    assert all(torch.equal(q.codes[i], mx4.quantize(w[0]).codes) for i in range(3))


@pytest.mark.parametrize("ids", ["one expert", "all dropped", "the last expert alone has one"])
@pytest.mark.parametrize("tokens,experts,n,k", [(600, 8, 500, 320), (2, 64, 130, 8000)])
def test_routings_far_from_even(ids, tokens, experts, n, k):
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    top = 2
    chosen = torch.full((tokens, top), 3 if ids == "one expert" else -1, device="cuda")
    if ids == "the last expert alone has one":
        chosen[tokens - 1, 1] = experts - 1
    x, dy, w = _codes(1, tokens, k), _codes(2, tokens, n), _codes(3, experts, n, k)
    weights = torch.full((tokens, top), 0.5, device="cuda")
    y, z, r = ex.matmul(x, mx4.quantize(w), chosen, weights, keep=True)
    assert torch.equal(y, ex.matmul(x, mx4.quantize(w), chosen, weights))
    dx, dweights, dw = ex.matmul_grad(dy, x, z, mx4.quantize(w, dim=-2), r, weights)
    for e in range(experts):
        times = (chosen == e).double().sum(1, keepdim=True) * 0.5
        assert torch.equal(dw[e], ((times * dy.double()).t() @ x.double()).float())
    times = [(chosen == e).double().sum(1, keepdim=True) * 0.5 for e in range(experts)]
    assert torch.equal(y, sum(t * (x.double() @ w[e].double().t()) for e, t in enumerate(times)).float())
    assert torch.equal(dx, sum(t * (dy.double() @ w[e].double()) for e, t in enumerate(times)).float())
    assert bool((dweights[chosen < 0] == 0).all()) and mx4.status() is None


def test_rows_past_31_bits():
    """More than 2^31 elements gathered, added up again and rounded by columns."""
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    tokens, top, h = 140000, 8, 2056
    assert tokens * top * h > 2 ** 31
    x = torch.tensor(TABLE, device="cuda", dtype=torch.bfloat16)[torch.randint(0, 8, (tokens, h), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")]
    ids = torch.randint(0, 16, (tokens, top), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    r = ex.sort(ids, 16)
    z = ex.gather(x, r)
    for row in (0, 1, tokens * top // 2, tokens * top - 2, tokens * top - 1):
        assert torch.equal(z[row], x[r.slots[row].item() // top])
    assert torch.equal(ex.combine(z, r), 8 * x)              # eight times a number of three bits
    dz, dweights = ex.combine_grad(x, z, r)
    assert torch.equal(dz, z)
    assert bool((dweights == dweights[:, :1]).all())         # the same products in the same order
    del dz
    q, one = mx4.quantize(z, dim=-2), mx4.quantize(z[-64:].contiguous(), dim=-2)
    assert q.length % 64 == 0 and torch.equal(q.codes[:, -32:], one.codes[:, :32])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,top,experts,h,f", [(5, 2, 7, 96, 80), (300, 3, 5, 256, 200)])
def test_two_projections_with_a_gate_between(dtype, tokens, top, experts, h, f):
    """An experts' layer of two products, call by call: rows behind the last segment are nobody's, whatever lies there.

    The first product's rows come from codes, so they are exact (rounded once to `dtype`); what is rounded of them is compared bit for
    bit; the second product's sums are off by f 2^-23 of their magnitudes and half a unit, the sum over the choices by (top + 1) 2^-24."""
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    x, w1, w2 = _codes(1, tokens, h).to(dtype), _codes(2, experts, 2 * f, h) / 8, _codes(3, experts, h, f)
    g = torch.Generator().manual_seed(4)
    ids, weights = torch.randint(-1, experts, (tokens, top), generator=g).cuda(), torch.rand(tokens, top, generator=g).cuda()
    r = ex.sort(ids, experts, 32)
    rows = r.slots.numel()
    z = mx4.grouped_matmul(mx4.quantize(x, routing=r), mx4.quantize(w1), r.offsets, dtype, out=torch.full((rows, 2 * f), float("nan"), dtype=dtype, device="cuda"))
    a = torch.relu(z[:, :f]) * z[:, f:]
    q = mx4.quantize(a)
    u = mx4.grouped_matmul(q, mx4.quantize(w2), r.offsets, dtype, out=torch.full((rows, h), float("nan"), dtype=dtype, device="cuda"))
    y = ex.combine(u, r, weights)

    end, half = r.offsets[-1].item(), torch.finfo(dtype).eps / 2
    assert bool(torch.isnan(z[end:]).all()) and bool(torch.isnan(u[end:]).all()) and not bool(torch.isnan(z[:end]).any())
    slots, at = r.slots.cpu().long(), r.rows.cpu().long()
    want, bound = torch.zeros(tokens, h, dtype=torch.float64), torch.zeros(tokens, h, dtype=torch.float64)
    xs, w1s, w2s, av = x.cpu().double(), w1.cpu().double(), w2.cpu().double(), ref.values(*ref.quantize(a[:end].float()), f)
    codes, scales = ref.unpack(mx4.Mx4(q.codes[:end], q.scales[:end], f))
    assert all(torch.equal(p, s) for p, s in zip((codes, scales), ref.quantize(a[:end].float())))
    for t in range(tokens):
        for j in range(top):
            e, i, c = ids[t, j].item(), at[t, j].item(), weights[t, j].item()
            if e < 0:
                continue
            assert slots[i] == t * top + j and torch.equal(z[i].cpu(), (w1s[e] @ xs[t]).float().to(dtype))
            part, size = w2s[e] @ av[i], w2s[e].abs() @ av[i].abs()
            want[t] += c * part
            bound[t] += c * (f * 2.0 ** -23 * size + half * part.abs())
            bound[t] += (top + 1) * 2.0 ** -24 * c * (1 + half) * size
    assert bool(((y.cpu().double() - want).abs() <= bound * (1 + half) + half * want.abs() + torch.finfo(dtype).tiny).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,pitch,shift", [(1, 3, 0), (96, 96, 0), (97, 104, 0), (97, 104, 5), (1030, 1032, 0), (1032, 1040, 8), (2050, 2056, 1)])
def test_nothing_is_written_beside_the_results(dtype, h, pitch, shift):
    """Results into views: what lies before, behind and between their rows stays as it was. (Every sum is a multiple of 1/4 below 2^22: the
    order of addition, which alignment changes, does not show.)"""
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    from ozaki_blackwell_b200._lib import lib
    tokens, top, experts = 37, 3, 5
    x = _codes(1, tokens, h).to(dtype)
    r = ex.sort(torch.randint(-1, experts, (tokens, top), generator=torch.Generator().manual_seed(2)).cuda(), experts, 8)
    rows, kind = r.slots.numel(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]

    def view(n):
        flat = torch.full((shift + n * pitch + 64,), 7.0, dtype=dtype, device="cuda")
        return flat, flat[shift: shift + n * pitch].view(n, pitch)[:, :h]

    def untouched(flat, n):
        part = flat[shift: shift + n * pitch].view(n, pitch)
        return bool((flat[:shift] == 7).all()) and bool((flat[shift + n * pitch:] == 7).all()) and bool((part[:, h:] == 7).all())

    flat, out = view(rows)
    z = ex.gather(x, r, out=out)
    assert torch.equal(z, ex.gather(x, r)) and untouched(flat, rows)
    flat, out = view(tokens)
    assert torch.equal(ex.combine(z, r, out=out), ex.combine(z.contiguous(), r)) and untouched(flat, tokens)
    flat, out = view(rows)
    weights, dw = torch.full((tokens, top), 0.5, device="cuda"), torch.empty(tokens, top, device="cuda")
    assert lib.ozb_expert_combine_grad(tokens, top, h, x.data_ptr(), kind, h, z.data_ptr(), z.stride(0), rows, r.rows.data_ptr(), r.slots.data_ptr(), weights.data_ptr(),
                                       out.data_ptr(), pitch, dw.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    dz, dweights = ex.combine_grad(x, z.contiguous(), r, weights)
    assert torch.equal(out, dz) and torch.equal(dw, dweights) and untouched(flat, rows)
    q = mx4.quantize(x)
    flat, out = view(tokens)
    assert torch.equal(mx4.dequantize(q, dtype, out=out), x) and untouched(flat, tokens)

"""The gradients of the experts' layer written over its operands."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("over", ["x", "dy", "z"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_over_an_operand(over, dtype):
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    from ozaki_blackwell_b200._lib import lib
    tokens, top, experts, n = 150, 2, 4, 160
    k = n
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(tokens, n, generator=g).cuda().to(dtype) for _ in range(2))
    w = torch.randn(experts, n, k, generator=g).cuda()
    wq, wt = mx4.quantize(w), mx4.quantize(w, dim=-2)
    ids, weights = torch.randint(-1, experts, (tokens, top), generator=g).cuda(), torch.rand(tokens, top, generator=g).cuda()
    _, z, r = ex.matmul(x, wq, ids, weights, keep=True)
    want = ex.matmul_grad(dy, x, z, wt, r, weights)
    rows, kind = z.shape[0], {torch.float32: 0, torch.bfloat16: 1}[dtype]
    held = {"x": x.clone(), "dy": dy.clone(), "z": z.clone()}
    dx = held[over]
    dweights, dw = torch.empty_like(weights), torch.empty(experts, n, k, dtype=dtype, device="cuda")
    need = lib.ozb_expert_mx4_grad_work(rows, n, k, kind)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    p = lambda t: t.data_ptr()  # noqa: E731
    assert lib.ozb_expert_mx4_grad(tokens, top, experts, n, k, rows, p(held["dy"]), kind, n, p(held["x"]), k, p(held["z"]), n, p(wt.codes), wt.codes.stride(1),
                                   wt.codes.stride(0), p(wt.scales), wt.scales.stride(1), wt.scales.stride(0), p(r.offsets), p(r.rows), p(r.slots), p(weights), p(dx), k,
                                   p(dweights), p(dw), k, n * k, p(work), need, torch.cuda.current_stream().cuda_stream) == 0
    for got, exp in zip((dx[:tokens], dweights, dw), want):
        assert torch.equal(got, exp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,top,experts,n,k", [(40, 2, 3, 97, 65), (900, 2, 2, 3001, 1090), (700, 1, 9, 1037, 2049)])
def test_the_layer_with_pitches(dtype, tokens, top, experts, n, k):
    """Every operand and result of the two calls in rows wider than itself: the same numbers, and nothing written beside them."""
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    from ozaki_blackwell_b200._lib import lib
    kind, pad = {torch.float32: 0, torch.bfloat16: 1}[dtype], {torch.float32: 4, torch.bfloat16: 8}[dtype]
    wide = lambda c: (c + pad - 1) // pad * pad + pad  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(tokens, c, generator=g, device="cuda").to(dtype) for c in (k, n))
    w = torch.randn(experts, n, k, generator=g, device="cuda")
    wq, wt = mx4.quantize(w), mx4.quantize(w, dim=-2)
    ids = torch.randint(-1, experts, (tokens, top), generator=g, device="cuda", dtype=torch.int32)
    weights = torch.rand(tokens, top, generator=g, device="cuda")
    want_y, want_z, r = ex.matmul(x, wq, ids, weights, keep=True)
    want = ex.matmul_grad(dy, x, want_z, wt, r, weights)
    rows, p, st = r.slots.numel(), (lambda t: t.data_ptr()), torch.cuda.current_stream().cuda_stream

    def held(t):
        out = torch.full((*t.shape[:-1], wide(t.shape[-1])), 7.0, dtype=t.dtype, device="cuda")
        out[..., : t.shape[-1]] = t
        return out

    blank = lambda *shape: torch.full((*shape[:-1], wide(shape[-1])), 7.0, dtype=dtype, device="cuda")  # noqa: E731
    xw, dyw, z, y, dx, dw = held(x), held(dy), blank(rows, n), blank(tokens, n), blank(tokens, k), blank(experts, n, k)
    maps = [torch.full_like(t, -7) for t in (r.offsets, r.rows, r.slots)]
    need = lib.ozb_expert_mx4_work(tokens, top, experts, n, k, kind, 64)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert lib.ozb_expert_mx4(tokens, top, experts, n, k, p(xw), kind, wide(k), p(ids), 4, p(weights), p(wq.codes), wq.codes.stride(1), wq.codes.stride(0), p(wq.scales),
                              wq.scales.stride(1), wq.scales.stride(0), 64, *map(p, maps), p(z), wide(n), p(y), wide(n), p(work), need, st) == 0
    assert all(torch.equal(a, b) for a, b in zip(maps, (r.offsets, r.rows, r.slots)))
    end = r.offsets[-1].item()
    assert torch.equal(y[:, :n], want_y) and torch.equal(z[:end, :n], want_z[:end]) and bool((z[end:] == 7).all())
    need = lib.ozb_expert_mx4_grad_work(rows, n, k, kind)
    work, dweights = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty_like(weights)
    assert lib.ozb_expert_mx4_grad(tokens, top, experts, n, k, rows, p(dyw), kind, wide(n), p(xw), wide(k), p(z), wide(n), p(wt.codes), wt.codes.stride(1), wt.codes.stride(0),
                                   p(wt.scales), wt.scales.stride(1), wt.scales.stride(0), *map(p, maps), p(weights), p(dx), wide(k), p(dweights), p(dw), wide(k),
                                   n * wide(k), p(work), need, st) == 0
    assert torch.equal(dx[:, :k], want[0]) and torch.equal(dw[..., :k], want[2])
    # the products' rows lie otherwise, so dots may be added up in another order: n + 1 roundings of FP32 each, of the sum of magnitudes
    rows_of = r.rows.long().clamp(min=0)
    size = (want_z[rows_of].double().abs() * dy[:, None].double().abs()).sum(-1)
    assert bool(((dweights.double() - want[1].double()).abs() <= 2 * (n + 1) * 2.0 ** -24 * size + 1e-30).all())
    for t, c in ((xw, k), (dyw, n), (z, n), (y, n), (dx, k), (dw, k)):
        assert bool((t[..., c:] == 7).all())

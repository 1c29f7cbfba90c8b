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

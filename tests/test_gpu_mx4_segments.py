"""Segments along k that are not whole instructions of 64: the product says so (NaN and the status word) instead of taking a neighbour's
values or losing its own; the last segment may end where the vectors end.

Tolerance of a product over a range of length r: as in test_gpu_mx4.py, r 2^-23 of the sum of magnitudes and half a unit of the type."""
import pytest
import torch

import mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ARG = 10001


def _status():
    from ozaki_blackwell_b200._lib import lib
    return lib.ozb_status()


def _packed(n, k, seed):
    from ozaki_blackwell_b200 import mx4
    return mx4.quantize(torch.randn(n, k, generator=torch.Generator().manual_seed(seed)).cuda())


def _check(y, a, b, dtype):
    exact, size = a @ b.t(), a.abs() @ b.abs().t()
    bound = a.shape[1] * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * exact.abs() + torch.finfo(dtype).smallest_normal
    assert bool(((y.cpu().double() - exact).abs() <= bound).all())


# few tokens; tokens as lanes; pairs of CTAs
@pytest.mark.parametrize("m,n", [(20, 150), (140, 1500), (1100, 3100)])
@pytest.mark.parametrize("dtype", TYPES)
def test_segments_that_are_not_whole(m, n, dtype):
    from ozaki_blackwell_b200 import mx4
    r, offsets = 448, [0, 100, 192, 192, 320, 321, 321, 384, 448]
    a, b = _packed(m, r, 1), _packed(n, r, 2)
    y = mx4.segment_matmul(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), dtype)
    av, bv = ref.of(a), ref.of(b)
    for g, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if lo == hi:
            assert bool((y[g] == 0).all())                 # nothing to take from the wrong place
        elif lo % 64 or hi % 64:
            assert bool(torch.isnan(y[g]).all())
        else:
            _check(y[g], av[:, lo:hi], bv[:, lo:hi], dtype)
    assert _status() == ARG and _status() == 0             # told once


@pytest.mark.parametrize("r", [1, 33, 70, 100, 321, 513])
@pytest.mark.parametrize("m,n", [(5, 40), (140, 3000), (1100, 3100)])
def test_the_last_segment_ends_where_the_vectors_end(m, n, r):
    from ozaki_blackwell_b200 import mx4
    first = r // 128 * 64
    offsets = [0, first, r, r, 2 ** 31 - 1]                # offsets behind the end are cut to it
    a, b = _packed(m, r, 3), _packed(n, r, 4)
    for q in (a, b):
        q.scales[:, (r + 31) // 32:] = 255                 # what lies behind the last block may hold anything
    y = mx4.segment_matmul(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), torch.float32)
    av, bv = ref.of(a), ref.of(b)
    _check(y[0], av[:, :first], bv[:, :first], torch.float32)
    _check(y[1], av[:, first:], bv[:, first:], torch.float32)
    assert bool((y[2:] == 0).all()) and _status() == 0


def test_gradient_of_the_layer_over_a_routing_of_unknown_padding():
    from ozaki_blackwell_b200 import experts as ex
    from ozaki_blackwell_b200 import mx4
    g = torch.Generator().manual_seed(5)
    tokens, top, n, k = 40, 2, 96, 160
    ids = torch.cat([torch.zeros(64), torch.ones(10), torch.full((6,), 2)]).int().reshape(tokens, top).cuda()   # experts with 64, 10 and 6 rows
    x, dy = (torch.randn(tokens, c, generator=g).cuda().bfloat16() for c in (k, n))
    w = torch.randn(3, n, k, generator=g).cuda()
    wq, wt = mx4.quantize(w), mx4.quantize(w, dim=-2)
    weights = torch.rand(tokens, top, generator=g).cuda()
    _, z, r = ex.matmul(x, wq, ids, weights, keep=True)
    dx, dweights, dw = ex.matmul_grad(dy, x, z, wt, r, weights)
    # segments padded to 64, not said so: the same
    for a, b in zip(ex.matmul_grad(dy, x, z, wt, ex.Routing(r.offsets, r.rows, r.slots), weights), (dx, dweights, dw)):
        assert torch.equal(a, b)
    assert _status() == 0
    # not padded, not said so: the experts whose rows begin or end inside 64 have no gradient, the others theirs
    p = ex.sort(ids, 3)
    assert p.offsets.tolist() == [0, 64, 74, 80]
    dense = torch.zeros(80, n, dtype=torch.bfloat16, device="cuda")
    dense[p.rows.reshape(-1).long()] = z[r.rows.reshape(-1).long()]
    got = ex.matmul_grad(dy, x, dense, wt, ex.Routing(p.offsets, p.rows, p.slots), weights)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dweights)
    assert torch.equal(got[2][0], dw[0]) and bool(torch.isnan(got[2][1:]).all())
    assert _status() == ARG
    with pytest.raises(ValueError):
        ex.matmul_grad(dy, x, dense, wt, p, weights)       # known not to be padded

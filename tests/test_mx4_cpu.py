"""Argument checks of the 4-bit and expert entry points: they come before any device work, so they are tested without one."""
import ctypes

import pytest
import torch

from ozaki_blackwell_b200._lib import lib

P = ctypes.c_void_p(4096)          # never dereferenced: every call below is refused
ARG, SIZE = 10001, 10006


def _quantize(X=P, type=0, nvec=4, len=64, ldx=64, by_rows=1, rule=0, rows=None, slots=None, top=0, tokens=0, planes=1, plane_x=0, codes=P, ldq=32, plane_q=0,
              scales=P, lds=16, plane_s=0):
    return lib.ozb_mx4_quantize(X, type, nvec, len, ldx, by_rows, rule, rows, slots, top, tokens, planes, plane_x, codes, ldq, plane_q, scales, lds, plane_s, None)


@pytest.mark.parametrize("bad", [dict(X=None), dict(type=3), dict(type=-1), dict(nvec=0), dict(len=0), dict(len=-1), dict(len=2 ** 31 - 1), dict(ldx=63),
                                 dict(by_rows=0, ldx=3), dict(rule=2), dict(codes=None), dict(codes=ctypes.c_void_p(4104)), dict(ldq=24), dict(ldq=16),
                                 dict(scales=None), dict(scales=ctypes.c_void_p(4104)), dict(lds=8), dict(lds=0), dict(slots=P), dict(rows=P),
                                 dict(rows=P, slots=P, top=1), dict(rows=P, slots=P, tokens=4), dict(rows=P, slots=P, top=1, tokens=4, planes=2), dict(planes=0), dict(planes=2, plane_q=8), dict(planes=2, plane_q=16, plane_s=8),
                                 dict(X=ctypes.c_void_p(4098)), dict(X=ctypes.c_void_p(4097), type=1)])
def test_quantize(bad):
    assert _quantize(**bad) == ARG


def test_dequantize():
    call = lambda **b: lib.ozb_mx4_dequantize(*{**dict(codes=P, ldq=32, scales=P, lds=16, nvec=4, len=64, Y=P, type=1, ldy=64), **b}.values(), None)  # noqa: E731
    for bad in (dict(codes=None), dict(scales=None), dict(Y=None), dict(nvec=0), dict(len=0), dict(len=65), dict(ldy=63), dict(type=4), dict(Y=ctypes.c_void_p(4097))):
        assert call(**bad) == ARG, bad


def test_products():
    dense = dict(M=4, N=4, K=64, X=P, ldx=32, Xs=P, ldxs=16, W=P, ldw=32, Ws=P, ldws=16, Y=P, type=0, ldy=4)
    call = lambda **b: lib.ozb_mx4_gemm(*{**dense, **b}.values(), None)  # noqa: E731
    for bad in (dict(M=0), dict(N=0), dict(K=0), dict(K=65), dict(K=2 ** 31 - 1), dict(X=None), dict(Xs=None), dict(W=None), dict(Ws=None), dict(Y=None),
                dict(ldx=16), dict(ldxs=8), dict(ldy=3), dict(type=3), dict(Y=ctypes.c_void_p(4098)), dict(W=ctypes.c_void_p(4104)), dict(M=-5)):
        assert call(**bad) == ARG, bad
    grouped = dict(groups=2, R=4, N=4, K=64, offsets=P, X=P, ldx=32, Xs=P, ldxs=16, W=P, ldw=32, plane_w=128, Ws=P, ldws=16, plane_ws=32, Y=P, type=0, ldy=4)
    call = lambda **b: lib.ozb_mx4_gemm_grouped(*{**grouped, **b}.values(), None)  # noqa: E731
    for bad in (dict(groups=0), dict(R=0), dict(N=0), dict(K=0), dict(offsets=None), dict(offsets=ctypes.c_void_p(4098)), dict(plane_w=8), dict(plane_ws=8), dict(ldy=3)):
        assert call(**bad) == ARG, bad
    assert call(groups=1025) == SIZE
    segments = dict(groups=2, M=4, N=4, R=64, offsets=P, A=P, lda=32, As=P, ldas=16, B=P, ldb=32, Bs=P, ldbs=16, Y=P, type=0, ldy=4, plane_y=16)
    call = lambda **b: lib.ozb_mx4_gemm_segments(*{**segments, **b}.values(), None)  # noqa: E731
    for bad in (dict(groups=0), dict(M=0), dict(N=0), dict(R=0), dict(R=65), dict(offsets=None), dict(As=None), dict(ldb=8)):
        assert call(**bad) == ARG, bad
    assert call(groups=1025) == SIZE


def test_planes_in_one_another():
    """Several matrices do not overlap: neither results, which would be written twice, nor the codes of weights."""
    assert _quantize(planes=2, plane_x=256, plane_q=112, plane_s=64) == ARG and _quantize(planes=2, plane_x=256, plane_q=128, plane_s=48) == ARG
    stack = lambda planes: lib.ozb_mx4_gemm_grouped(2, 4, 4, 64, P, P, 32, P, 16, P, 32, planes[0], P, 16, planes[1], P, 0, 4, None)  # noqa: E731
    assert stack((0, 64)) == stack((112, 64)) == ARG
    for plane in (0, 15):
        assert lib.ozb_mx4_gemm_segments(2, 4, 4, 64, P, P, 32, P, 16, P, 32, P, 16, P, 0, 4, plane, None) == ARG
    need = lib.ozb_expert_mx4_work(3, 2, 4, 8, 64, 0, 64)
    layer = lambda planes: lib.ozb_expert_mx4(3, 2, 4, 8, 64, P, 0, 64, P, 4, None, P, 32, planes[0], P, 16, planes[1], 64, None, None, None, None, 0, P, 8, P, need, None)  # noqa: E731
    assert layer((0, 128)) == layer((240, 128)) == ARG
    need = lib.ozb_expert_mx4_grad_work(256, 8, 64, 0)
    grad = lambda planes: lib.ozb_expert_mx4_grad(3, 2, 4, 8, 64, 256, P, 0, 8, P, 64, P, 8, P, 16, planes[0], P, 16, planes[1], P, P, P, None, P, 64, P, P, 64, planes[2], P, need, None)  # noqa: E731
    assert grad((0, 1024, 512)) == grad((1008, 1024, 512)) == grad((1024, 1024, 0)) == grad((1024, 1024, 511)) == ARG


def test_sort():
    assert lib.ozb_expert_sort_rows(3, 2, 4, 1) == 6
    assert lib.ozb_expert_sort_rows(3, 2, 4, 64) == (6 + 4 * 63) // 64 * 64      # four segments of at most 64
    assert lib.ozb_expert_sort_rows(1, 2, 100, 8) == 16                           # two slots touch two experts at most
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1025, 1), (1, 1, 1, 0), (1, 1, 1, 257), (2 ** 20, 2 ** 12, 1, 1)):
        assert lib.ozb_expert_sort_rows(*bad) == -ARG, bad
    assert lib.ozb_expert_sort_scratch(128, 8, 64) == 0 and lib.ozb_expert_sort_scratch(1025, 1, 64) == 2 * 64 * 4
    base = dict(T=3, top=2, experts=4, ids=P, id_bytes=4, align=1, R=6, offsets=P, rows=P, slots=P, scratch=None, bytes=0)
    call = lambda **b: lib.ozb_expert_sort(*{**base, **b}.values(), None)  # noqa: E731
    for bad in (dict(T=0), dict(top=0), dict(experts=0), dict(ids=None), dict(id_bytes=2), dict(align=0), dict(align=257), dict(R=5), dict(align=64), dict(offsets=None),
                dict(rows=None), dict(slots=None), dict(T=3000, R=6000), dict(ids=ctypes.c_void_p(4100), id_bytes=8), dict(T=2 ** 20, top=2 ** 12)):
        assert call(**bad) == ARG, bad
    assert call(experts=1025) == SIZE


def test_rows():
    base = dict(T=3, top=2, H=8, X=P, type=0, ldx=8, R=6, rows=P, slots=P, Y=ctypes.c_void_p(8192), ldy=8)
    call = lambda **b: lib.ozb_expert_gather(*{**base, **b}.values(), None)  # noqa: E731
    for bad in (dict(R=0), dict(H=0), dict(X=None), dict(type=5), dict(ldx=7), dict(T=0), dict(rows=None), dict(slots=None), dict(top=0), dict(Y=None), dict(Y=P), dict(ldy=7)):
        assert call(**bad) == ARG, bad
    base = dict(T=3, top=2, H=8, Z=P, type=0, R=6, ldz=8, rows=P, weights=None, Y=ctypes.c_void_p(8192), ldy=8)
    call = lambda **b: lib.ozb_expert_combine(*{**base, **b}.values(), None)  # noqa: E731
    for bad in (dict(T=0), dict(top=0), dict(H=0), dict(Z=None), dict(R=0), dict(ldz=7), dict(rows=None), dict(weights=ctypes.c_void_p(2)), dict(Y=None), dict(Y=P), dict(ldy=7)):
        assert call(**bad) == ARG, bad
    base = dict(T=3, top=2, H=8, dY=P, type=0, lddy=8, Z=P, ldz=8, R=6, rows=P, slots=P, weights=None, dZ=ctypes.c_void_p(8192), lddz=8, dweights=P)
    call = lambda **b: lib.ozb_expert_combine_grad(*{**base, **b}.values(), None)  # noqa: E731
    for bad in (dict(T=0), dict(dY=None), dict(Z=None), dict(dZ=None), dict(dZ=P), dict(rows=None), dict(slots=None), dict(dweights=None), dict(lddy=7), dict(ldz=7), dict(lddz=7), dict(R=0)):
        assert call(**bad) == ARG, bad


def test_the_layer_in_one_call():
    assert lib.ozb_expert_mx4_work(4, 2, 8, 64, 96, 1, 64) > 0 and lib.ozb_expert_mx4_grad_work(512, 64, 96, 1) > 0
    for bad in ((0, 2, 8, 64, 96, 1, 1), (4, 0, 8, 64, 96, 1, 1), (4, 2, 0, 64, 96, 1, 1), (4, 2, 1025, 64, 96, 1, 1), (4, 2, 8, 0, 96, 1, 1), (4, 2, 8, 64, 0, 1, 1),
                (4, 2, 8, 64, 96, 3, 1), (4, 2, 8, 64, 96, 1, 0), (4, 2, 8, 64, 96, 1, 257)):
        assert lib.ozb_expert_mx4_work(*bad) == 0, bad
    for bad in ((0, 64, 96, 1), (512, 0, 96, 1), (512, 64, 0, 1), (512, 64, 96, 5)):
        assert lib.ozb_expert_mx4_grad_work(*bad) == 0, bad
    need = lib.ozb_expert_mx4_work(3, 2, 4, 8, 64, 0, 64)
    base = dict(T=3, top=2, experts=4, N=8, K=64, X=P, type=0, ldx=64, ids=P, id_bytes=4, weights=None, W=P, ldw=32, plane_w=256, Ws=P, ldws=16, plane_ws=128, align=64,
                offsets=None, rows=None, slots=None, Z=None, ldz=0, Y=P, ldy=8, work=P, bytes=need)
    call = lambda **b: lib.ozb_expert_mx4(*{**base, **b}.values(), None)  # noqa: E731
    for bad in (dict(T=0), dict(top=0), dict(experts=0), dict(N=0), dict(K=0), dict(X=None), dict(type=7), dict(ldx=63), dict(ids=None), dict(id_bytes=1), dict(W=None), dict(ldw=16),
                dict(plane_w=8), dict(plane_ws=8), dict(Ws=None), dict(ldws=8), dict(align=0), dict(align=300), dict(offsets=P), dict(rows=P, slots=P), dict(Z=P, ldz=7), dict(Y=None),
                dict(ldy=7), dict(work=None), dict(bytes=need - 1), dict(work=ctypes.c_void_p(4100))):
        assert call(**bad) == ARG, bad
    assert call(experts=1025) == SIZE
    need = lib.ozb_expert_mx4_grad_work(256, 8, 64, 0)
    base = dict(T=3, top=2, experts=4, N=8, K=64, R=256, dY=P, type=0, lddy=8, X=P, ldx=64, Z=P, ldz=8, Wt=P, ldwt=16, plane_wt=1024, Wts=P, ldwts=16, plane_wts=1024, offsets=P, rows=P,
                slots=P, weights=None, dX=P, lddx=64, dweights=P, dW=P, lddw=64, plane_dw=512, work=P, bytes=need)
    call = lambda **b: lib.ozb_expert_mx4_grad(*{**base, **b}.values(), None)  # noqa: E731
    for bad in (dict(T=0), dict(R=0), dict(N=0), dict(K=0), dict(dY=None), dict(X=None), dict(Z=None), dict(Wt=None), dict(Wts=None), dict(offsets=None), dict(rows=None), dict(slots=None),
                dict(dX=None), dict(dweights=None), dict(dW=None), dict(lddy=7), dict(ldx=63), dict(ldz=7), dict(lddx=63), dict(lddw=63), dict(work=None), dict(bytes=need - 1), dict(type=9),
                dict(plane_wt=8)):
        assert call(**bad) == ARG, bad
    assert call(experts=1025) == SIZE


def test_host_tensors_are_refused():
    from ozaki_blackwell_b200 import experts, mx4
    x = torch.zeros(4, 64)
    with pytest.raises(TypeError):
        mx4.quantize(x)
    with pytest.raises(TypeError):
        mx4.dequantize(mx4.Mx4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 16, dtype=torch.uint8), 64))
    with pytest.raises(TypeError):
        mx4.dequantize(mx4.Mx4(torch.zeros(4, 32), torch.zeros(4, 16), 64))
    with pytest.raises(ValueError):
        experts.sort(torch.zeros(4, 2, dtype=torch.int32), 3)
    with pytest.raises(TypeError):
        experts.matmul(x, None, None)


def test_the_wheel_carries_the_modules():
    from ozaki_blackwell_b200 import build_wheel
    assert {"mx4.py", "experts.py"} <= set(build_wheel.PY_FILES)

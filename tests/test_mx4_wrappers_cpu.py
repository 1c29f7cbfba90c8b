"""Refusals of the torch wrappers of the 4-bit and expert operators, on tensors that say they are on a GPU and hold nothing, with a
library that only notes its calls: what is refused never gets that far."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ozaki_blackwell_b200 import experts, mx4

pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer")   # empty tensors have none


@pytest.fixture
def gpu(monkeypatch):
    """gpu(*shape): a tensor on a GPU that is not there; gpu.calls: the library's calls so far, as their arguments."""
    calls = []
    for module in (mx4, experts):
        monkeypatch.setattr(module, "_call", lambda index, entry, *args: calls.append(args))

    def make(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda:0")

    make.calls = calls
    with FakeTensorMode():
        yield make


def _routing(gpu, tokens=4, top=2, rows=8):
    return experts.Routing(gpu(4, dtype=torch.int32), gpu(tokens, top, dtype=torch.int32), gpu(rows, dtype=torch.int32), 1)


def test_combine_needs_a_row_for_each_of_the_routing(gpu):
    r = _routing(gpu)
    for rows in (1, 7):
        with pytest.raises(ValueError, match="8 rows"):
            experts.combine(gpu(rows, 16), r)
    assert not gpu.calls
    for rows in (8, 9):     # more do no harm
        assert experts.combine(gpu(rows, 16), r).shape == (4, 16)
    assert len(gpu.calls) == 2


def test_status_is_the_library_s(monkeypatch):
    """mx4.status: nothing where all went well, the library's error where a wait expired or segments were refused."""
    from ozaki_blackwell_b200 import OzakiError
    codes = iter([0, 10004, 10001])
    monkeypatch.setattr(mx4, "_lib", type("Library", (), {"ozb_status": staticmethod(lambda: next(codes))}))
    assert mx4.status() is None
    for code in (10004, 10001):
        with pytest.raises(OzakiError) as e:
            mx4.status()
        assert e.value.code == code


def _stack(gpu, experts_, n, k):
    u8 = dict(dtype=torch.uint8)
    return mx4.Mx4(gpu(experts_, n, k // 2, **u8), gpu(experts_, n, 16, **u8), k)


def test_a_gradient_that_is_cut_is_said(gpu, recwarn):
    """The calls take no part in autograd: on an operand that requires a gradient they warn, unless autograd is off."""
    x, dy, z = gpu(4, 64), gpu(4, 32), gpu(8, 32)
    ids, weights, r = gpu(4, 2, dtype=torch.int32), gpu(4, 2), _routing(gpu)
    w, wt, padded = _stack(gpu, 3, 32, 64), _stack(gpu, 3, 64, 32), _routing(gpu)._replace(align=64)
    calls = {"quantize": (lambda: mx4.quantize(x), [x]), "gather": (lambda: experts.gather(x, r), [x]), "combine": (lambda: experts.combine(z, r, weights), [z, weights]),
             "combine_grad": (lambda: experts.combine_grad(dy, z, r, weights), [dy, z, weights]),
             "matmul": (lambda: experts.matmul(x, w, ids, weights), [x, weights]),
             "matmul_grad": (lambda: experts.matmul_grad(dy, x, z, wt, padded, weights), [dy, x, z, weights])}
    cut = lambda: [str(v.message) for v in recwarn.list if "autograd" in str(v.message)]  # noqa: E731
    for name, (call, operands) in calls.items():
        call()
        assert not cut(), name                      # nothing requires a gradient
        for t in operands:
            t.requires_grad_()
            with torch.no_grad():
                call()
            assert not cut(), name                  # as inside a torch.autograd.Function
            with pytest.warns(UserWarning, match=f"{name} takes no part in autograd"):
                call()
            t.requires_grad_(False)


def test_sizes_past_32_bits_are_refused(gpu):
    """The library counts in 32 bits; a larger size is refused here, not cut to its low bits."""
    much, u8, i32 = 2 ** 32 + 4, dict(dtype=torch.uint8), dict(dtype=torch.int32)
    x, ids, r = gpu(4, 64), gpu(4, 2, **i32), _routing(gpu)
    codes = lambda n, k: mx4.Mx4(gpu(n, max(16, k // 2), **u8), gpu(n, max(16, k // 32), **u8), k)  # noqa: E731
    for call in (lambda: mx4.quantize(gpu(much, 1)), lambda: mx4.quantize(gpu(much, 1), dim=-2), lambda: mx4.quantize(gpu(1, much)), lambda: mx4.quantize(gpu(much, 1, 1)),
                 lambda: mx4.quantize(x, routing=r._replace(slots=gpu(much, **i32))),
                 lambda: mx4.dequantize(codes(much, 32)), lambda: mx4.dequantize(codes(1, much)),
                 lambda: mx4.matmul(codes(much, 32), codes(4, 32)), lambda: mx4.matmul(codes(4, 32), codes(much, 32)), lambda: mx4.matmul(codes(1, much), codes(1, much)),
                 lambda: experts.sort(ids, much), lambda: experts.sort(ids, 4, much), lambda: experts.sort(gpu(much, 1, **i32), 4), lambda: experts.sort(gpu(1, much, **i32), 4),
                 lambda: experts.gather(x, r._replace(slots=gpu(much, **i32))), lambda: experts.gather(gpu(much, 1), r._replace(rows=gpu(much, 1, **i32))),
                 lambda: experts.combine(gpu(much, 1), r), lambda: experts.combine(gpu(8, much), r),
                 lambda: experts.matmul(gpu(much, 64), _stack(gpu, 3, 32, 64), gpu(much, 1, **i32)), lambda: experts.matmul(x, _stack(gpu, 3, 32, 64), gpu(4, much, **i32))):
        with pytest.raises(ValueError):
            call()
    assert not gpu.calls


def test_the_text_of_a_refusal_names_what_is_refused():
    """One code stands for every refused argument: a misaligned row and an overlapping stack too."""
    from ozaki_blackwell_b200 import OzakiError
    text = str(OzakiError(10001))
    assert all(word in text for word in ("positive", "aligned", "overlap", "segments"))

"""The 4-bit format and the expert operators in 64 bits (or whole numbers), straight from their definitions, for the tests."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def power(e):
    """2^e exactly (torch's pow on a GPU is not)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantize(x, rule="floor"):
    """x [n, k] on the CPU -> (codes [n, kp], scale bytes [n, kp / 32]) with k padded by zeros to kp, a multiple of 32."""
    x = x.detach().cpu().double()
    n, k = x.shape
    kp = -(-k // 32) * 32
    b = torch.zeros(n, kp, dtype=torch.float64)
    b[:, :k] = x
    b = b.reshape(n, kp // 32, 32)
    finite = torch.isfinite(b).all(-1)
    b = torch.where(finite[..., None], b, 0.0)
    amax = b.abs().amax(-1)
    e = torch.full(amax.shape, -127, dtype=torch.long)
    for c in range(-127, 128):   # the definition of either rule as a condition on e, tried from below
        if rule == "floor":
            e = torch.where(amax >= 2.0 ** (c + 2), c, e)          # largest c with 2^(c + 2) <= amax
        else:
            e = torch.where(amax > 6 * 2.0 ** (c - 1), c, e)       # smallest c with amax <= 6 * 2^c
    v = b / power(e)[..., None]
    d = (v.abs()[..., None] - GRID).abs()
    # nearest; of two at the same distance the even code
    code = torch.where(d == d.amin(-1, keepdim=True), torch.tensor([0, 101, 2, 103, 4, 105, 6, 107]), 1000).amin(-1) % 100
    code = torch.where(v.signbit(), code + 8, code)
    scale = torch.where(finite, e + 127, 255)
    return torch.where(finite[..., None], code, 0).reshape(n, kp).to(torch.uint8), scale.to(torch.uint8)


def values(code, scale, k):
    """Codes [..., kp] (one to an element) and scale bytes [..., kp / 32] -> float64 [..., k]."""
    code, scale = code.cpu().long(), scale.cpu().long()
    v = GRID[code % 8] * (1 - 2 * (code // 8))
    s = torch.where(scale == 255, torch.nan, power(scale - 127))
    return (v * s.repeat_interleave(32, -1))[..., :k]


def unpack(q):
    """(codes one to an element, scale bytes) of an Mx4, without what lies behind the last block."""
    blocks = -(-q.length // 32)
    c = q.codes[..., : 16 * blocks].cpu()
    return torch.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], 32 * blocks), q.scales[..., :blocks].cpu()


def of(q):
    """The float64 values of an Mx4."""
    return values(*unpack(q), q.length)


def sort(ids, experts, align):
    """offsets, rows, slots as lists, slot by slot."""
    flat = ids.reshape(-1).tolist()
    per = [[s for s, e in enumerate(flat) if e == x] for x in range(experts)]
    offsets, rows = [0], [-1] * len(flat)
    for p in per:
        for i, s in enumerate(p):
            rows[s] = offsets[-1] + i
        offsets.append(offsets[-1] + -(-len(p) // align) * align)
    return offsets, rows

"""Cases of the low-bit and expert operators: the microscaled 4-bit format (E2M1 values, one power of two per 32 of them), products on
it, and the sorting of tokens by expert that the experts' products need.

`run` computes them in elementary torch operations in 32 bits, or, with `own` set, by this package's calls. `exact` gives the
same from the definitions in 64 bits. The format: a vector is cut into blocks of 32; a block's scale is 2^(s - 127) with a byte s
(255: the block is not a number), a value is a 4-bit code 0 .. 15 (sign, then 0 0.5 1 1.5 2 3 4 6) times that scale. Two codes to
a byte, the earlier one in the low half; rows of codes and of scales start on 16-byte boundaries.
"""
import math

import torch

own = False

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _up(n, to):
    return -(-n // to) * to


def _type(case):
    return getattr(torch, case["type"])


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the activations of a prompt before a 4-bit product: rows of the hidden size, blocks along them
        {"name": "quantise prompt rows", "kind": "quantise", "rows": 2048, "cols": 7168, "axis": 1, "rule": "floor", "type": "bfloat16"},
        # an optimiser's 32-bit weights with blocks down the columns (the transposed operand of a backward product), odd sizes
        {"name": "quantise odd columns", "kind": "quantise", "rows": 4099, "cols": 2051, "axis": 0, "rule": "ceil", "type": "float32"},
        # one new token through a wide projection: reads the weights once
        {"name": "product one token", "kind": "product", "m": 1, "n": 18432, "k": 7168, "type": "bfloat16"},
        # a ragged batch in full output precision, K not a multiple of a block
        {"name": "product ragged", "kind": "product", "m": 333, "n": 1030, "k": 2085, "type": "float32"},
        # a prompt through the repository's wide product shape
        {"name": "product prompt", "kind": "product", "m": 2048, "n": 18432, "k": 7168, "type": "bfloat16"},
        # a decoding step of a small batch: few rows, many experts, the touched experts' weights are the work
        {"name": "experts decode", "kind": "experts", "tokens": 4, "top": 4, "experts": 32, "n": 2048, "k": 4096, "type": "bfloat16"},
        # a prompt through the same layer
        {"name": "experts prompt", "kind": "experts", "tokens": 2048, "top": 4, "experts": 32, "n": 2048, "k": 4096, "type": "bfloat16"},
        # the layer's backward pass: gradients of the tokens, of the routing weights and of the experts' weights
        {"name": "experts backward", "kind": "backward", "tokens": 2048, "top": 4, "experts": 16, "n": 1536, "k": 2048, "type": "bfloat16"},
        # routing of a decoding step: the smallest call, all latency
        {"name": "sort decode", "kind": "sort", "tokens": 16, "top": 4, "experts": 64, "h": 2048, "align": 1, "dropped": 0, "type": "bfloat16"},
        # routing of a large training batch, segments padded to whole blocks, some slots dropped
        {"name": "sort batch", "kind": "sort", "tokens": 16384, "top": 8, "experts": 128, "h": 2048, "align": 64, "dropped": 1, "type": "bfloat16"},
        # bringing a few tokens back, odd width, 32 bits
        {"name": "combine decode", "kind": "combine", "tokens": 7, "top": 2, "experts": 8, "h": 4101, "grad": 0, "type": "float32"},
        # bringing a batch back and the gradient of that
        {"name": "combine with gradient", "kind": "combine", "tokens": 8192, "top": 8, "experts": 64, "h": 2048, "grad": 1, "type": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantise", "product", "product", "experts", "backward", "sort", "combine"])
    some = lambda: rng.choice(["bfloat16", "float16", "float32"])  # noqa: E731
    if kind == "quantise":
        return {"kind": kind, "rows": _log(rng, 1, 4200), "cols": _log(rng, 17, 8000), "axis": rng.randint(0, 1), "rule": rng.choice(["floor", "ceil"]), "type": some()}
    if kind == "product":
        return {"kind": kind, "m": _log(rng, 1, 2048), "n": _log(rng, 16, 16384), "k": _log(rng, 33, 7168), "type": some()}
    if kind == "experts":
        return {"kind": kind, "tokens": _log(rng, 1, 2048), "top": rng.randint(1, 4), "experts": rng.randint(4, 32), "n": _log(rng, 65, 2048), "k": _log(rng, 96, 4096), "type": some()}
    if kind == "backward":
        return {"kind": kind, "tokens": _log(rng, 5, 2048), "top": rng.randint(1, 4), "experts": rng.randint(4, 16), "n": _log(rng, 65, 1536), "k": _log(rng, 96, 2048), "type": rng.choice(["bfloat16", "float32"])}
    if kind == "sort":
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "top": rng.randint(1, 8), "experts": _log(rng, 8, 128), "h": _log(rng, 33, 2048), "align": rng.choice([1, 32, 64]), "dropped": rng.randint(0, 1), "type": some()}
    return {"kind": kind, "tokens": _log(rng, 1, 8192), "top": rng.randint(1, 8), "experts": _log(rng, 8, 64), "h": _log(rng, 33, 2048), "grad": rng.randint(0, 1), "type": some()}


def _power(e):
    """2^e in 32 bits, exactly, for whole e from -127 on (ldexp and pow on a GPU may be a last place off)."""
    e = e.int()
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).view(torch.float32)


# ---- what a program has in hand ----------------------------------------------------------------------------------------

def _pack(x):
    """Codes and scales of the rows of x (last axis), as a checkpoint holds them."""
    k = x.shape[-1]
    kp = _up(k, 32)
    b = torch.zeros(*x.shape[:-1], kp, device=x.device)
    b[..., :k] = x
    b = b.reshape(*x.shape[:-1], kp // 32, 32)
    s = (torch.frexp(b.abs().amax(-1))[1] - 1 - 2).clamp(-127, 127)
    v = b * _power(-s[..., None])
    a = v.abs()
    c = (a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()
    c = (c + 8 * torch.signbit(v).byte()).reshape(*x.shape[:-1], kp)
    codes = torch.zeros(*x.shape[:-1], _up(kp // 2, 16), dtype=torch.uint8, device=x.device)
    codes[..., : kp // 2] = c[..., 0::2] | (c[..., 1::2] << 4)
    scales = torch.zeros(*x.shape[:-1], _up(kp // 32, 16), dtype=torch.uint8, device=x.device)
    scales[..., : kp // 32] = (s + 127).to(torch.uint8)
    return codes, scales


def _capacity(slots, experts, align):
    return (slots + min(experts, slots) * (align - 1)) // align * align


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    kind, s = case["kind"], dict(case)
    s["dtype"] = _type(case)
    if kind == "quantise":
        # rows of different magnitude and a few outliers, as activations and weights have them
        x = normal(case["rows"], case["cols"]) * torch.exp2((3 * normal(case["rows"], 1)).clamp(-8, 8))
        x *= 1 + 30 * (torch.rand(1, case["cols"], device="cuda", generator=g) < 0.01)
        s["x"] = x.to(_type(case))
    elif kind == "product":
        s["x"] = _pack(normal(case["m"], case["k"]))
        s["w"] = _pack(normal(case["n"], case["k"]) * case["k"] ** -0.5)
    else:
        t, top, e = case["tokens"], case["top"], case["experts"]
        # scores with favourites among the experts, each token's `top` best of them
        score = normal(t, e) + 0.5 * normal(1, e)
        k = min(top, e)
        best = torch.topk(score, k, dim=-1)
        ids = torch.cat([best.indices] + [best.indices[:, :1]] * (top - k), 1).to(torch.int32)
        if case.get("dropped"):
            ids = torch.where(torch.rand(t, top, device="cuda", generator=g) < 0.05, -1, ids)
        s["ids"] = ids.contiguous()
        s["weights"] = torch.softmax(torch.cat([best.values] + [best.values[:, :1]] * (top - k), 1), -1).contiguous()
        s["longest"] = int(torch.bincount(ids.clamp(min=0).reshape(-1), minlength=e).max())
        if kind in ("experts", "backward"):
            s["x"] = normal(t, case["k"]).to(_type(case))
            w = normal(e, case["n"], case["k"]) * case["k"] ** -0.5
            if kind == "experts":
                s["w"] = _pack(w)
            else:
                s["wt"] = _pack(w.transpose(1, 2).contiguous())
                rows = _capacity(t * top, e, 64)
                s["routing"] = _sorted(ids, e, 64, rows)
                s["dy"] = normal(t, case["n"]).to(_type(case))
                s["z"] = normal(rows, case["n"]).to(_type(case))  # the forward pass's rows
        elif kind == "sort":
            s["x"] = normal(t, case["h"]).to(_type(case))
        else:
            rows = _capacity(t * top, e, 1)
            s["routing"] = _sorted(ids, e, 1, rows)
            s["z"] = normal(rows, case["h"]).to(_type(case))
            s["dy"] = normal(t, case["h"]).to(_type(case))
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _values(packed, k):
    """The numbers that codes and scales stand for, in 32 bits."""
    codes, scales = packed
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)[..., :k].int()]
    e = scales[..., : _up(k, 32) // 32].repeat_interleave(32, -1)[..., :k]
    return torch.where(e == 255, torch.nan, v * _power(e.int() - 127))


def _rounded(x, rule="floor"):
    """x (last axis in blocks of 32) rounded to the format, in 32 bits."""
    k = x.shape[-1]
    b = torch.nn.functional.pad(x.float(), (0, _up(k, 32) - k)).unflatten(-1, (-1, 32))
    mantissa, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # amax = mantissa 2^e, 0.5 <= mantissa < 1
    e = e - 3 + ((mantissa > 0.75) if rule == "ceil" else 0)   # "ceil": the largest value does not pass 6
    e = e.clamp(min=-127)
    v = b * _power(-e)
    a = v.abs()
    up = lambda p: (a >= p).float()  # noqa: E731
    past = lambda p: (a > p).float()  # noqa: E731
    q = 0.5 * (past(0.25) + up(0.75) + past(1.25) + up(1.75)) + past(2.5) + up(3.5) + 2 * past(5.0)
    return (torch.copysign(q, v) * _power(e)).flatten(-2)[..., :k]


def _sorted(ids, experts, align, rows):
    """Slots in the order of their experts (stable), each expert's segment padded to a multiple of `align`."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    counts = torch.zeros(experts + 1, dtype=torch.long, device=ids.device).scatter_add(0, key, torch.ones_like(key))
    offsets = torch.nn.functional.pad(((counts[:experts] + align - 1) // align * align).cumsum(0), (1, 0))
    key_sorted, order = torch.sort(key, stable=True)
    place = offsets[key_sorted] + torch.arange(len(flat), device=ids.device) - (counts.cumsum(0) - counts)[key_sorted]
    kept = key_sorted < experts
    row_of = torch.full_like(flat, -1).scatter(0, order, torch.where(kept, place, -1))
    slot_of = torch.full((rows + 1,), -1, dtype=torch.long, device=ids.device).scatter(0, torch.where(kept, place, rows), order)[:rows]
    return {"offsets": offsets.int(), "rows": row_of.int().reshape(ids.shape), "slots": slot_of.int()}


def _gathered(x, slots, top):
    return torch.where(slots[:, None] >= 0, x.float()[slots.clamp(min=0).long() // top], 0.0)


def _windows(offsets, longest, rows):
    """For each expert the rows of its segment, and which of them are there."""
    at = offsets[:-1, None].long() + torch.arange(longest, device=offsets.device)
    return at.clamp(max=rows - 1), at < offsets[1:, None]


def _grouped(x, w, offsets, longest):
    """Row r of expert e's segment times w[e]^T."""
    at, there = _windows(offsets, longest, len(x))
    z = torch.bmm(torch.where(there[..., None], x[at], 0.0), w.transpose(1, 2))
    out = torch.zeros(len(x) + 1, w.shape[1], device=x.device)
    out[torch.where(there, at, len(x))] = z
    return out[:-1]


def _combined(z, rows, weights):
    z = torch.where(rows[..., None] >= 0, z.float()[rows.clamp(min=0).long()], 0.0)
    return (z * weights[..., None]).sum(1) if weights is not None else z.sum(1)


def _combined_grad(dy, z, r, weights):
    dy, slots, rows = dy.float(), r["slots"].long(), r["rows"]
    w = weights.reshape(-1)[slots.clamp(min=0)]
    dz = torch.where(slots[:, None] >= 0, w[:, None] * dy[slots.clamp(min=0) // rows.shape[1]], 0.0)
    dots = (z.float() * dy[slots.clamp(min=0) // rows.shape[1]]).sum(-1)
    return dz, torch.where(rows >= 0, dots[rows.clamp(min=0).long()], 0.0)


def _run_plain(s):
    kind, dtype = s["kind"], s["dtype"]
    if kind == "quantise":
        return {"values": _rounded(s["x"] if s["axis"] == 1 else s["x"].t(), s["rule"]).to(dtype)}
    if kind == "product":
        return {"y": (_values(s["x"], s["k"]) @ _values(s["w"], s["k"]).t()).to(dtype)}
    if kind == "sort":
        r = _sorted(s["ids"], s["experts"], s["align"], _capacity(s["ids"].numel(), s["experts"], s["align"]))
        return {**r, "x": _gathered(s["x"], r["slots"], s["top"]).to(dtype)}
    if kind == "combine":
        r = s["routing"]
        out = {"y": _combined(s["z"], r["rows"], s["weights"]).to(dtype)}
        if s["grad"]:
            dz, dw = _combined_grad(s["dy"], s["z"], r, s["weights"])
            out.update(dz=dz.to(dtype), dweights=dw)
        return out
    if kind == "experts":
        r = _sorted(s["ids"], s["experts"], 1, s["ids"].numel())
        x = _rounded(_gathered(s["x"], r["slots"], s["top"]))
        z = _grouped(x, _values(s["w"], s["k"]), r["offsets"], s["longest"]).to(dtype)
        return {"y": _combined(z, r["rows"], s["weights"]).to(dtype)}
    r, longest = s["routing"], _up(s["longest"], 64)
    dz, dweights = _combined_grad(s["dy"], s["z"], r, s["weights"])
    dz = dz.to(dtype)
    dx = _grouped(_rounded(dz), _values(s["wt"], s["n"]), r["offsets"], longest).to(dtype)
    at, there = _windows(r["offsets"], longest, len(dz))
    left = _rounded(dz.t()).t()[at] * there[..., None]
    right = _rounded(_gathered(s["x"], r["slots"], s["top"]).t()).t()[at] * there[..., None]
    return {"dx": _combined(dx, r["rows"], None).to(dtype), "dweights": dweights, "dw": torch.bmm(left.transpose(1, 2), right).to(dtype)}


# ---- this package's calls ------------------------------------------------------------------------------------------------

def _run_own(s):
    from ozaki_blackwell_b200 import experts, mx4
    kind, dtype = s["kind"], s["dtype"]
    if kind == "quantise":
        return {"values": mx4.dequantize(mx4.quantize(s["x"], dim=s["axis"] - 2, rule=s["rule"]), dtype)}
    if kind == "product":
        return {"y": mx4.matmul(mx4.Mx4(*s["x"], s["k"]), mx4.Mx4(*s["w"], s["k"]), dtype)}
    if kind == "sort":
        r = experts.sort(s["ids"], s["experts"], s["align"])
        return {"offsets": r.offsets, "rows": r.rows, "slots": r.slots, "x": experts.gather(s["x"], r)}
    if kind == "experts":
        return {"y": experts.matmul(s["x"], mx4.Mx4(*s["w"], s["k"]), s["ids"], s["weights"])}
    r = experts.Routing(**s["routing"])
    if kind == "combine":
        out = {"y": experts.combine(s["z"], r, s["weights"])}
        if s["grad"]:
            out["dz"], out["dweights"] = experts.combine_grad(s["dy"], s["z"], r, s["weights"])
        return out
    dx, dweights, dw = experts.matmul_grad(s["dy"], s["x"], s["z"], mx4.Mx4(*s["wt"], s["n"]), r, s["weights"])
    return {"dx": dx, "dweights": dweights, "dw": dw}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what each pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    kind, size = case["kind"], torch.finfo(_type(case)).bits // 8
    packed = 17 / 32  # bytes of a value: half a byte, and a byte for 32
    if kind == "quantise":
        n = case["rows"] * case["cols"]
        return {"bytes": int(n * (2 * size + packed)), "flops": 4 * n}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": int((m + n) * k * packed + m * n * size), "flops": 2 * m * n * k}
    t, top, e = case["tokens"], case["top"], case["experts"]
    slots = t * top
    if kind == "sort":
        return {"bytes": int(12 * slots + 4 * e + (t + slots) * case["h"] * size), "flops": slots}
    if kind == "combine":
        once = slots * case["h"] * size + t * case["h"] * size + 8 * slots
        return {"bytes": int(once * (1 + 2 * case["grad"])), "flops": (2 + 4 * case["grad"]) * slots * case["h"]}
    touched = e * (1 - (1 - min(top, e) / e) ** t)  # experts that some token goes to
    weights, product = case["n"] * case["k"], 2 * slots * case["n"] * case["k"]
    if kind == "experts":
        return {"bytes": int(touched * weights * packed + t * (case["n"] + case["k"]) * size), "flops": product}
    rows = (2 * t + slots) * case["n"] * size + 2 * t * case["k"] * size
    return {"bytes": int(touched * weights * packed + e * weights * size + rows), "flops": 2 * product}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_values(packed, k):
    codes, scales = packed
    low, high = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    c[..., 0::2], c[..., 1::2] = low, high
    c = c[..., :k]
    sign, m = 1 - 2 * (c >= 8).double(), c % 8
    # exponent field m // 2 and one mantissa bit: below 2 the values are m / 2, then (1 + bit / 2) 2^(field - 1)
    v = torch.where(m < 2, m / 2, (1 + (m % 2) / 2) * _exact_power(torch.div(m, 2, rounding_mode="floor") - 1))
    s = scales.double()[..., : _up(k, 32) // 32]
    return sign * v * _exact_power(s - 127).repeat_interleave(32, -1)[..., :k]


def _exact_rounded(x, rule="floor"):
    """Nearest value of the format, ties to the even code, by distance."""
    x = x.double()
    k = x.shape[-1]
    out = torch.empty_like(x)
    if not x.numel():
        return out
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    for a in range(0, k, 4096):  # whole blocks at a time
        b = x[..., a : min(k, a + 4096)]
        n = b.shape[-1]
        b = torch.cat([b, torch.zeros(*b.shape[:-1], _up(n, 32) - n, dtype=torch.float64, device=x.device)], -1)
        b = b.reshape(*b.shape[:-1], -1, 32)
        most = b.abs().max(-1).values
        if rule == "floor":
            e = torch.floor(torch.log2(most.clamp(min=2.0 ** -200))) - 2
        else:
            e = torch.ceil(torch.log2((most / 6).clamp(min=2.0 ** -200)))
        e = e.clamp(-127, 127)
        # logarithms next to a border: put right by comparing
        if rule == "floor":
            e = torch.where((most >= _exact_power(e + 3)) & (e < 127), e + 1, e)
            e = torch.where((most < _exact_power(e + 2)) & (e > -127), e - 1, e)
        else:
            e = torch.where((most > 6 * _exact_power(e)) & (e < 127), e + 1, e)
            e = torch.where((most <= 3 * _exact_power(e)) & (e > -127), e - 1, e)
        scale = _exact_power(e)[..., None]
        v = b / scale
        # the even codes of a pair at equal distance come first in this order
        order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)
        best, at = (v.abs() - grid[order[0]]).abs(), torch.zeros_like(v)
        for i in order[1:].tolist():
            d = (v.abs() - grid[i]).abs()
            at = torch.where(d < best, grid[i], at)
            best = torch.minimum(d, best)
        out[..., a : a + n] = (torch.sign(v) * at * scale).reshape(*v.shape[:-2], -1)[..., :n]
    return out


def _exact_segments(ids, experts, align):
    """Each expert's slots in their order, and where its segment begins."""
    flat, segments, begin = ids.reshape(-1).cpu(), [], 0
    for e in range(experts):
        at = torch.nonzero(flat == e).reshape(-1)
        segments.append((begin, at.to(ids.device)))
        begin += _up(len(at), align)
    return segments, begin


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantise":
        return {"values": _exact_rounded(s["x"] if case["axis"] == 1 else s["x"].t().contiguous(), case["rule"])}
    if kind == "product":
        return {"y": _exact_values(s["x"], case["k"]) @ _exact_values(s["w"], case["k"]).t()}
    t, top, e, ids = case["tokens"], case["top"], case["experts"], s["ids"]
    weights = s["weights"].double().reshape(-1)
    if kind == "sort":
        segments, end = _exact_segments(ids, e, case["align"])
        rows = _capacity(t * top, e, case["align"])
        slots = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
        row_of = torch.full((t * top,), -1, dtype=torch.int32, device="cuda")
        for begin, at in segments:
            slots[begin : begin + len(at)] = at.int()
            row_of[at] = torch.arange(begin, begin + len(at), dtype=torch.int32, device="cuda")
        offsets = torch.tensor([b for b, _ in segments] + [end], dtype=torch.int32, device="cuda")
        x = torch.zeros(rows, case["h"], dtype=torch.float64, device="cuda")
        x[slots >= 0] = s["x"].double()[torch.div(slots[slots >= 0], top, rounding_mode="floor").long()]
        return {"offsets": offsets, "rows": row_of.reshape(t, top), "slots": slots, "x": x}
    if kind == "combine":
        segments, _ = _exact_segments(ids, e, 1)
        y = torch.zeros(t, case["h"], dtype=torch.float64, device="cuda")
        dz, dw = torch.zeros(t * top, case["h"], dtype=torch.float64, device="cuda"), torch.zeros(t * top, dtype=torch.float64, device="cuda")
        for begin, at in segments:
            z, of = s["z"][begin : begin + len(at)].double(), torch.div(at, top, rounding_mode="floor")
            y.index_add_(0, of, weights[at, None] * z)
            dz[begin : begin + len(at)] = weights[at, None] * s["dy"].double()[of]
            dw[at] = (s["dy"].double()[of] * z).sum(1)
        return {"y": y, "dz": dz, "dweights": dw.reshape(t, top)} if case["grad"] else {"y": y}
    if kind == "experts":
        y = torch.zeros(t, case["n"], dtype=torch.float64, device="cuda")
        x = _exact_rounded(s["x"])
        for i, (_, at) in enumerate(_exact_segments(ids, e, 1)[0]):
            of = torch.div(at, top, rounding_mode="floor")
            z = x[of] @ _exact_values((s["w"][0][i], s["w"][1][i]), case["k"]).t()
            y.index_add_(0, of, weights[at, None] * z.to(_type(case)).double())  # the rows between the two calls have the type of x
        return {"y": y}
    dx = torch.zeros(t, case["k"], dtype=torch.float64, device="cuda")
    dweights = torch.zeros(t * top, dtype=torch.float64, device="cuda")
    dw = torch.zeros(e, case["n"], case["k"], dtype=torch.float64, device="cuda")
    for i, (begin, at) in enumerate(_exact_segments(ids, e, 64)[0]):
        of = torch.div(at, top, rounding_mode="floor")
        dy = s["dy"].double()[of]
        dweights[at] = (dy * s["z"][begin : begin + len(at)].double()).sum(1)
        dz = (weights[at, None] * dy).to(_type(case)).double()
        part = _exact_rounded(dz) @ _exact_values((s["wt"][0][i], s["wt"][1][i]), case["n"]).t()
        dx.index_add_(0, of, part.to(_type(case)).double())
        if len(at):
            dw[i] = _exact_rounded(dz.t().contiguous()) @ _exact_rounded(s["x"].double()[of].t().contiguous()).t()
    return {"dx": dx, "dweights": dweights.reshape(t, top), "dw": dw}

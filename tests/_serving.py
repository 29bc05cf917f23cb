"""64-bit references of the serving calls and the tolerances that follow from their roundings (numpy, or torch on any device)."""
import math

import torch

TYPES = {"int8": torch.int8, "bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
AMAX = (4.5, 4.75, 4.25)


def codes(shape, seed, device="cuda"):
    """Every int8 code that the quantiser gives, evenly."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return torch.randint(-127, 128, shape, dtype=torch.int8, device=device, generator=g)


def starts(lengths, device="cuda"):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def attention64(q, k, v, amax, causal):
    """One sequence: q [n, H, D], k, v [m, Hkv, D] int8 -> (o, scales): float64 [n, H, D], the output in real units, and two of that shape for
    tolerance(): sum_j p_j |v_j| with the p of a row adding up to 1, and sum_j |v_j| / sum_j p_j over the keys that the row sees, the largest p being 1."""
    n, H, D = q.shape
    m, Hkv = k.shape[0], k.shape[1]
    if n == 0 or m == 0:
        none = torch.zeros((n, H, D), dtype=torch.float64, device=q.device)
        return none, (none, none)
    scale = float(torch.tensor(amax[0])) * float(torch.tensor(amax[1])) / 127.0 ** 2 / math.sqrt(D)
    kk, vv = (x.double().repeat_interleave(H // Hkv, 1).transpose(0, 1) for x in (k, v))
    s = q.double().transpose(0, 1) @ kk.transpose(1, 2) * scale
    seen = torch.ones((n, m), dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(m - n)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / torch.where(l > 0, l, 1.0), 0.0)
    real = float(torch.tensor(amax[2])) / 127.0
    each = torch.where(l > 0, (seen.double() @ vv.abs()) / torch.where(l > 0, l, 1.0), 0.0)
    return (p @ vv).transpose(0, 1) * real, ((p @ vv.abs()).transpose(0, 1) * real, each.transpose(0, 1) * real)


def tolerance(o, scales, keys, o_type, amax, o_amax, rows, own=None):
    """Elementwise bound of |result - o|, o in real units.  `rows`: query rows per key head that the call allows (max_seq_q * heads of a group); `own`: those that the
    sequence has.  In a call that allows more than eight, a sequence with up to eight may be computed with either P (below), so the larger bound holds.
      P        fp16: half a step, 2^-11 relative, of every p; below 2^-14 half a step is 2^-25 of the row's largest p, which is 1 or more.  Up to eight rows: whole
               numbers of 16 bits, half a step, 2^-17 of the largest p, for every key.
      exp2     2^-22; its argument (|a| <= 24 where p matters) is off by half a step of the factor and of its rounding (2^-24 relative each) and, up to
               eight rows, of a difference: 24 * 3 * 2^-24 * ln 2 < 2^-18.3; with the rest 2^-18 together.
      sums     keys additions in fp32, half a step (2^-24) each, of sums at most sum p |v|.
      output   half a step of its type relative to the result (int8: half a code)."""
    out = torch.full_like(o, 0.5 * o_amax / 127.0) if o_type == "int8" else o.abs() * (torch.finfo(TYPES[o_type]).eps / 2)
    tiny = 0.0 if o_type != "fp16" else 2.0 ** -25            # half a step below fp16's smallest normal number
    spread, each = scales
    whole, half = each * 2.0 ** -17, spread * 2.0 ** -11 + each * 2.0 ** -25
    of_p = whole if rows <= 8 else half if own is None or own > 8 else torch.maximum(whole, half)
    return out * 1.001 + of_p + spread * (2.0 ** -18 + keys * 2.0 ** -24) + tiny + 1e-12


def real_units(o, o_type, o_amax):
    return o.double() * (o_amax / 127.0) if o_type == "int8" else o.double()


def check(got, want, scales, keys, o_type, amax, o_amax, rows, what="", own=None):
    want_c = want.clamp(-o_amax, o_amax) if o_type == "int8" else want
    err = (real_units(got, o_type, o_amax) - want_c).abs()
    tol = tolerance(want_c, scales, keys, o_type, amax, o_amax, rows, own)
    over = err > tol
    assert not bool(over.any()), f"{what}: {int(over.sum())} of {over.numel()} off, worst {float((err / tol).max()):.3g} times the tolerance"


def rotate64(x, positions, inv_freq, magnitude, interleaved):
    """x float64 [T, heads, D]."""
    half = inv_freq.numel()
    if half == 0:
        return x
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def quantise64(y, amax):
    """clamp(floor(y * (127 / amax) + 1/2), -127, 127); not a number gives 0."""
    z = torch.floor(y * (127.0 / float(torch.tensor(amax, dtype=torch.float32))) + 0.5).clamp(-127, 127)
    return torch.nan_to_num(z, nan=0.0).to(torch.int8)


def assert_same(got, want):
    assert got.shape == want.shape
    off = int((got != want).sum())
    assert off == 0, f"{off} of {want.numel()} codes differ"

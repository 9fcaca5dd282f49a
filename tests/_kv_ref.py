"""Float64 restatements, for the tests, of the block cache's values, attention over a cache, the accumulated
weights, eviction and rotary positions with several axes, and the error that the kernels' formats allow."""

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}


def block_scale(x, kind):
    """The smallest power of two, 2^-126 at least, that brings max |x| within the type."""
    most = x.abs().max().item()
    if not math.isfinite(most):
        return math.nan
    e = -126
    if most > 0:
        m, xp = math.frexp(most / TOP[kind])  # (exact: TOP has 7 or 3 bits; the quotient's comparison below decides)
        e = max(-126, xp - 1)
        while most > TOP[kind] * 2.0 ** e:
            e += 1
        while e > -126 and most <= TOP[kind] * 2.0 ** (e - 1):
            e -= 1
    return 2.0 ** e


def round_codes(y, kind):
    """y (float64, within the type's range) rounded to the type's values, ties to even."""
    if kind == torch.int8:
        return torch.round(y)
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(y), e - 4)
    return torch.round(y / step) * step


def held(x, kind, block):
    """The values, in float64, of a block cache holding the tokens x (..., T, D)."""
    x = x.double().clone()
    flat = x.reshape(-1, *x.shape[-2:])
    for s in flat:
        for j in range(x.shape[-2] // block):
            b = s[j * block:(j + 1) * block]
            unit = block_scale(b, kind)
            b.copy_(torch.full_like(b, math.nan) if math.isnan(unit) else round_codes(b / unit, kind) * unit)
    return flat.reshape(x.shape)


def visible(n, L, causal):
    """Which of the n tokens held each of the last L rows sees."""
    t = torch.arange(n)[None]
    return t <= torch.arange(n - L, n)[:, None] if causal else torch.ones((L, n), dtype=torch.bool)


def attend(q, k, v, causal=True, scale=None):
    """Attention of the last L tokens' rows q (H, L, D) over one sequence's k, v (Hkv, n, D): the output, the
    weights' sums (Hkv, n), and how far a kernel may be from each (before the output's own rounding) apart from
    the rounding of p: see `bounds`."""
    H, L, D = q.shape
    Hkv, n = k.shape[0], k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    see = visible(n, L, causal)
    out = torch.zeros((H, L, D), dtype=torch.float64)
    mass = torch.zeros((H, L, D), dtype=torch.float64)  # sum p |v|
    slack = torch.zeros((H, L), dtype=torch.float64)    # how far ln p may be off
    sums, sums_slack = torch.zeros((Hkv, n), dtype=torch.float64), torch.zeros((Hkv, n), dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for h in range(H):
        g = h // (H // Hkv)
        s = torch.where(see, q[h] @ k[g].T * scale, torch.tensor(-math.inf, dtype=torch.float64))
        p = torch.softmax(s, 1)
        kk, vv = torch.where(torch.isfinite(k[g]), k[g], 0.0), torch.where(torch.isfinite(v[g]), v[g], 0.0)
        out[h], mass[h] = p @ vv, p @ vv.abs()
        # float32 products and sums of D terms, a query row's operand off by 2^-25 of its largest element
        reach = (q[h].abs() @ kk.abs().T + q[h].abs().amax(1, keepdim=True) * kk.abs().sum(1)[None]) * scale
        reach = torch.where(see, reach, 0.0).amax(1)
        top = torch.where(see, s.abs(), 0.0).amax(1)
        slack[h] = ((D + 4) * reach + 8 * top + 8 * math.log(n + 1) + 8) * 2.0 ** -24
        sums[g] += p.sum(0)
        sums_slack[g] += (p * (2 * slack[h][:, None])).sum(0)
    return out, mass, slack, sums, sums_slack


def bounds(out, mass, slack, n, dtype):
    """The largest error of the fused kernel: p' is rounded to float16 (2^-12 of a term) for half-precision
    results and kept to 2^-22 for float32 ones, what is below 2^-14 of the largest term to 2^-25 of it; then
    float32 sums over n keys, and the result's rounding."""
    p = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    return mass * (p + 2 * slack[..., None] + (2 * n + 16) * 2.0 ** -24) + HALF_STEP[dtype] * out.abs() + 2.0 ** -25 * (dtype == torch.float16)


def chosen(w, keep, recent):
    """The kept indices of one head with the weights w (n,)."""
    n = len(w)
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)
    key = [math.inf if math.isnan(x) else x for x in w.tolist()]
    nan = [math.isnan(x) for x in w.tolist()]
    first = sorted(range(n - recent), key=lambda i: (not nan[i], -key[i], i))[:keep - recent]
    return sorted(first) + list(range(n - recent, n))


def pair_axes(sections, interleaved):
    n = len(sections)
    if interleaved:
        return [i % n if i // n < sections[i % n] else 0 for i in range(sum(sections))]
    return [a for a in range(n) for _ in range(sections[a])]


def rope_axes(x, pos, sections, n_dims=None, mode=2, interleaved=False, freq_base=10000.0, freq_scale=1.0, inverse=False):
    """x (B, H, S, D), pos (axes, B, S): the rotation in float64 and its error bound but for the rounding of the
    result: float32 turns (2 pi 2^-26), sine and cosine (two steps of 2^-24) and two roundings of the rotation."""
    nd = x.shape[-1] if n_dims is None else n_dims
    half = nd // 2
    x = x.double()
    out, slack = x.clone(), torch.zeros_like(x)
    for i, a in enumerate(pair_axes(sections, interleaved)):
        angle = pos[a].double() * (freq_scale * freq_base ** (-2.0 * i / nd))
        c, s = torch.cos(angle)[:, None], torch.sin(-angle if inverse else angle)[:, None]
        lo, hi = (i, i + half) if mode == 2 else (2 * i, 2 * i + 1)
        out[..., lo] = x[..., lo] * c - x[..., hi] * s
        out[..., hi] = x[..., lo] * s + x[..., hi] * c
        size = (x[..., lo].abs() + x[..., hi].abs()) * (2 * math.pi * 2.0 ** -26 + 4 * 2.0 ** -24 + angle.abs()[:, None] * 2.0 ** -50)
        slack[..., lo], slack[..., hi] = size, size
    return out, slack

"""Plain 64-bit forms of the serving operators, one sequence and head at a
time, and the error bounds that the tests hold the kernels to."""
import math

import torch

# largest relative error of one rounding to the type
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def rotate(x, positions, freqs, layout="half", magnitude=1.0, inverse=False):
    """x [tokens, heads, dim], freqs radians a position (python floats)."""
    y = x.double().clone()
    n = len(freqs)
    f = torch.tensor(freqs, dtype=torch.float64, device=x.device)
    angle = positions.double()[:, None] * f * (-1.0 if inverse else 1.0)
    c, s = angle.cos()[:, None] * magnitude, angle.sin()[:, None] * magnitude
    first = slice(0, n) if layout == "half" else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if layout == "half" else slice(1, 2 * n, 2)
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def rows_of(pages, scale, slots):
    """Values of the cache rows `slots`, [n, kv heads, dim], fp64."""
    p, r = slots // pages.shape[2], slots % pages.shape[2]
    if scale is None:
        return pages[p, :, r].double()
    raw = pages.view(torch.uint8)[p, :, r].view(pages.dtype)
    return raw.double() * scale[p, :, r].double()[..., None]


def attend(q, k, v, first, window, scale):
    """q [n, heads, dim] at positions first .. first + n - 1 over k, v [m, kv heads, dim].
    Returns (out, sum of p |v|, lse, keys seen), all fp64; a masked key has no part in anything."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device=q.device)
    mag, lse = torch.zeros_like(out), torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    m = k.shape[0]
    if not n or not m:
        return out, mag, lse
    pos = torch.arange(first, first + n, device=q.device)[:, None]
    key = torch.arange(m, device=q.device)[None]
    seen = key <= pos
    if window:
        seen &= key > pos - window
    some = seen.any(1)
    for h in range(heads):
        kk, vv = k[:, h // group].double(), v[:, h // group].double()
        t = torch.where(seen, (q[:, h].double() @ kk.T) * scale, -math.inf)  # -inf where an infinite key points away
        p = torch.where(some[:, None], torch.softmax(t, -1), 0.0)
        fine = torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
        o = p @ fine
        odd = ~torch.isfinite(vv)
        if odd.any():  # an infinity or NaN in v reaches exactly the rows that see it
            for j in odd.any(1).nonzero().flatten().tolist():
                o = o + torch.where(seen[:, j:j + 1] & odd[j][None], vv[j][None].expand_as(o), 0.0)
        out[:, h], mag[:, h] = o, p @ fine.abs()
        lse[:, h] = torch.where(some, torch.logsumexp(t, -1), -math.inf)
    return out, mag, lse


def attention_bound(want, mag, dtype, keys, vmax):
    """Elementwise error allowed: one rounding of the output, one of every
    weight (bounded by the sum of p |v|), weights below the type's smallest
    normal (2^-24 each, fp16), and scores off by 2^-13 (a dot product of up to
    256 fp32 terms), which move numerator and denominator."""
    u = UNIT[dtype]
    return u * want.abs() + (u + 2.0 ** -12) * mag + keys * 2.0 ** -24 * vmax

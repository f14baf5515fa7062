"""Plain 64-bit forms of the decoder-attention operators, written from their
definitions with numpy; the GPU tests compare with these."""
import numpy as np

U16 = 2.0 ** -8    # half a unit in the last place of bf16, relative
UH = 2.0 ** -11    # of fp16


def bf16(x):
    """x rounded to bf16 (nearest, ties to even), as float32."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return (((b + 0x7FFF + ((b >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


def frequencies(rot, base=10000.0, kind="none", factor=1.0, context=0.0, slow=1.0, fast=32.0):
    i = np.arange(rot // 2)
    f = np.float64(base) ** (-2.0 * i / rot)
    if kind == "linear":
        f = f / factor
    elif kind == "base":
        f = (base * factor ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
    elif kind == "parts":
        keep = np.clip((context * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


def rotate(x, table, positions, layout, transpose=False):
    """x [tokens, heads, d] in 64 bits; table [positions, rot / 2, 2]."""
    x = np.asarray(x, np.float64)
    c, s = (np.asarray(table, np.float64)[positions][:, None, :, i] for i in (0, 1))
    s = -s if transpose else s
    half = c.shape[-1]
    first, second = ((slice(0, half), slice(half, 2 * half)) if layout == "half" else
                     (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    y = x.copy()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def e4m3_values():
    """The value of each of the 256 codes."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if (c & 127) == 127 else (-x if c & 128 else x)
    return v


VALUES = e4m3_values()
_GRID = VALUES[:127]  # codes 0 .. 126: the values >= 0, ascending


def e4m3(x):
    """Codes of x: nearest, ties to even, |x| above 448 to 448, NaN to NaN."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    a = np.where(np.isnan(a), 0.0, a)
    hi = np.clip(np.searchsorted(_GRID, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _GRID[hi] - a, a - _GRID[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(_GRID[hi] == a, hi, code)
    code = np.where(np.signbit(x), code | 128, code)
    return np.where(np.isnan(x), 127, code).astype(np.uint8)


def exponent(amax):
    """Smallest e in [-100, 119] with amax <= 448 * 2^e; 0 for amax 0."""
    if amax == 0:
        return 0
    e = -100
    while e < 119 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def append(codes, scales, x, starts, before, pages):
    """The 64-bit x [tokens, heads, d] into codes [pages, heads, page, d] and
    scales [pages, heads], in place."""
    page = codes.shape[2]
    for s in range(len(before)):
        done, n = 0, starts[s + 1] - starts[s]
        while done < n:
            at = before[s] + done
            p, slot = pages[s][at // page], at % page
            m = min(n - done, page - slot)
            part = x[starts[s] + done: starts[s] + done + m]
            for h in range(codes.shape[1]):
                v = part[:, h]
                v = np.where(np.isfinite(v), v, np.nan)
                e = exponent(np.nanmax(np.abs(v), initial=0.0) if np.isfinite(v).any() else 0.0)
                if slot:
                    was = int(np.log2(scales[p, h]))
                    if e > was:
                        codes[p, h, :slot] = e4m3(VALUES[codes[p, h, :slot]] * 2.0 ** (was - e))
                    e = max(e, was)
                codes[p, h, slot: slot + m] = e4m3(v * 2.0 ** -e)
                scales[p, h] = 2.0 ** e
            done += m


def attention(q, k, v, scale, sees):
    """q [n, d], k and v [m, d] in 64 bits, sees[i] keys of query i: (o, lse,
    sum of p |v|: what a relative error of the weights can change o by)."""
    with np.errstate(all="ignore"):
        x = scale * (q @ k.T)
        x = np.where(np.arange(k.shape[0])[None] < np.asarray(sees)[:, None], x, -np.inf)
        top = np.max(x, axis=1, initial=-np.inf, keepdims=True)
        p = np.exp(x - np.where(np.isneginf(top), 0.0, top))
        p = np.where(np.isneginf(x), 0.0, p)
        total = p.sum(1, keepdims=True)
        lse = np.where(total[:, 0] > 0, np.where(np.isneginf(top), 0.0, top)[:, 0] + np.log(total[:, 0]), -np.inf)
        w = np.where(total > 0, p / total, 0.0)
    vv = np.where((w > 0).any(0)[:, None], v, 0.0)  # a key that nothing sees does not count
    return w @ vv, lse, w @ np.abs(vv)

"""Plain numpy restatement of the operators on a paged key/value cache, in 64 bits, and the number formats they use.
Test infrastructure only."""
import numpy as np


def bf16_bits(x):
    """Nearest bfloat16, ties to even, as uint16."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def encode(x, kind):
    return bf16_bits(x) if kind == "bf16" else np.asarray(x, np.float16).view(np.uint16)


def decode(u, kind):
    if kind == "bf16":
        return (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return u.view(np.float16).astype(np.float64)


def _e4m3_table():
    t = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        t[c] = np.nan if c & 127 == 127 else -v if c & 128 else v
    return t


E4M3 = _e4m3_table()
_SIZES = E4M3[:127]          # 0 ... 448, ascending


def e4m3_code(x):
    """Nearest e4m3 code of what is at most 448 in size, ties to the even code; NaN where not finite."""
    x = np.asarray(x, np.float64)
    size = np.minimum(np.abs(np.where(np.isfinite(x), x, 0)), 448.0)
    hi = np.clip(np.searchsorted(_SIZES, size), 1, 126)
    lo = hi - 1
    down, up = size - _SIZES[lo], _SIZES[hi] - size
    c = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.where(np.isfinite(x), c | np.where(np.signbit(x), 128, 0), 0x7F).astype(np.uint8)


def need_of(amax):
    """Smallest 2^e, -64 <= e <= 119, with amax <= 448 * 2^e."""
    for e in range(-64, 120):
        if amax <= 448 * 2.0 ** e:
            return 2.0 ** e
    return 2.0 ** 119


def turn(x, pos, cos, sin, rotary, interleaved, sections=None, positions=None):
    """x [heads][dim] (64 bits) of one row; pos: its position; positions: one for each axis."""
    y = np.array(x, np.float64)
    half = rotary // 2
    axis = np.repeat(np.arange(len(sections)), sections) if positions is not None else None
    for i in range(half):
        t = positions[axis[i]] if positions is not None else pos
        c, s = (cos[t, i], sin[t, i]) if 0 <= t < len(cos) else (np.nan, np.nan)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    return y


def attend(q, keys, values, scale, visible):
    """q [rows][dim]; keys, values [context][dim]; visible [rows][context]. (out, lse, sum w |v|, largest score's size)."""
    rows = len(q)
    out, lse, size = np.zeros_like(q), np.full(rows, -np.inf), np.zeros_like(q)
    top = np.zeros(rows)
    for r in range(rows):
        at = np.nonzero(visible[r])[0]
        if not len(at):
            continue
        with np.errstate(all="ignore"):
            s = (keys[at] @ q[r]) * scale
            top[r] = (np.abs(keys[at]) @ np.abs(q[r])).max() * abs(scale)
            m = s.max()
            if m == -np.inf:
                continue
            w = np.exp(s - m)
            l = w.sum()
            out[r], lse[r], size[r] = (w @ values[at]) / l, m + np.log(l), (w @ np.abs(values[at])) / l
    return out, lse, size, top

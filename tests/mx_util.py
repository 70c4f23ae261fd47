"""Plain restatement of the microscaled form in numpy, in 64 bits (include/qagg.h): what the library's calls are compared with."""
import numpy as np

FP4, INT8 = 4, 8
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(x, fmt):
    """x: [columns, rows] -> (elements [columns, blocks, 32], scale bytes [columns, blocks])."""
    x = np.asarray(x, np.float64)
    n, m = x.shape
    b = -(-m // 32)
    g = np.zeros((n, b * 32))
    g[:, :m] = x
    g = g.reshape(n, b, 32)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    top = np.abs(g).max(-1, initial=0.0)
    e = np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - (2 if fmt == FP4 else 0)
    e = np.where(top > 0, np.maximum(e, -127), -127)
    a = np.abs(np.ldexp(g, -e[..., None]))
    if fmt == INT8:
        el = np.minimum(np.rint(a * 64), 127) / 64  # rint: ties to even
    else:
        step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
        el = np.minimum(np.rint(a / step) * step, 6.0)
    el = np.where(np.signbit(g), -el, el)
    return el, np.where(bad, 255, e + 127).astype(np.uint8)


def tile(bytes_):
    """scale bytes [columns, blocks] -> the stored array."""
    n, b = bytes_.shape
    full = np.zeros((-(-n // 128) * 128, -(-b // 4) * 4), np.uint8)
    full[:n, :b] = bytes_
    # [tile of columns, 32-column group, column in it][tile of blocks, block] -> tiles of [column % 32][group][block]
    return full.reshape(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4).transpose(0, 3, 2, 1, 4).ravel().copy()


def pack(x, fmt):
    """Stored codes and scales of x ([columns, rows]), as uint8 arrays."""
    el, s = quantize(x, fmt)
    n = el.shape[0]
    if fmt == INT8:
        codes = (el * 64).astype(np.int8).view(np.uint8).reshape(n, el.shape[1] * 32)
    else:
        c = np.searchsorted(LEVELS, np.abs(el)).astype(np.uint8) + 8 * np.signbit(el).astype(np.uint8)
        c = np.where((s == 255)[..., None], 0, c).astype(np.uint8).reshape(n, el.shape[1] * 32)
        codes = c[:, 0::2] | (c[:, 1::2] << 4)
    return np.ascontiguousarray(codes).ravel(), tile(s)


def values(x, fmt):
    """What the packed x stands for, [columns, rows] in 64 bits."""
    el, s = quantize(x, fmt)
    v = np.ldexp(el, s.astype(np.int64)[..., None] - 127)
    v = np.where((s == 255)[..., None], np.nan, v)
    return v.reshape(x.shape[0], el.shape[1] * 32)[:, : x.shape[1]]

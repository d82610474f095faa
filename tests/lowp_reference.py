"""The low-precision operators in 64 bits, from their definitions: codes of 8 and 4 bits with scales, the root-mean-square norm
in front of them, and the product of two sets of codes.  Nothing here uses the library."""
import numpy as np

BLOCK = 32
INT8, MXFP8, MXFP4 = 0, 1, 2
TOP_POWER = {MXFP8: 8, MXFP4: 2}


def grid(fmt):
    """The non-negative numbers of the format by code, ascending."""
    if fmt == MXFP4:
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    e, f = np.divmod(np.arange(127), 8)
    return np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))


def blocks_of(d):
    return (d + BLOCK - 1) // BLOCK


def split_blocks(x):
    n, d = x.shape
    out = np.zeros((n, blocks_of(d) * BLOCK))
    out[:, :d] = x
    return out.reshape(n, blocks_of(d), BLOCK)


def round_to(v, fmt):
    """Codes (without sign) of the numbers nearest to v >= 0: halfway to the even code, beyond the last one to it."""
    g = grid(fmt)
    mid = (g[:-1] + g[1:]) / 2
    code = np.searchsorted(mid, v, side="left")
    tie = (code < len(mid)) & (v == mid[np.minimum(code, len(mid) - 1)])
    return code + (tie & (code % 2 == 1))


def mx_codes(x, fmt):
    """(codes [n][nb][32], one per element, sign included; biased scales [n][nb]) of 64-bit rows."""
    b = split_blocks(np.asarray(x, dtype=np.float64))
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(top)
    with np.errstate(divide="ignore", invalid="ignore"):
        power = np.floor(np.log2(np.where(bad | (top == 0), 1.0, top)))
    # log2 rounds: put the power right where it does
    safe = np.where(bad | (top == 0), 1.0, top)
    power = power - (safe < np.ldexp(1.0, power.astype(int))) + (safe >= np.ldexp(1.0, power.astype(int) + 1))
    biased = np.clip(power - TOP_POWER[fmt] + 127, 0, 254).astype(int)
    biased = np.where(top == 0, 0, biased)
    scaled = np.where(bad[..., None], 0.0, b) * np.ldexp(1.0, 127 - biased)[..., None]
    code = round_to(np.abs(scaled), fmt) | np.where(np.signbit(scaled), 8 if fmt == MXFP4 else 128, 0)
    code = np.where(bad[..., None], 0, code)
    return code.astype(np.uint8), np.where(bad, 255, biased).astype(np.uint8)


def pack(code, fmt):
    """One code per element [n][nb][32] -> the bytes of a row [n][nb * 16 or 32]."""
    n = code.shape[0]
    flat = code.reshape(n, -1)
    return flat.copy() if fmt == MXFP8 else (flat[:, 0::2] | (flat[:, 1::2] << 4)).astype(np.uint8)


def unpack(bytes_, fmt):
    return bytes_ if fmt == MXFP8 else np.stack((bytes_ & 15, bytes_ >> 4), -1).reshape(bytes_.shape[0], -1)


def mx_values(bytes_, scales, fmt):
    """64-bit values [n][nb * 32] of packed codes."""
    c = unpack(bytes_, fmt).astype(int)
    half = 8 if fmt == MXFP4 else 128
    g = np.append(grid(fmt), np.nan) if fmt == MXFP8 else grid(fmt)
    v = np.where(c >= half, -1.0, 1.0) * g[c % half]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return v * np.repeat(s, BLOCK, axis=1)


def int8_codes(y, fixed=0.0):
    """(codes, scales) in the arithmetic of 32 bits that the definition names."""
    y = np.asarray(y, dtype=np.float32)
    f = np.float32
    with np.errstate(all="ignore"):
        if fixed:
            v = y * (f(1) / f(fixed))
            return np.rint(np.clip(np.where(np.isnan(v), f(0), v), f(-127), f(127))).astype(np.int8), \
                np.full(len(y), fixed, np.float32)
        top = np.abs(y).max(-1)
        bad = ~np.isfinite(top)
        pre = np.where(top < f(2.0 ** -90), f(2.0 ** 64), f(1))
        inv = np.where((top > 0) & ~bad, f(127) / (top * pre), f(0)).astype(np.float32)
        v = y * pre[:, None].astype(np.float32) * inv[:, None]
        code = np.rint(np.clip(v, f(-127), f(127)))
        return np.where(bad[:, None], 0, code).astype(np.int8), np.where(bad, f(np.nan), top / f(127)).astype(np.float32)


def rms_norm(x, residual, weight, eps):
    h = np.asarray(x, dtype=np.float64)
    if residual is not None:
        h = h + np.asarray(residual, dtype=np.float64)
    y = h / np.sqrt((h ** 2).mean(-1, keepdims=True) + eps)
    return y if weight is None else y * np.asarray(weight, dtype=np.float64)


def between(values, y, delta, quantised):
    """Whether every value is one that some y' with |y' - y| <= delta |y| is quantised to."""
    around = [quantised(y * (1 + s)) for s in (-delta, 0.0, delta)]
    lo, hi = np.minimum.reduce(around), np.maximum.reduce(around)
    return (values >= lo) & (values <= hi)

"""Rows of 4-bit codes with a scale and a zero point per group, in 64 bits, from their definitions.  Nothing here uses the
library."""
import numpy as np

F32, F16, BF16 = 0, 1, 2
TOP = {F32: float(np.finfo(np.float32).max), F16: 65504.0, BF16: float(2.0 ** 128 - 2.0 ** 120)}


def round_to_type(v, kind):
    """64-bit numbers rounded to fp32 and from there to the type, halfway to even, as 64-bit numbers."""
    with np.errstate(over="ignore"):
        v = np.asarray(v, dtype=np.float64).astype(np.float32)
        if kind == F32:
            return v.astype(np.float64)
        if kind == F16:
            return v.astype(np.float16).astype(np.float64)
    bits = np.ascontiguousarray(v).view(np.uint32)
    up = (bits + 0x7fff + ((bits >> 16) & 1)) & np.uint32(0xffff0000)
    return np.where(np.isfinite(v), up.astype(np.uint32).view(np.float32), v).astype(np.float64)


def groups_of(d, group):
    return (d + group - 1) // group


def split(x, group):
    n, d = x.shape
    out = np.zeros((n, groups_of(d, group) * group))
    out[:, :d] = x
    return out.reshape(n, -1, group)


def quantise(x, group, scale_type, with_zeros):
    """(codes, one per element [n][groups][group]; scales; zeros)."""
    g = split(np.asarray(x, dtype=np.float64), group)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    if with_zeros:
        low, high = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
        scale = round_to_type(np.minimum((high - low) / 15, TOP[scale_type]), scale_type)
    else:
        scale = round_to_type(np.minimum(np.abs(g).max(-1) / 7, TOP[scale_type]), scale_type)
    some = np.where(scale > 0, scale, 1.0)
    zero = np.clip(np.rint(-low / some), 0, 15) * (scale > 0) if with_zeros else np.full(scale.shape, 8.0)
    code = np.clip(np.rint(g / some[..., None]) * (scale > 0)[..., None] + zero[..., None], 0, 15)
    return code.astype(np.uint8), np.where(bad, np.nan, scale), zero.astype(np.uint8)


def pack(code):
    flat = code.reshape(code.shape[0], -1)
    return (flat[:, 0::2] | (flat[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed, group):
    flat = np.stack((packed & 15, packed >> 4), -1)
    return flat.reshape(packed.shape[0], -1, group)


def values(code, scale, zero, d):
    with np.errstate(invalid="ignore"):
        v = (code.astype(np.float64) - zero.astype(np.float64)[..., None]) * scale[..., None]
    return v.reshape(code.shape[0], -1)[:, :d]

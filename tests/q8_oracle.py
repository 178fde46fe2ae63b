"""The 8-bit row format and the operators on it, restated in 64-bit numpy from their definition: codes are found by
searching the list of e4m3 values, scales by comparing with 448 * 2^p, everything else by the formulas."""
import numpy as np
import torch

GROUP = 32
NAN_CODE = 0x7F
TORCH_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_CODES = {"f32": 0, "f16": 1, "bf16": 2}


def _code_values():
    values = np.empty(256)
    for c in range(256):
        exponent, mantissa = (c >> 3) & 15, c & 7
        v = (mantissa / 8) * 2.0 ** -6 if exponent == 0 else (1 + mantissa / 8) * 2.0 ** (exponent - 7)
        values[c] = -v if c & 128 else v
    values[[0x7F, 0xFF]] = np.nan
    return values


CODE_VALUES = _code_values()
MAGNITUDES = CODE_VALUES[:0x7F]  # ascending, code = index, 448 the last


def groups(n):
    return -(-n // GROUP)


def scale_bytes(top):
    """Smallest b of 0..246 with top <= 448 * 2^(b - 127), else 246; 0 for zero."""
    table = 448 * 2.0 ** (np.arange(247) - 127.0)
    return np.minimum(np.searchsorted(table, top, side="left"), 246).astype(np.uint8)


def codes_of(y):
    """Nearest e4m3 code, ties to the even code, saturating; NaN and infinities get the NaN code."""
    a = np.minimum(np.abs(np.nan_to_num(y, nan=0.0, posinf=0.0, neginf=0.0)), 448.0)
    hi = np.clip(np.searchsorted(MAGNITUDES, a, side="left"), 0, len(MAGNITUDES) - 1)
    lo = np.maximum(hi - 1, 0)
    below, above = a - MAGNITUDES[lo], MAGNITUDES[hi] - a
    pick = np.where(below < above, lo, np.where(above < below, hi, np.where(lo % 2 == 0, lo, hi)))
    pick = np.where(MAGNITUDES[hi] == a, hi, pick)
    code = pick.astype(np.uint8) | np.where(np.signbit(y), 128, 0).astype(np.uint8)
    return np.where(np.isfinite(y), code, np.uint8(NAN_CODE))


def pack(x):
    """(codes, scale bytes) of the rows of x, float64 of any leading shape."""
    n = x.shape[-1]
    codes = np.empty(x.shape, np.uint8)
    scales = np.empty((*x.shape[:-1], groups(n)), np.uint8)
    for g in range(groups(n)):
        part = x[..., g * GROUP:(g + 1) * GROUP]
        top = np.where(np.isfinite(part), np.abs(part), 0).max(-1)
        scales[..., g] = scale_bytes(top)
        with np.errstate(invalid="ignore"):
            codes[..., g * GROUP:(g + 1) * GROUP] = codes_of(part / 2.0 ** (scales[..., g:g + 1].astype(float) - 127))
    return codes, scales


def unpack(codes, scales):
    s = 2.0 ** (scales.astype(float) - 127)
    return CODE_VALUES[codes] * np.repeat(s, GROUP, -1)[..., :codes.shape[-1]]


def rounded(x, kind):
    """float64 rounded once to the type, saturating at its largest finite value (every value of a code is an f32 value, so
    the way through f32 adds no rounding)."""
    top = torch.finfo(TORCH_TYPES[kind]).max
    return torch.from_numpy(np.clip(x, -top, top)).to(torch.float32).to(TORCH_TYPES[kind])


def sigmoid(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + e), e / (1 + e))


def silu_mul(g, u):
    return g * sigmoid(g) * u


def silu_mul_grad(g, u, dh):
    """(dgate, dup, size of dgate's terms before they are added)"""
    s, q = sigmoid(g), sigmoid(-g)
    return dh * u * s * (1 + g * q), dh * g * s, np.abs(dh * u) * s * (1 + np.abs(g) * q)


# ---- the same for large shapes, in torch on whatever device x is on -----------------------------------------------

def torch_pack(x):
    """pack() with scales taken from the binary exponent and codes by torch's own conversion; exact for 32-bit inputs."""
    x = x.float()
    n = x.shape[-1]
    full = groups(n) * GROUP
    g = torch.nn.functional.pad(x, (0, full - n)).unflatten(-1, (-1, GROUP))
    good = g.isfinite()
    top = torch.where(good, g.abs(), 0).amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)
    b = torch.where(top > 0, (exponent + 118 + (mantissa > 0.875)).clamp(0, 246), 0)
    inverse = ((254 - b) << 23).to(torch.int32).view(torch.float32)
    codes = torch.where(good, (g * inverse).clamp(-448, 448), 0).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(good, codes, NAN_CODE)
    return codes.flatten(-2)[..., :n], b.squeeze(-1).to(torch.uint8)


def torch_unpack(codes, scales):
    s = torch.exp2(scales.double() - 127).repeat_interleave(GROUP, -1)[..., :codes.shape[-1]]
    return codes.view(torch.float8_e4m3fn).double() * s

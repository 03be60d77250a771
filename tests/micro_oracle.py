"""The ray-head operators (vorotracing_amd.micro) from their definitions, in
64-bit numpy: the oracle of their tests.  Values of the inputs' types are
exact in float64, so quantised results are compared bit for bit."""
import numpy as np
import torch
from scipy.special import erfc

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# every e4m3 magnitude, by code 0..126 (127 is NaN)
E4M3 = np.array([(c % 8) * 2.0 ** -9 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) for c in range(127)])


def nearest(values, a):
    """Index of the entry of ascending `values` nearest to each a >= 0; a tie
    goes to the even index, what lies above the last to the last."""
    hi = np.clip(np.searchsorted(values, a), 1, len(values) - 1)
    lo = hi - 1
    dl, dh = a - values[lo], values[hi] - a
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def _blocks(x, fill=0.0):
    rows, width = x.shape
    n = -(-width // 32)
    b = np.full((rows, n * 32), fill)
    b[:, :width] = x
    return b.reshape(rows, n, 32)


def scale_code(top, largest):
    """Biased exponent of 2^(floor(log2 top) - largest), at least 0."""
    e = np.frexp(top)[1] - 1
    return np.where(top > 0, np.maximum(e - largest + 127, 0), 0).astype(np.int64)


def mx4(x):
    """(codes u8 (rows, 16 blocks), scales u8 (rows, blocks), values f64) of f64 rows."""
    b = _blocks(np.asarray(x, np.float64))
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    c = scale_code(np.abs(b).max(-1, initial=0.0), 2)
    q = b / np.exp2(c - 127.0)[..., None]
    i = nearest(E2M1, np.abs(q))
    sign = np.signbit(b)
    code = np.where(bad[..., None], 0, i + 8 * sign).reshape(b.shape[0], b.shape[1] * 32)
    packed = (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8)
    v = np.where(sign, -1.0, 1.0) * E2M1[i] * np.exp2(c - 127.0)[..., None]
    v = np.where(bad[..., None], np.nan, v).reshape(b.shape[0], b.shape[1] * 32)[:, :np.shape(x)[1]]
    return packed, np.where(bad, 255, c).astype(np.uint8), v


def ckpt8(x):
    """(codes u8 (rows, width), scales u8 (rows, blocks), values f64) of f64 rows."""
    x = np.asarray(x, np.float64)
    b = _blocks(x)
    fine = np.isfinite(b)
    c = scale_code(np.where(fine, np.abs(b), 0.0).max(-1, initial=0.0), 7)
    q = np.where(fine, b, 0.0) / np.exp2(c - 127.0)[..., None]
    i = nearest(E4M3, np.abs(q))
    i = np.where((i == 0) & (q != 0), 1, i)
    sign = np.signbit(np.where(fine, b, 0.0))
    code = np.where(fine, i + 128 * sign, 127).reshape(x.shape[0], b.shape[1] * 32)[:, :x.shape[1]].astype(np.uint8)
    v = np.where(fine, np.where(sign, -1.0, 1.0) * E4M3[i] * np.exp2(c - 127.0)[..., None], np.nan)
    return code, c.astype(np.uint8), v.reshape(x.shape[0], b.shape[1] * 32)[:, :x.shape[1]]


def act(z, name):
    with np.errstate(over="ignore", invalid="ignore"):
        if name == "relu":
            return np.where(np.isnan(z), z, np.maximum(z, 0.0))
        if name == "silu":
            return z / (1 + np.exp(-z))
        if name == "gelu":
            return 0.5 * z * erfc(-z * np.sqrt(0.5))
    return z


def slope(z, name):
    if name == "relu":
        return np.where(np.isnan(z), z, (z > 0).astype(np.float64))
    if name == "silu":
        s = 1 / (1 + np.exp(-np.clip(z, -700, 700)))
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * erfc(-z * np.sqrt(0.5)) + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    return np.where(np.isnan(z), z, 1.0)


def act_error(z, name):
    """How far an f32 evaluation of act may be from act(z): a few roundings
    (2^-24 each, 8 counted as 2^-21) of each factor; the exponent of exp and of
    erfc carries its argument's rounding, up to z^2 times."""
    if name in ("none", "relu"):
        return np.zeros_like(z)
    return 2.0 ** -21 * (1 + z * z) * np.abs(act(z, name)) + 2.0 ** -126


def slope_error(z, name):
    if name in ("none", "relu"):
        return np.zeros_like(z)
    if name == "silu":
        s = 1 / (1 + np.exp(-np.clip(z, -700, 700)))
        parts = s + np.abs(z) * s * (1 - s)
    else:
        parts = 0.5 * erfc(-z * np.sqrt(0.5)) + np.abs(z) * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    return 2.0 ** -21 * (1 + z * z) * np.abs(parts) + 2.0 ** -126


def rounding(v, dtype):
    """Half a step of `dtype` at magnitude |v|, one rounding of a result: 2^-p of it
    for p = 24, 11, 8 significant bits, half the smallest subnormal at least."""
    p, least = {torch.float32: (24, -150), torch.float16: (11, -25), torch.bfloat16: (8, -134)}[dtype]
    return np.abs(v) * 2.0 ** -p + 2.0 ** least


def held(v, dtype):
    """v with what is past the type's largest value as the infinity it rounds to (65504 + 16 in f16)."""
    if dtype != torch.float16:
        return v
    with np.errstate(invalid="ignore"):
        return np.where(np.abs(v) >= 65520.0, np.copysign(np.inf, v), v)


def f64(t):
    return t.detach().to("cpu", torch.float64).numpy()

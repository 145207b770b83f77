"""Plain 64-bit forms of the MLA attention operators (numpy), for the tests:
cache rows packed and unpacked, rotary positions, the append, the attention."""
import numpy as np

ROPE = 64
F16, BF16, FP8_F16, FP8_BF16 = 1, 30, 101, 130
FORMATS = [F16, BF16, FP8_F16, FP8_BF16]
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step relative to the value


def kind(fmt):
    return "f16" if fmt in (F16, FP8_F16) else "bf16"


def is_fp8(fmt):
    return fmt in (FP8_F16, FP8_BF16)


def row_bytes(fmt, latent):
    return (latent + 128 + latent // 32 + 15) // 16 * 16 if is_fp8(fmt) else 2 * (latent + ROPE)


# ---------------------------------------------------------------- 16-bit types
def to_bits(x, t):
    """float array -> bit pattern of type t (round to nearest even), from fp32."""
    x = np.asarray(x, np.float32)
    if t == "f16":
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, t):
    b = np.asarray(b, np.uint16)
    if t == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(x, t):
    return np.asarray(x, np.float32).astype(np.float64) if t == "f32" else from_bits(to_bits(x, t), t)


# -------------------------------------------------------------------- e4m3
_b = np.arange(256)
_e, _m = (_b >> 3) & 15, (_b & 7).astype(np.float64)
E4M3 = np.where(_e == 0, _m * 2.0 ** -9, (8 + _m) * 2.0 ** (_e.astype(np.float64) - 10)) * np.where(_b < 128, 1, -1)
E4M3[[127, 255]] = np.nan


def quantize(lat):
    """Codes (uint8) and scale bytes of latent rows [n, L] (float64 of fp32 values), the definition."""
    n, L = lat.shape
    g = lat.reshape(n, L // 32, 32)
    amax = np.max(np.abs(g), -1)
    bad = ~np.isfinite(g).all(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        k = np.ceil(np.log2(np.where(bad | (amax == 0), 1.0, amax) / 448.0))
    k = np.where(amax == 0, -15, np.clip(k, -15, 7)).astype(int)
    # log2 may round at the border: settle by comparison
    k = np.where((~bad) & (amax > 448.0 * 2.0 ** k) & (k < 7), k + 1, k)
    k = np.where((~bad) & (k > -15) & (amax <= 448.0 * 2.0 ** (k - 1.0)), k - 1, k)
    v = np.clip(np.where(bad[..., None], 0.0, g) / 2.0 ** k[..., None].astype(np.float64), -448, 448)
    pos = E4M3[:127]
    a = np.abs(v)
    hi = np.clip(np.searchsorted(pos, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - pos[lo], pos[hi] - a
    pick = np.where(dh < dl, hi, np.where(dl < dh, lo, np.where(lo % 2 == 0, lo, hi)))
    codes = (pick + np.where(np.signbit(v), 128, 0)).astype(np.uint8)
    scale = np.where(bad, 255, k + 127).astype(np.uint8)
    return codes.reshape(n, L), scale


def pack(lat, rope, fmt):
    """Cache rows as bytes."""
    lat, t = np.asarray(lat, np.float64), kind(fmt)
    n, L = lat.shape
    if not is_fp8(fmt):
        return to_bits(np.concatenate([lat, rope], 1), t).view(np.uint8).reshape(n, row_bytes(fmt, L))
    codes, scale = quantize(lat)
    out = np.zeros((n, row_bytes(fmt, L)), np.uint8)
    out[:, :L] = codes
    out[:, L:L + 128] = to_bits(rope, t).view(np.uint8).reshape(n, 128)
    out[:, L + 128:L + 128 + L // 32] = scale
    return out


def unpack(rows, L, fmt):
    """[n, L + 64] values (float64) that cache rows stand for."""
    t = kind(fmt)
    rows = np.ascontiguousarray(rows)
    if not is_fp8(fmt):
        return from_bits(rows.view(np.uint16), t)
    sb = rows[:, L + 128:L + 128 + L // 32].astype(np.float64)
    sc = np.where(sb == 255, np.nan, 2.0 ** (sb - 127))
    lat = E4M3[rows[:, :L]] * np.repeat(sc, 32, 1)
    return np.concatenate([lat, from_bits(np.ascontiguousarray(rows[:, L:L + 128]).view(np.uint16), t)], 1)


# -------------------------------------------------------------------- rotary
def freqs(dim=64, theta=10000.0, scale=40.0, orig=4096.0, fast=32.0, slow=1.0):
    i = np.arange(dim // 2, dtype=np.float64)
    f = theta ** (-2 * i / dim)
    if scale == 1.0:
        return f
    lo = max(np.floor(dim * np.log(orig / (fast * 2 * np.pi)) / (2 * np.log(theta))), 0)
    hi = min(np.ceil(dim * np.log(orig / (slow * 2 * np.pi)) / (2 * np.log(theta))), dim // 2 - 1)
    hi = max(hi, lo + 1)
    ramp = np.clip((i - lo) / (hi - lo), 0, 1)
    return f / scale * ramp + f * (1 - ramp)


def rotate(x, pos, f, half=False, mscale=1.0):
    """x [tokens, ..., dim] (float64) rotated by pos [tokens]."""
    m = len(f)
    a = np.outer(np.asarray(pos, np.float64), f)
    shape = (len(pos),) + (1,) * (x.ndim - 2) + (m,)
    c, s = (np.cos(a) * mscale).reshape(shape), (np.sin(a) * mscale).reshape(shape)
    p, q = (x[..., :m], x[..., m:]) if half else (x[..., 0::2], x[..., 1::2])
    u, v = p * c - q * s, p * s + q * c
    return np.concatenate([u, v], -1) if half else np.stack([u, v], -1).reshape(x.shape)


def rmsnorm(x, w, eps):
    return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * np.asarray(w, np.float64)


# ----------------------------------------------------------------- attention
def attend(q, kv, sees, scale, L):
    """q [tokens, heads, L + 64], kv [rows, L + 64], sees [tokens, rows] bool.
    out, lse, and the two sizes that the error bounds need: A = mean of |v|
    under the weights, and S = the largest scale * sum |q k|."""
    T, h, _ = q.shape
    out, A = np.zeros((T, h, L)), np.zeros((T, h, L))
    lse, S = np.full((T, h), -np.inf), np.zeros((T, h))
    for t in range(T):
        r = np.flatnonzero(sees[t])
        if not len(r):
            continue
        k = kv[r]
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (q[t] @ k.T)
            m = np.max(s, 1, keepdims=True)
            p = np.exp(s - m)
            l = p.sum(1, keepdims=True)
            p /= l
            out[t], A[t] = p @ k[:, :L], p @ np.abs(k[:, :L])
            lse[t] = (m + np.log(l))[:, 0]
            S[t] = np.max(abs(scale) * (np.abs(q[t]) @ np.abs(k).T), 1)
    return out, lse, A, S


def attend_bounds(out, lse, A, S, t):
    """Largest errors of the kernel's outputs.  A score is a sum of 36 steps
    of 16 exact products in fp32 that may be cut instead of rounded: off by
    40 * 2^-23 * S at most (d).  A weight is off by that, by the exponential's
    2^-21 and by half a step of its 16-bit form; the weighted sum by as much
    of A, plus the sums' own fp32 errors (2^-20 of A covers the few tiles and
    partial results of these tests); the result is rounded once more."""
    u = U[t]
    d = 40 * 2.0 ** -23 * S
    tol = (u + 2 * (np.exp(d) - 1) + 2.0 ** -20)[..., None] * A * 1.01 + u * np.abs(out) + 2.0 ** -24
    return tol, d + 2.0 ** -20 * (1 + np.abs(lse))

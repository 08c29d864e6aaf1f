"""Plain numpy statement of the 4-bit page format and of the operators around
it, in 64 bits: the quantizer, the page layout byte by byte, the attention and
the norm with the position rotation.  Shared by the mx4 and rope tests."""
import numpy as np

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
RANGE = {"k": (-24, 15), "v": (-22, 7)}
TILE = 32


def quantize(x, kind):
    """(codes uint8, exponents int, values f64) of rows x [..., D]; 999 stands
    for the exponent of a NaN block."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    lo, hi = RANGE[kind]
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    amax = np.abs(b).max(-1)
    e = np.full(amax.shape, hi)
    for k in range(hi, lo - 1, -1):
        e = np.where(amax <= 7 * 2.0 ** k, k, e)
    y = np.abs(b) / 2.0 ** e[..., None]
    # nearest value, the even code where two are as near
    code = np.zeros(y.shape, np.int64)
    for c in range(1, 8):
        mid = (VALUES[c - 1] + VALUES[c]) / 2
        code = np.where((y > mid) | ((y == mid) & (c % 2 == 0)), c, code)
    sign = np.signbit(b)
    val = np.where(sign, -1.0, 1.0) * VALUES[code] * 2.0 ** e[..., None]
    code = code + 8 * sign
    val = np.where(bad[..., None], np.nan, val)
    return (code.astype(np.uint8).reshape(x.shape), np.where(bad, 999, e), val.reshape(x.shape))


def scale_byte(e, kind):
    e = np.asarray(e)
    if kind == "k":
        return np.where(e == 999, 255, e + 127).astype(np.uint8)
    return np.where(e == 999, 0x7E, 4 * (e + 23)).astype(np.uint8)


def code_place(D, kind, slot, dim):
    """(byte offset in the tile, nibble) of a token's code; slot in 0..31."""
    if kind == "k":
        j, m = (slot % 8) // 4, 4 * (slot // 8) + slot % 4
        h, b = dim // 128, dim % 128 // 32
        return ((j * (D // 128) + h) * 4 + b) * 256 + m * 16 + dim % 32 // 2, dim % 2
    c, t, n = dim // 64, 2 * (dim % 64 // 32) + dim % 2, dim % 32 // 2
    return c * 1024 + (slot // 8 * 16 + n) * 16 + 4 * t + slot % 8 // 2, slot % 2


def scale_place(D, kind, slot, block):
    if kind == "k":
        j, m = (slot % 8) // 4, 4 * (slot // 8) + slot % 4
        H = D // 128
        return 16 * D + (block % 4 * 16 + m) * 2 * H + j * H + block // 4
    return 16 * D + (slot // 8 * (D // 32) + block) * 8 + slot % 8


def page_bytes(Hkv, D, PT):
    return Hkv * 2 * (PT // TILE) * 17 * D


def write_rows(pages, Hkv, D, PT, bt, seqs, pos, k, v):
    """Rows k, v [n][Hkv][D] into the page bytes (uint8, flat)."""
    dims = np.arange(D)
    blocks = np.arange(D // 32)
    for kind, x in (("k", k), ("v", v)):
        code, e, _ = quantize(x, kind)
        sb = scale_byte(e, kind)
        for i, (s, p) in enumerate(zip(seqs, pos)):
            page, slot = int(bt[s, p // PT]), int(p % PT)
            for h in range(Hkv):
                base = (((page * Hkv + h) * 2 + (kind == "v")) * (PT // TILE) + slot // TILE) * 17 * D
                off, nib = code_place(D, kind, slot % TILE, dims)
                nib = np.broadcast_to(nib, dims.shape)
                for shift in (0, 4):
                    w = nib == shift // 4
                    at = base + off[w]
                    pages[at] = (pages[at] & (0xF0 >> shift)) | (code[i, h, w] << shift)
                pages[base + scale_place(D, kind, slot % TILE, blocks)] = sb[i, h]


def attend(q, k, v, scale, limits):
    """softmax(scale q.k) v of rows q [n][Hq][D] over k, v [L][Hkv][D] in 64
    bits; row i attends the first limits[i] tokens (none: zeros)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, Hq, D = q.shape
    G = Hq // k.shape[1]
    out = np.zeros(q.shape)
    for i in range(n):
        L = int(limits[i])
        if L <= 0:
            continue
        for h in range(Hq):
            s = scale * (k[:L, h // G] @ q[i, h])
            p = np.exp(s - s.max())
            out[i, h] = (p / p.sum()) @ v[:L, h // G]
    return out


def rope(x, freqs, positions, axis, adjacent, weight=None, eps=0.0):
    """Rows x [n][heads][D] normed over D and rotated: pair i by
    positions[axis[i]] * freqs[i]."""
    x = np.array(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    half = len(freqs)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
    ang = np.asarray(positions, np.float64)[axis].T * np.asarray(freqs, np.float64)  # [n][half]
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    u, w = x[..., a].copy(), x[..., b].copy()
    x[..., a] = u * c - w * s
    x[..., b] = w * c + u * s
    return x

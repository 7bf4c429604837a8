"""The 4-bit numbers of the cache and of the 4-bit weights, restated in numpy (64 bits) for the tests."""
import numpy as np


def quantise(x, group):
    """x [..., n] fp16 -> codes [..., ceil(n / group) * group], s and m [..., groups] (fp16)."""
    x = np.asarray(x, np.float16)
    n = x.shape[-1]
    ng = -(-n // group)
    codes = np.zeros(x.shape[:-1] + (ng * group,), np.uint8)
    s = np.zeros(x.shape[:-1] + (ng,), np.float16)
    m = np.zeros_like(s)
    for g in range(ng):
        v = x[..., g * group: (g + 1) * group].astype(np.float64)
        bad = ~np.isfinite(v).all(-1)
        v = np.where(bad[..., None], 0.0, v)
        lo, hi = v.min(-1), v.max(-1)
        sg = ((hi.astype(np.float32) - lo.astype(np.float32)) / np.float32(15)).astype(np.float16)
        with np.errstate(divide="ignore", invalid="ignore"):
            c = np.rint((v - lo[..., None]) / sg.astype(np.float64)[..., None])
        c = np.where((sg == 0)[..., None], 0.0, c).clip(0, 15)
        codes[..., g * group: g * group + v.shape[-1]] = c
        s[..., g] = np.where(bad, np.float16(np.nan), sg)
        m[..., g] = np.where(bad, np.float16(np.nan), lo.astype(np.float16))
    return codes, s, m


def values(codes, s, m):
    group = codes.shape[-1] // s.shape[-1]
    c = codes.astype(np.float64).reshape(s.shape + (group,))
    return (c * s.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]).reshape(codes.shape)


def to_f16(v):
    """What reading back gives: fp16, limited to +-65504."""
    with np.errstate(over="ignore"):
        return np.where(v > 65504, 65504.0, v).astype(np.float16)


def k_rows(codes):
    """[..., 32 ng] codes -> [..., 16 ng] bytes of cache rows: word j ng + g, feature f in nibble (f >> 1) + 4 (f & 1)."""
    ng = codes.shape[-1] // 32
    out = np.zeros(codes.shape[:-1] + (16 * ng,), np.uint8)
    for g in range(ng):
        for j in range(4):
            for f in range(8):
                p = (f >> 1) + 4 * (f & 1)
                out[..., 4 * (j * ng + g) + p // 2] |= codes[..., 32 * g + 8 * j + f] << (4 * (p & 1))
    return out


def v_rows(codes):
    """Unit i ng + g (16 bits), feature f in nibble f."""
    ng = codes.shape[-1] // 32
    out = np.zeros(codes.shape[:-1] + (16 * ng,), np.uint8)
    for g in range(ng):
        for i in range(8):
            for f in range(4):
                out[..., 2 * (i * ng + g) + f // 2] |= codes[..., 32 * g + 4 * i + f] << (4 * (f & 1))
    return out


def w4_arrays(codes, s, m, group):
    """Codes [out, 128 nb] and (s, m) [out, groups] -> the arrays of et_w4_pack."""
    out, width = codes.shape
    nb = width // 128
    arr = np.zeros((out // 16, nb, 2, 32, 16), np.uint8)
    params = np.zeros((out // 16, nb, 16, 128 // group, 2), np.float16)
    for r in range(out):
        p, h, i = r // 16, (r // 8) % 2, r % 8
        for b in range(nb):
            for n in range(4):
                for j in range(4):
                    for f in range(8):
                        q = (f >> 1) + 4 * (f & 1)
                        arr[p, b, h, 4 * i + j, 4 * n + q // 2] |= codes[r, 128 * b + 32 * n + 8 * j + f] << (4 * (q & 1))
            for g in range(128 // group):
                at = b * (128 // group) + g
                if at < s.shape[1]:
                    params[p, b, r % 16, g] = s[r, at], m[r, at]
    return arr, params


def attention(q, k, v, limits, scale, mask=None):
    """One head in 64 bits: q [n, d], k [L, d], v [L, dv]; row r sees the first limits[r] tokens."""
    out = np.zeros((q.shape[0], v.shape[1]))
    for r in range(q.shape[0]):
        n = int(limits[r])
        if n <= 0:
            continue
        x = (k[:n] @ q[r]) * scale
        seen = np.ones(n, bool)
        if mask is not None:
            seen = mask[r, :n] != -np.inf
            x = x + np.where(seen, mask[r, :n], 0.0)
        if not seen.any():
            continue
        x = x[seen]
        p = np.exp(x - (x.max() if not np.isnan(x).all() else 0.0))
        out[r] = (p[:, None] * v[:n][seen]).sum(0) / p.sum()
    return out

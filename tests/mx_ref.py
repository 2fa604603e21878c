"""Plain NumPy forms of MXFP4, the 4-bit cache's layout and attention over it, in 64 bits."""
import numpy as np

MAGS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([MAGS, -MAGS])


def encode(x):
    """codes [..., 32 n] and scale bytes [..., n] of x [..., 32 n] (f32), by the midpoints of the magnitudes."""
    b = np.asarray(x, np.float32).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    bits = np.abs(b).max(-1).view(np.uint32)
    e = (bits >> 23).astype(np.int64)
    ok = np.isfinite(b).all(-1)
    byte = np.where(~ok, 255, np.where(bits == 0, 127, np.maximum(e - 2, 0)))
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.abs(b.astype(np.float64)) * np.exp2(127.0 - byte)[..., None]
        code = np.zeros(b.shape, np.int64)
        for i in range(1, 8):
            mid = (MAGS[i - 1] + MAGS[i]) / 2
            code += (a >= mid) if i % 2 == 0 else (a > mid)
    code = np.where(ok[..., None], code + 8 * np.signbit(b), 0)
    return code.reshape(x.shape).astype(np.uint8), byte.astype(np.uint8)


def decode(code, byte):
    with np.errstate(over="ignore"):
        s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return (VALUES[code].reshape(byte.shape + (32,)) * s[..., None]).reshape(code.shape)


def rounded(x):
    """x as MXFP4 holds it: [..., n] with any n, f64."""
    n = x.shape[-1]
    pad = np.zeros(x.shape[:-1] + (-n % 32,), np.float32)
    return decode(*encode(np.concatenate([np.asarray(x, np.float32), pad], -1)))[..., :n]


def pack(code):
    return (code[..., ::2] | code[..., 1::2] << 4).astype(np.uint8)


def matrix(x):
    """data and scales arrays of a matrix [rows, cols], rows filled up to whole blocks."""
    pad = np.zeros((x.shape[0], -x.shape[1] % 32), np.float32)
    code, byte = encode(np.concatenate([np.asarray(x, np.float32), pad], 1))
    return pack(code), byte


def pages(k, v, page_len):
    """The bytes of whole pages whose tokens have K and V rows k, v [pages * page_len, n_kv, hd]."""
    n_kv, hd = k.shape[1:]
    n, kb = k.shape[0] // page_len, hd // 32
    out = np.zeros((n, n_kv, page_len * hd * 17 // 16), np.uint8)
    for p in range(n):
        for h in range(n_kv):
            parts = []
            for x, apart in ((k, False), (v, True)):
                code, byte = encode(x[p * page_len:(p + 1) * page_len, h])
                data = pack(code)
                if apart:
                    data = data.reshape(page_len // 8, 8, 16, kb).transpose(0, 2, 1, 3)
                parts += [data.reshape(-1), byte.reshape(page_len // 8, 8, kb).transpose(0, 2, 1).reshape(-1)]
            out[p, h] = np.concatenate(parts)
    return out


def attend(q, keys, k, v, pos, scale, window):
    """One query row q [heads, hd] at position pos over the tokens at positions `keys` with rows k, v
    [len(keys), n_kv, hd], in f64.  No token in sight: zeros."""
    heads, n_kv = q.shape[0], k.shape[1]
    see = (keys <= pos) & (keys > pos - window if window else keys >= 0)
    out = np.zeros(q.shape)
    if not see.any():
        return out
    for h in range(heads):
        kk, vv = k[see, h * n_kv // heads], v[see, h * n_kv // heads]
        s = kk @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        out[h] = p @ vv / p.sum()
    return out

"""The roundings of the 4-bit attention, made again in NumPy: what its parts of q and of the weights leave of
an output, and what would be missing without some of them.

q times scale log2 e is a sum of eight E2M1 parts, each an eighth of the one before; its products with K are exact
and summed in f32.  A weight is exp2 of an f32 difference, to one last place, and a sum of three bf16 parts, each cut
off; their products with V are summed in f32, as are the weights.
"""
import numpy as np

from tests import mx_ref


Q_PARTS = 8


def split(x, parts):
    """x f32 [..., hd] as the sum of its parts, f64."""
    x = x.astype(np.float64).reshape(x.shape[:-1] + (-1, 32))
    field = (np.abs(x).max(-1).astype(np.float32).view(np.uint32) >> 23).astype(np.int64)
    top, left = np.maximum(field - 1, 0), x.copy()
    for p in range(parts):
        unit = np.exp2(np.maximum(top - 3 * p, 0) - 127.0)[..., None]
        a, code = np.abs(left) / unit, np.zeros(left.shape, np.int64)
        for i in range(1, 8):
            mid = (mx_ref.MAGS[i - 1] + mx_ref.MAGS[i]) / 2
            code += (a >= mid) if i % 2 == 0 else (a > mid)
        left = left - np.sign(left) * mx_ref.MAGS[code] * unit
    return (x - left).reshape(x.shape[:-2] + (-1,))


def attend(rng, q, k, v, scale, n_q, n_p=3):
    """One head's row q [hd] f32 over the tokens k, v [n, hd] that it sees, with n_q parts of q and n_p of the weights."""
    f32 = np.float32
    x = q * (f32(scale) * f32(1.4426950408889634))
    s = f32(0)
    whole = split(x, n_q)
    for p in range(n_q, 0, -1):                            # the smallest parts first
        less = split(x, p - 1) if p > 1 else 0 * whole
        s = (s + k @ (whole - less)).astype(f32)
        whole = less
    w = np.exp2((s - s.max()).astype(np.float64)).astype(f32)
    w = (w * (1 + 2.0 ** -23 * rng.uniform(-1, 1, w.shape))).astype(f32)
    total, out, left = f32(0), np.zeros(v.shape[1], f32), w.copy()
    pieces = []
    for _ in range(n_p):
        pieces.append((left.view(np.uint32) & 0xFFFF0000).view(f32))
        left = left - pieces[-1]
    for at in range(0, len(w), 32):
        for piece in pieces[::-1]:
            out = (out + piece[at:at + 32].astype(np.float64) @ v[at:at + 32]).astype(f32)
        total = f32(total + w[at:at + 32].sum(dtype=f32))
    return (out * (f32(1) / total)).astype(np.float64)


def error(got, want, size):
    """Root mean square of the difference, in units of the mean sum of magnitudes of each row and head."""
    return float(np.sqrt(np.mean(((got - want) / size.mean(-1, keepdims=True)) ** 2)))


def limit(parts, want, size, steps=20, times=4):
    """What an output may be off by, in the units of `error`: four times what the parts' roundings leave by themselves,
    and the sums in the matrix units, which cut off what is below their last place, half a place (2^-24) a step: a
    row here has up to 4 chunks of 32 tokens with three parts each, and 4 waves' and 4 blocks' sums joined."""
    return times * error(parts, want, size) + steps * 2.0 ** -24 * error(want, 0 * want, size)


FORMS = ["decode", "prompt16", "prompt32", "runs", "runs32"]


def case(make, hd, form):
    """Cache, batch and query rows of a form of the call whose rows see 70 to 100 tokens at most, so that the parts'
    errors are not averaged away: single tokens, prompts in tiles of 16 and of 32 columns, and long sequences
    that several blocks share, of which only a few pages are there.  make: the class of a test's cache."""
    heads = {"decode": 4, "prompt16": 2, "prompt32": 8, "runs": 4, "runs32": 4}[form]
    lens = {"decode": [24, 40, 60, 33, 5, 48, 64, 17], "runs": [2500, 1400], "runs32": [2500]}.get(form, [48, 40])
    rows = {"decode": None, "runs": None, "runs32": [70]}.get(form, lens)
    c = make(hd + len(form), lens, rows, 2, hd, 32)
    if form.startswith("runs"):
        for s, n in enumerate(lens):
            last = (n - 1) // 32
            there = {last, last - 1, last - 2, 20}
            c.table[s, [t for t in range(c.width) if t not in there]] = -1
    return c, heads, c.rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)


def outputs(c, heads, q, scale, n_q, n_p, every=1):
    """Rows and heads (every so many of them): the places, f64 outputs, their sums of magnitudes, and those with the parts."""
    rng = np.random.default_rng(1)
    kd, vd = mx_ref.rounded(c.k), mx_ref.rounded(c.v)
    places, want, size, got, count = [], [], [], [], 0
    for row, s, pos in c.each_row():
        at = np.array([c.slot(s, t) for t in range(pos + 1) if c.slot(s, t) is not None])
        for h in range(heads):
            count += 1
            if count % every:
                continue
            k, v = kd[at, h * c.n_kv // heads], vd[at, h * c.n_kv // heads]
            p = k @ q[row, h].astype(np.float64) * scale
            p = np.exp(p - p.max())
            p /= p.sum()
            places.append((row, h))
            want.append(p @ v)
            size.append(p @ np.abs(v))
            got.append(attend(rng, q[row, h], k, v, scale, n_q, n_p))
    return tuple(np.array(places).T), np.array(want), np.array(size), np.array(got)


SHORT_FORMS = ["prompt16", "prompt32"]                     # (single tokens run the kernel of the former)
SHORT_STEPS = 5                                            # three parts of one chunk, its wave's sum, the division
SHORT_SCALE = 12                                           # over sqrt(hd): scores far apart


def short_case(make, hd, form):
    """The same for rows that see 20 tokens at most, one chunk, so that q is what they are off by."""
    group = 2 if form == "prompt16" else 8
    c = make(3 * hd + len(form), [20], [20], 2, hd, 32)
    return c, 2 * group, c.rng.standard_normal((20, 2 * group, hd)).astype(np.float32)

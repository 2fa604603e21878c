"""How near attention over shared prefixes has to come to 64 bits, element by element."""
import numpy as np

LAMBDA = 8.0


def attention_near(k, v, q, lens, starts, prefix_slots, prefix_lens, slots, scale, window=0):
    """many_ref.attention's arguments, finite wherever a row looks.  The rows' results in 64 bits and a bound of the
    error of each element in f32, with u = 2^-24, p the weights, o the result, s the scores (times scale):

      u [ L sqrt((2 hd + 16) sum_t p_t^2 (v_t - o)^2 A_t^2)      A_t = scale sum |q k_t|
        + sum_t p_t |v_t - o| (2 A_t + 5 |s_t - max s| + 40)
        + L sqrt(n + 80) (sum_t p_t |v_t| + |o|) + 8 sum_t p_t |v_t| ]

    A weight that is off by a factor of 1 + e moves o by p_t (v_t - o) e.  First line: up to 2 hd + 16 roundings of a score's
    products and sums, each up to u A_t, another set for each token.  Second: what tokens share, so that it may add up:
    q's rounding (A_t; twice, for the second order), the scale's and log2 e's (3 |s_t - max s|: a factor of all scores, of which
    a constant's part cancels), the exponent's subtraction (|s_t - max s| and up to 8 below the maximum), exp2 itself and the
    factors between maxima, waves and runs (40).  Third: n weights' sums and those of what waves and runs leave (80 at
    most), each rounding up to u of the sum of magnitudes; products, the division and its product.
    Sums of m independent roundings of mean zero are below L sqrt(m) u but for once in exp(L^2 / 2) / 2 = 4e13 times."""
    n_slots, max_seq, n_kv, hd = k.shape
    heads, u = q.shape[1], 2.0 ** -24
    want, off = np.zeros(q.shape), np.zeros(q.shape)
    for g in range(len(starts) - 1):
        for r in range(starts[g], starts[g + 1]):
            n, lp = int(lens[r]), int(prefix_lens[g])
            t = np.arange(max(0, n - window) if window else 0, n)
            own = slots[r] if slots.ndim == 1 else slots[r, np.clip(t - lp, 0, slots.shape[1] - 1)]
            at = np.where(t < lp, prefix_slots[g], own), t
            kk, vv = (x[at].transpose(1, 0, 2).astype(np.float64) for x in (k, v))       # [n_kv, tokens, hd]
            qq = q[r].astype(np.float64).reshape(n_kv, -1, hd)
            s = qq @ kk.transpose(0, 2, 1) * scale
            a = np.abs(qq) @ np.abs(kk).transpose(0, 2, 1) * abs(scale)
            top = s.max(-1, keepdims=True)
            p = np.exp(s - top)
            p /= p.sum(-1, keepdims=True)
            o = p @ vv
            w, m = (p * a) ** 2, p * (2 * a + 5 * (top - s) + 40)
            spread = w @ vv ** 2 - 2 * o * (w @ vv) + w.sum(-1, keepdims=True) * o ** 2
            apart = np.stack([[m[i, j] @ np.abs(vv[i] - o[i, j]) for j in range(m.shape[1])] for i in range(n_kv)])
            mass = p @ np.abs(vv)
            want[r] = o.reshape(heads, hd)
            off[r] = (u * (LAMBDA * np.sqrt((2 * hd + 16) * np.maximum(spread, 0)) + apart +
                           LAMBDA * np.sqrt(len(t) + 80) * (mass + np.abs(o)) + 8 * mass)).reshape(heads, hd)
    return want, off


def bf16(x):
    """Rounded to the nearest bf16."""
    return (((np.asarray(x, np.float32).view(np.uint32).astype(np.uint64) + 0x7FFF +
              (np.asarray(x, np.float32).view(np.uint32) >> 16 & 1)) >> 16 << 16).astype(np.uint32)).view(np.float32)


def want(b, window=0):
    """attention_near of a batch (test_gpu_many.Batch)."""
    return attention_near(b.k, b.v, b.q.reshape(-1, b.heads, b.hd), b.lens, b.starts, b.prefix_slots, b.prefix, b.slots, b.hd ** -0.5,
                          window)


_OWN = np.random.default_rng(5).integers(0, 60, 40).tolist()

# name, window, and sizes: a few tokens; several runs to a tile, which a second launch joins, in each head dimension; two
# tiles of columns to a block; groups beside each other
CASES = [
    ("shapes-64", 0, dict(seed=1, sizes=[5], prefix=[37], own=[9, 0, 3, 21, 1], n_kv=3, group=3, hd=64)),
    ("shapes-128", 0, dict(seed=1, sizes=[5], prefix=[37], own=[9, 0, 3, 21, 1], n_kv=2, group=5, hd=128)),
    ("shapes-256", 0, dict(seed=1, sizes=[5], prefix=[37], own=[9, 0, 3, 21, 1], n_kv=2, group=16, hd=256)),
    ("long-64", 0, dict(seed=5, sizes=[7], prefix=[3001], own=[97, 0, 97, 300, 97, 1, 97], n_kv=1, group=4, hd=64)),
    ("long-128", 0, dict(seed=5, sizes=[7], prefix=[3001], own=[97, 0, 97, 300, 97, 1, 97], n_kv=8, group=1, hd=128)),
    ("long-256", 0, dict(seed=5, sizes=[7], prefix=[3001], own=[97, 0, 97, 300, 97, 1, 97], n_kv=1, group=2, hd=256)),
    ("long-window", 1500, dict(seed=6, sizes=[7], prefix=[3001], own=[97, 1, 97, 300, 97, 1, 97], n_kv=2, group=4, hd=128)),
    ("wide", 0, dict(seed=15, sizes=[23, 1, 17], prefix=[2100, 30, 700], own=_OWN + [3], n_kv=1, group=6, hd=128)),
    ("wide-window", 2080, dict(seed=15, sizes=[23, 1, 17], prefix=[2100, 30, 700], own=_OWN + [3], n_kv=1, group=6, hd=128)),
    ("many-rows", 0, dict(seed=3, sizes=[64], prefix=[70], own=np.random.default_rng(3).integers(0, 25, 64).tolist(), n_kv=2,
                          group=1, hd=256)),
]


def lora_near(a):
    """An Adapters' rows (test_gpu_many) in 64 bits, and a bound of each element's error in f32: with v = A x, S_i = sum |A_i x|,
    scale c

      u |c| (L sqrt(2 k sum_i B_i^2 S_i^2) + (L sqrt(2 rank) + 4) sum_i |B_i v_i|) + 2 u (|base| + |y|)

    2 k roundings of up to u S_i for each v_i, which B carries on, and 2 rank of up to u sum |B_i v_i|; the scale, its product, the
    last sum."""
    x, base = a.x[:, :a.k].astype(np.float64), a.base[:, :a.m].astype(np.float64)
    y, off, u = base.copy(), np.zeros_like(base), 2.0 ** -24
    for r, p in enumerate(a.pick):
        if 0 <= p < a.n:
            c = 1.0 if a.scales is None else float(a.scales[p])
            aa, bb = a.a[p].astype(np.float64), a.b[p].astype(np.float64)
            v, s = aa @ x[r], np.abs(aa) @ np.abs(x[r])
            y[r] += c * (bb @ v)
            off[r] = u * abs(c) * (LAMBDA * np.sqrt(2 * a.k * (bb ** 2 @ s ** 2)) +
                                   (LAMBDA * np.sqrt(2 * a.rank) + 4) * (np.abs(bb) @ np.abs(v)))
    return y, off + 2 * u * (np.abs(base) + np.abs(y))


# name and sizes: one launch and two, bf16 and f32, rank in several tiles, more than 64 rows
LORA_CASES = [
    ("one-launch", dict(seed=1, n=4, rank=8, m=576, k=576, rows=3)),
    ("rows13", dict(seed=2, n=6, rank=16, m=512, k=4096, rows=13)),
    ("f32-rank64", dict(seed=3, n=5, rank=64, m=640, k=2048, rows=70, fmt="f32")),
    ("rank256", dict(seed=4, n=2, rank=256, m=100, k=700, rows=5)),
]

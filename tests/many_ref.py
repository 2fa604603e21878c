"""The operators for many continuations decoded together, in 64 bits with numpy."""
import numpy as np


def attention(k, v, q, lens, starts, prefix_slots, prefix_lens, slots, scale, window=0, out=None):
    """k, v [n_slots, max_seq, n_kv, hd], q [rows, heads, hd], slots [rows, stride] or [rows].  Returns the rows'
    results in 64 bits (rows of no group: out's) and how far f32 may be off for each row and head."""
    n_slots, max_seq, n_kv, hd = k.shape
    heads = q.shape[1]
    got = np.zeros(q.shape) if out is None else out.astype(np.float64)
    off = np.zeros(q.shape[:2])
    for g in range(len(starts) - 1):
        for r in range(starts[g], starts[g + 1]):
            n, lp = max(int(lens[r]), 0), max(int(prefix_lens[g]), 0)
            cells = []
            for t in range(max(0, n - window) if window else 0, n):
                if t < lp:
                    s = prefix_slots[g]
                elif slots.ndim == 1:
                    s = slots[r]
                else:
                    s = slots[r, t - lp] if t - lp < slots.shape[1] else -1
                if 0 <= s < n_slots and t < max_seq:
                    cells.append((s, t))
            got[r] = 0
            if not cells:
                continue
            at = tuple(np.array(cells).T)
            for h in range(heads):
                kk, vv = (x[at][:, h // (heads // n_kv)].astype(np.float64) for x in (k, v))
                qq = q[r, h].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk @ qq * scale
                    p = np.exp(s - s.max())
                    got[r, h] = (p / p.sum()) @ vv
                    # A score's hd products and sums, its scaling, and exp's argument are off by at most
                    # (hd + 8) 2^-24 of the sum of the products' magnitudes, which is what a weight is off
                    # relatively, as is their sum; n tokens' sums by 2^-24 each.
                    # (Infinities and NaN are compared as such.)
                    kk, vv, qq = (np.where(np.isfinite(x), np.abs(x), 0) for x in (kk, vv, qq))
                    off[r, h] = vv.max() * (2 * (hd + 8) * 2.0 ** -24 * (kk @ qq).max() * abs(scale) +
                                            2 * (len(cells) + 64) * 2.0 ** -24)
    return got, off


def select(logits, scores, n_out):
    """logits [groups, width, vocab], scores [groups, width] -> tokens, parents, scores [groups, n_out]."""
    groups, width, vocab = logits.shape
    tokens, parents, best = (np.zeros((groups, n_out), t) for t in (np.uint32, np.int32, np.float64))
    parents[:], best[:] = -1, -np.inf
    for g in range(groups):
        cand = []
        for b in range(width):
            z = logits[g, b].astype(np.float64)
            if not np.isfinite(scores[g, b]) or np.isnan(z).any() or z.max() == np.inf or z.max() == -np.inf:
                continue
            logp = z - (z.max() + np.log(np.exp(z - z.max()).sum()))
            top = np.argsort(-z, kind="stable")[:n_out]
            cand += [(-(scores[g, b] + logp[t]), b, i, t) for i, t in enumerate(top) if z[t] > -np.inf]
        for i, (s, b, _, t) in enumerate(sorted(cand)[:n_out]):
            tokens[g, i], parents[g, i], best[g, i] = t, b, -s
    return tokens, parents, best


def lora(base, x, a, b, scales, pick):
    """In 64 bits, and how far f32 may be off: an element's k products and sums, then rank's, the scale and the sum with base."""
    y, off = base.astype(np.float64), np.abs(base).astype(np.float64) * 2.0 ** -23
    k, rank = a.shape[2], a.shape[1]
    for r, p in enumerate(pick):
        if 0 <= p < len(a):
            s = 1.0 if scales is None else float(scales[p])
            aa, bb, xx = a[p].astype(np.float64), b[p].astype(np.float64), x[r].astype(np.float64)
            y[r] += s * (bb @ (aa @ xx))
            off[r] += (k + rank + 8) * 2.0 ** -24 * abs(s) * (np.abs(bb) @ (np.abs(aa) @ np.abs(xx)))
    return y, off

"""Beam search over a model in 64 bits, every hypothesis fed from its beginning."""
import copy

import numpy as np

from tests import modelgen


def log_probs(z):
    return z - (z.max() + np.log(np.exp(z - z.max()).sum()))


def search(W, prompt, max_new, width, penalty=1.0, stops=()):
    """Hypotheses (tokens, score), best first, and the smallest gap between two scores that decided something."""
    state = modelgen.Ref64(W)
    for t in prompt:
        z = state.forward_one(int(t))
    live, done, gap = [([], 0.0, state, log_probs(z))], [], np.inf
    n_cand = min(64, width * (1 + len(stops)))

    def finish(tok, score, n):
        done.append((score / n ** penalty, -len(done), tok, score))
        done.sort(reverse=True)
        del done[width:]

    def near(x):
        nonlocal gap
        x = np.sort(np.asarray(x))[::-1]
        if len(x) > 1:
            gap = min(gap, float(np.min(x[:-1] - x[1:])))

    for n in range(1, max_new + 1):
        cand = sorted(((s + lp[t], -b, -int(t)) for b, (_, s, _, lp) in enumerate(live) for t in np.argsort(-lp)[:n_cand + 1]),
                      reverse=True)
        near([c[0] for c in cand[:n_cand + 1]])
        nxt = []
        for i, (s, b, t) in enumerate(cand[:n_cand]):
            if len(nxt) == width:
                break
            tok, _, st, _ = live[-b]
            if -t in stops:
                if i < width:
                    finish(tok, s, n)
                continue
            nxt.append((tok + [-t], s, st))
        if not nxt or n == max_new:
            for tok, s, _ in nxt:
                finish(tok, s, n)
            break
        best = max(nxt[0][1] / (n + 1) ** penalty, nxt[0][1] / max_new ** penalty)
        if len(done) == width:
            gap = min(gap, abs(best - done[-1][0]))
            if best <= done[-1][0]:
                break
        live = []
        for tok, s, st in nxt:
            st = copy.copy(st)
            st.K, st.Vc = st.K.copy(), st.Vc.copy()
            live.append((tok, s, st, log_probs(st.forward_one(tok[-1]))))
    near([d[0] for d in done])
    return [(tok, score) for _, _, tok, score in done], gap

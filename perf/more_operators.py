"""Operators for many continuations decoded together, as cases that can be timed.

A case is one pass of one of four kinds.  With `own` false a pass computes the
operator in its plain form, from elementary torch operations; with `own` true it
makes the calls of include/atlas_kernels.h that a program makes.

  prefix   attention of one new token for each of a batch's rows, over an f32 cache
           of slots.  The rows of a group see the same first tokens (a prompt, a
           system prompt), kept once; then each its own.
  select   beam search's choice: the best continuations of a group's beams over
           the vocabulary, by the sum of log probabilities.
  reorder  beams take over the states of the beams they continue.
  lora     low-rank adapters, another one for each row, beside a shared
           projection whose output is given.

Sizes of a batch's members follow from the case, values from the seed.
"""
import ctypes as C
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"


def listed():
    return [
        # four beams of the 135M-sized model early in a conversation: the smallest call, latency
        dict(name="prefix_135m_beams4", kind="prefix", mode="beams", groups=1, rows=4, prefix=19, own=7, heads=9, kv=3,
             hd=64, window=0),
        # eight beams of a 7B model that continue a long document
        dict(name="prefix_7b_beams8", kind="prefix", mode="beams", groups=1, rows=8, prefix=4001, own=97, heads=32,
             kv=32, hd=128, window=0),
        # a grouped-query 1B model: conversations over five system prompts
        dict(name="prefix_1b_requests40", kind="prefix", mode="requests", groups=5, rows=40, prefix=2047, own=600,
             heads=32, kv=8, hd=64, window=0),
        # 64 requests over one long system prompt, grouped-query heads of 128
        dict(name="prefix_gqa_requests64", kind="prefix", mode="requests", groups=1, rows=64, prefix=8191, own=1023,
             heads=32, kv=8, hd=128, window=0),
        # one prompt, four beams, the vocabulary of the small models: latency
        dict(name="select_135m_beams4", kind="select", groups=1, width=4, vocab=49152, n_out=8),
        # eight prompts of eight beams over a 7B model's vocabulary
        dict(name="select_7b_beams8x8", kind="select", groups=8, width=8, vocab=100278, n_out=16),
        # the slots of each beam's tokens, 333 steps in, into the other of two tables
        dict(name="reorder_slots_beams8", kind="reorder", dtype="i32", states=1, groups=1, width=8, row=333, stride=512,
             in_place=False),
        # K and V of a 135M-sized model's 30 layers, 777 tokens in each beam's own cache
        dict(name="reorder_135m_caches", kind="reorder", dtype="f32", states=60, groups=1, width=6, row=777 * 192,
             stride=1024 * 192, in_place=True),
        # W_o of the 135M-sized model, one row: latency
        dict(name="lora_135m_row1", kind="lora", fmt="bf16", adapters=4, rank=8, rows=1, m=576, k=576),
        # a 7B model's W_o, a ragged batch of 13 requests
        dict(name="lora_7b_rows13", kind="lora", fmt="bf16", adapters=32, rank=16, rows=13, m=4096, k=4096),
        # up of a 7B model over packed prompts of five adapters
        dict(name="lora_7b_rows2047", kind="lora", fmt="bf16", adapters=5, rank=16, rows=2047, m=11008, k=4096),
        # adapters kept in f32, a wide rank, a middling batch
        dict(name="lora_1b_f32_rows70", kind="lora", fmt="f32", adapters=9, rank=64, rows=70, m=8192, k=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["prefix"] * 8 + ["select"] * 4 + ["reorder"] * 3 + ["lora"] * 5)
    if kind == "prefix":
        hd = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 3, 4, 8, 16, 32])
        heads = kv * rng.choice([g for g in (1, 1, 2, 3, 4, 5, 7, 8, 16) if kv * g <= 64])
        mode = rng.choice(["beams", "requests"])
        groups = _log(rng, 1, 16)
        rows = groups * _log(rng, 1, 16) if mode == "beams" else max(groups, _log(rng, 1, 96))
        # 60 million cache elements read, 400 million in all slots, scores of all rows and heads
        own_len = _log(rng, 1, min(1024, 30_000_000 // (rows * kv * hd)))
        prefix = _log(rng, 1, min(16384, 30_000_000 // (groups * kv * hd), 400_000_000 // ((rows + groups) * kv * hd) - own_len,
                                  18_000_000 // (rows * heads)))
        return dict(kind=kind, mode=mode, groups=groups, rows=rows, prefix=prefix, own=own_len, heads=heads, kv=kv, hd=hd,
                    window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    if kind == "select":
        vocab = _log(rng, 256, 128256)
        width = _log(rng, 1, 16)
        return dict(kind=kind, groups=_log(rng, 1, min(32, max(1, 6_400_000 // (vocab * width)))), width=width, vocab=vocab,
                    n_out=min(width * rng.choice([1, 2, 2, 3]), 64))
    if kind == "reorder":
        width, groups, states = rng.randint(2, 16), _log(rng, 1, 8), _log(rng, 1, 64)
        row = _log(rng, 1, min(262144, 40_000_000 // (width * groups * states)))
        return dict(kind=kind, dtype=rng.choice(["i32", "f32"]), states=states, groups=groups, width=width, row=row,
                    stride=row + rng.choice([0, 1, 4 * rng.randint(0, 64)]), in_place=rng.random() < 0.5)
    k, m = (rng.choice([_log(rng, 64, 12288), 64 * _log(rng, 1, 172)]) for _ in range(2))
    rank = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
    adapters = _log(rng, 1, min(64, max(1, 16_000_000 // (rank * (k + m)))))
    rows = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 256), _log(rng, 17, min(2048, 22_000_000 // max(k, m)))])
    return dict(kind=kind, fmt=rng.choice(["bf16", "bf16", "f32"]), adapters=adapters, rank=rank, rows=rows, m=m, k=k)


# ---- inputs ----------------------------------------------------------------------


def _gen(seed, *salt):
    s = seed & 0x7FFFFFFF
    for v in salt:
        s = (s * 1000003 + v + 1) & 0x7FFFFFFFFFFF
    return torch.Generator(device=DEV).manual_seed(s)


def _normal(g, shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _acts(g, rows, d):
    """Normal, with a log-normal scale for each channel, as a residual stream has."""
    return _normal(g, (rows, d)) * torch.exp(0.7 * _normal(g, (d,)))


def _members(c):
    """What describes a batch of `prefix`, on the host: each group's rows, its prompt's slot
    and length, each row's own tokens and their slots."""
    r = random.Random("%s %d %d %d %d" % (c["mode"], c["groups"], c["rows"], c["prefix"], c["own"]))
    n, groups = c["rows"], c["groups"]
    prefix = [c["prefix"]] + [r.randint(1, c["prefix"]) for _ in range(groups - 1)]
    if c["mode"] == "beams":
        # a beam writes its tokens into its own slot; the prompt is in the first beam's.
        # slots[b][i]: whose slot holds beam b's token i, after as many steps of choosing parents
        width = n // groups
        starts = [width * g for g in range(groups + 1)]
        picks = np.random.default_rng(r.randint(0, 2 ** 31))
        slots = np.zeros((n, c["own"]), np.int32)
        for g in range(groups):
            at = slice(starts[g], starts[g + 1])
            for i in range(c["own"]):
                if i:
                    parents = np.sort(picks.integers(0, width, width))
                    slots[at, :i] = slots[at, :i][parents]
                slots[at, i] = np.arange(starts[g], starts[g + 1])
        return dict(starts=starts, prefix=prefix, prefix_slots=starts[:-1], own=[c["own"]] * n, slots=slots, n_slots=n)
    # requests: a slot for each one's own tokens, a slot for each prompt
    cuts = sorted(r.sample(range(1, n), groups - 1))
    own_lens = [c["own"]] + [r.randint(0, c["own"]) for _ in range(n - 1)]
    return dict(starts=[0] + cuts + [n], prefix=prefix, prefix_slots=[n + g for g in range(groups)], own=own_lens,
                slots=np.arange(n, dtype=np.int32)[:, None], n_slots=n + groups)


def _max_seq(c):
    return c["prefix"] + c["own"] + 5


def _parents(c, seed):
    """Of each group's beams.  In place: those that are continued stay where they are."""
    r = np.random.default_rng(seed & 0x7FFFFFFF)
    w, out = c["width"], []
    for _ in range(c["groups"]):
        if c["in_place"]:
            live = r.permutation(w)[:max(1, w // 2)]
            p = live[r.integers(0, len(live), w)]
            p[live] = live
        else:
            p = np.sort(r.integers(0, w, w))
        out.append(p)
    return torch.from_numpy(np.stack(out).astype(np.int32)).to(DEV)


def _inputs(c, seed):
    kind = c["kind"]
    if kind == "prefix":
        b, i32 = _members(c), dict(dtype=torch.int32, device=DEV)
        row_prefix = np.repeat(b["prefix"], np.diff(b["starts"]))
        shape = (b["n_slots"], _max_seq(c), c["kv"], c["hd"])
        scale = torch.exp(0.5 * _normal(_gen(seed, 4), (c["kv"], c["hd"])))     # K's channels after RoPE differ
        return dict(k=_normal(_gen(seed, 1), shape).mul_(scale), v=_normal(_gen(seed, 2), shape),
                    q=_normal(_gen(seed, 3), (c["rows"], c["heads"], c["hd"])),
                    starts=torch.tensor(b["starts"], **i32), prefix_slots=torch.tensor(b["prefix_slots"], **i32),
                    prefix_lens=torch.tensor(b["prefix"], **i32), slots=torch.from_numpy(b["slots"]).to(DEV),
                    lens=torch.tensor(row_prefix + np.array(b["own"]), **i32))
    if kind == "select":
        g, rows = _gen(seed, 1), c["groups"] * c["width"]
        # a few likely tokens above the bulk
        z = _normal(g, (rows, c["vocab"])).mul_(2.0)
        z += 6 * (torch.rand(z.shape, generator=g, device=DEV) < 20.0 / c["vocab"])
        return dict(logits=z, scores=-30 - 3 * torch.rand((c["groups"], c["width"]), generator=g, device=DEV, dtype=torch.float64))
    if kind == "reorder":
        rows = c["groups"] * c["width"]
        if c["dtype"] == "i32":
            src = torch.randint(0, 128256, (c["states"], rows, c["stride"]), generator=_gen(seed, 1), device=DEV, dtype=torch.int32)
        else:
            src = _normal(_gen(seed, 1), (c["states"], rows, c["stride"]))
        return dict(src=src, parents=_parents(c, seed))
    dt = torch.bfloat16 if c["fmt"] == "bf16" else torch.float32
    g = _gen(seed, 1)
    # prompts lie packed, so that rows of an adapter follow each other; a batch's rows take any
    pick = torch.randint(0, c["adapters"] + 1, (c["rows"],), generator=g, device=DEV, dtype=torch.int32) - 1
    if c["rows"] > 16:
        pick = pick.sort().values
    elif c["rows"] == 1:
        pick = pick.clamp(min=0)
    return dict(a=(_normal(g, (c["adapters"], c["rank"], c["k"])) * c["k"] ** -0.5).to(dt),
                b=(_normal(g, (c["adapters"], c["m"], c["rank"])) * 0.02).to(dt),
                scales=0.5 + torch.rand((c["adapters"],), generator=g, device=DEV), pick=pick.contiguous(),
                x=_acts(_gen(seed, 2), c["rows"], c["k"]), base=_normal(_gen(seed, 3), (c["rows"], c["m"])))


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=case)
    new = dict(device=DEV)
    kind = case["kind"]
    if kind == "prefix":
        st.update(out=torch.empty_like(st["q"]), members=_members(case))
    elif kind == "select":
        n = (case["groups"], case["n_out"])
        st.update(tokens=torch.empty(n, dtype=torch.int32, **new), parents=torch.empty(n, dtype=torch.int32, **new),
                  best=torch.empty(n, dtype=torch.float64, **new))
    elif kind == "reorder":
        st["dst"] = st["src"] if case["in_place"] else torch.zeros_like(st["src"])
    else:
        st["y"] = torch.empty_like(st["base"])
    return st


# ---- the plain forms -------------------------------------------------------------


def _plain_prefix(st, c):
    kv, hd = c["kv"], c["hd"]
    group = c["heads"] // kv
    q = st["q"].view(-1, kv, group, hd) * hd ** -0.5
    b, outs = st["members"], []
    for g, (lo, hi) in enumerate(zip(b["starts"], b["starts"][1:])):
        n, lp, most = hi - lo, b["prefix"][g], max(b["own"][lo:hi])
        qg, length = q[lo:hi], st["lens"][lo:hi].long()
        k0, v0 = (st[x][b["prefix_slots"][g], :lp].transpose(0, 1).contiguous() for x in ("k", "v"))  # [kv, lp, hd]
        s0 = torch.matmul(qg.transpose(0, 1).reshape(kv, n * group, hd), k0.transpose(1, 2).contiguous())
        s0 = s0.view(kv, n, group, lp).transpose(0, 1)
        at = lp + torch.arange(most, device=DEV)
        slots = st["slots"][lo:hi].long().expand(n, most) if st["slots"].shape[1] == 1 else st["slots"][lo:hi, :most].long()
        k1, v1 = (st[x][slots, at].transpose(1, 2).contiguous() for x in ("k", "v"))  # [n, kv, most, hd]
        s1 = torch.matmul(qg, k1.transpose(2, 3).contiguous())
        pos = torch.arange(lp + most, device=DEV)
        seen = pos < length[:, None]
        if c["window"]:
            seen &= pos >= length[:, None] - c["window"]
        s = torch.cat([s0, s1], -1).masked_fill_(~seen[:, None, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p /= p.sum(-1, keepdim=True)
        o = torch.matmul(p[..., :lp].transpose(0, 1).reshape(kv, n * group, lp), v0).view(kv, n, group, hd).transpose(0, 1)
        outs.append(o + torch.matmul(p[..., lp:], v1))
    return torch.cat(outs).reshape(-1, c["heads"], hd)


def _plain_select(st, c):
    z = st["logits"].double()
    m = z.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(-1, keepdim=True))
    # candidates lie close: 64 bits
    cand = (st["scores"].view(-1, 1) + (z - lse)).view(c["groups"], -1)
    at, best = [], []
    for _ in range(c["n_out"]):
        i = cand.argmax(-1, keepdim=True)                # the first of equal ones
        at.append(i)
        best.append(cand.gather(1, i))
        cand.scatter_(1, i, -math.inf)
    at, best = torch.cat(at, 1), torch.cat(best, 1)
    return dict(tokens=(at % c["vocab"]).int(), parents=(at // c["vocab"]).int(), scores=best)


def _plain_reorder(st, c):
    base = torch.arange(c["groups"], device=DEV)[:, None] * c["width"]
    rows = (st["parents"].long() + base).view(-1)
    st["dst"][:, :, :c["row"]] = st["src"][:, rows, :c["row"]]
    return st["dst"][:, :, :c["row"]]


def _plain_lora(st, c):
    # every adapter's product, of which each row keeps its own's
    a, b = st["a"].float().flatten(0, 1), st["b"].float()
    v = torch.matmul(st["x"], a.t().contiguous()).view(-1, c["adapters"], c["rank"])
    pick = st["pick"][:, None] == torch.arange(c["adapters"], device=DEV)
    v = (v * torch.where(pick, st["scales"], 0.0)[..., None]).flatten(1)
    return st["base"] + torch.matmul(v, b.transpose(1, 2).reshape(-1, c["m"]).contiguous())


PLAIN = {"prefix": _plain_prefix, "select": _plain_select, "reorder": _plain_reorder, "lora": _plain_lora}


# ---- the framework's calls -------------------------------------------------------


def _call(st, c):
    """The entry point with the arguments that a program holds on to: device
    pointers, sizes, and the descriptions of its cache, batch or adapters."""
    from atlas_amd import _lib
    lib, p = _lib.load(), {n: t.data_ptr() for n, t in st.items() if isinstance(t, torch.Tensor)}
    if c["kind"] == "prefix":
        cache = _lib.SlotCacheC(p["k"], p["v"], st["k"].shape[0], st["k"].shape[1], c["kv"], c["hd"])
        # one slot for all of a row's own tokens: a table of one column
        stride = 0 if c["mode"] == "requests" else c["own"]
        batch = _lib.PrefixBatchC(p["starts"], p["prefix_slots"], p["prefix_lens"], p["lens"], p["slots"], stride,
                                  c["groups"], c["rows"], c["prefix"], c["own"])
        st["held"] = cache, batch
        wide = c["heads"] * c["hd"]
        return lib.atlas_prefix_attention_f32, (C.byref(cache), C.byref(batch), p["q"], wide, c["heads"], c["hd"] ** -0.5,
                                                c["window"], p["out"], wide)
    if c["kind"] == "select":
        return lib.atlas_beam_select_f32, (p["logits"], c["vocab"], c["vocab"], p["scores"], c["groups"], c["width"],
                                           c["n_out"], p["tokens"], p["parents"], p["best"])
    if c["kind"] == "reorder":
        each = 4 * c["groups"] * c["width"] * c["stride"]
        dst, src = ((C.c_void_p * c["states"])(*(p[x] + each * i for i in range(c["states"]))) for x in ("dst", "src"))
        return lib.atlas_beam_reorder, (dst, src, c["states"], 4 * c["row"], 4 * c["stride"], p["parents"], c["groups"],
                                        c["width"])
    lora = _lib.LoraC(1 if c["fmt"] == "bf16" else 0, p["a"], p["b"], p["scales"], c["adapters"], c["rank"], c["m"], c["k"])
    st["held"] = lora
    return lib.atlas_lora_add_f32, (C.byref(lora), p["pick"], p["x"], c["k"], p["base"], c["m"], p["y"], c["m"], c["rows"])


def _run_own(st, c):
    call = st.get("call")
    if call is None:
        from atlas_amd import _lib
        call = st["call"] = _call(st, c) + (_lib.check,)
    fn, args, check = call
    check(fn(*args))
    if c["kind"] == "prefix":
        return st["out"]
    if c["kind"] == "select":
        return dict(tokens=st["tokens"], parents=st["parents"], scores=st["best"])
    return st["dst"][:, :, :c["row"]] if c["kind"] == "reorder" else st["y"]


def run(state):
    c = state["case"]
    return _run_own(state, c) if own else PLAIN[c["kind"]](state, c)


# ---- 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    c, st = case, _inputs(case, seed)
    if c["kind"] == "prefix":
        b, group, outs = _members(c), c["heads"] // c["kv"], []
        which = np.repeat(np.arange(c["groups"]), np.diff(b["starts"]))
        for r, g in enumerate(which):
            lp, n = b["prefix"][g], b["prefix"][g] + b["own"][r]
            mine = b["slots"][r] if b["slots"].shape[1] > 1 or c["mode"] == "beams" else np.repeat(b["slots"][r], b["own"][r])
            slot = torch.from_numpy(np.concatenate([np.full(lp, b["prefix_slots"][g]), mine[:b["own"][r]]]).astype(np.int64)).to(DEV)
            at = torch.arange(n, device=DEV)
            if c["window"]:
                slot, at = slot[-c["window"]:], at[-c["window"]:]
            k, v = (st[x][slot, at].double().transpose(0, 1).contiguous() for x in ("k", "v"))
            q = st["q"][r].double().view(c["kv"], group, c["hd"])
            s = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(c["hd"])
            outs.append(torch.matmul(torch.softmax(s, -1), v).view(c["heads"], c["hd"]))
        return torch.stack(outs)
    if c["kind"] == "select":
        logp = torch.log_softmax(st["logits"].double(), -1).view(c["groups"], c["width"], c["vocab"])
        all_ = (st["scores"][..., None] + logp).flatten(1)
        best, at = torch.sort(all_, dim=-1, descending=True, stable=True)
        best, at = best[:, :c["n_out"]], at[:, :c["n_out"]]
        return dict(tokens=(at % c["vocab"]).int(), parents=(at // c["vocab"]).int(), scores=best.contiguous())
    if c["kind"] == "reorder":
        out, p = torch.empty_like(st["src"][:, :, :c["row"]]), st["parents"].cpu().tolist()
        for g in range(c["groups"]):
            for i, parent in enumerate(p[g]):
                out[:, g * c["width"] + i] = st["src"][:, g * c["width"] + parent, :c["row"]]
        return out
    y = st["base"].double()
    for i in range(c["adapters"]):
        rows = (st["pick"] == i).nonzero().view(-1)
        if len(rows):
            v = torch.matmul(st["x"][rows].double(), st["a"][i].double().t().contiguous())
            y[rows] += st["scales"][i].double() * torch.matmul(v, st["b"][i].double().t().contiguous())
    return y


# ---- what a pass cannot do without -----------------------------------------------


def work(case):
    c = case
    if c["kind"] == "prefix":
        b, cells, seen, at = _members(c), 0, 0, 0
        for g, (lo, hi) in enumerate(zip(b["starts"], b["starts"][1:])):
            lp, first, used = b["prefix"][g], b["prefix"][g], set()
            for r in range(lo, hi):
                n = lp + b["own"][r]
                start = max(0, n - c["window"]) if c["window"] else 0
                seen += n - start
                first = min(first, start)
                for i in range(max(start - lp, 0), b["own"][r]):
                    used.add((int(b["slots"][r][i if c["mode"] == "beams" else 0]), i))
            cells += lp - first + len(used)
        return {"bytes": 8 * cells * c["kv"] * c["hd"] + 8 * c["rows"] * c["heads"] * c["hd"],
                "flops": 4 * seen * c["heads"] * c["hd"]}
    if c["kind"] == "select":
        n = c["groups"] * c["width"] * c["vocab"]
        return {"bytes": 4 * n + 16 * c["groups"] * c["n_out"], "flops": 4 * n}
    if c["kind"] == "reorder":
        n, w = 4 * c["states"] * c["row"] * c["groups"], c["width"]
        # in place half of the beams are read and the others written; else every one is written, from about two thirds of them
        return {"bytes": n * w if c["in_place"] else n * (w + (2 * w + 2) // 3), "flops": 0}
    size = 2 if c["fmt"] == "bf16" else 4
    used = min(c["adapters"], c["rows"])
    return {"bytes": size * used * c["rank"] * (c["k"] + c["m"]) + 4 * c["rows"] * (c["k"] + 2 * c["m"]),
            "flops": 2 * c["rows"] * c["rank"] * (c["k"] + c["m"])}

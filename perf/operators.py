"""The 4-bit operators as cases that can be timed: MXFP4 matrices and the 4-bit KV cache.

A case is one pass of one of four kinds.  With `own` false a pass computes the
operator in its plain form, from elementary torch operations in 32 bits; with
`own` true it makes the calls of include/atlas_kernels.h that a program makes.

  quant  rows are encoded as MXFP4 and read back: a weight matrix when it is
         loaded, or the activations of a step before their product.
  gemm   y[n, m] = x[n, k] . w[m, k] of two MXFP4 matrices.  One row is decode,
         2..16 rows a ragged batch's step, more a prompt.
  write  the new tokens' K and V rows of a batch of sequences are encoded into
         the pages of a 4-bit KV cache and read back.
  attn   attention of a batch's query rows over that cache: one row for each
         sequence is decode, more are (chunks of) prompts, causal.

MXFP4 is a block of 32 elements of E2M1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign,
the first element of a byte in its low nibble) and a scale byte b of value
2^(b - 127).  Sequences' lengths follow from the case, values from the seed.
"""
import ctypes as C
import math
import random

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # the activations of one decode step of a 135M-sized model: the smallest call, all latency
        dict(name="quant_135m_row1", kind="quant", src="f32", rows=1, cols=576),
        # loading: one gate or up matrix of a bf16 checkpoint
        dict(name="quant_7b_weights", kind="quant", src="bf16", rows=11008, cols=4096),
        # W_o of the 135M-sized model, one decode row: launch and latency
        dict(name="gemm_135m_row1", kind="gemm", m=576, n=1, k=576),
        # gate and up of a 7B model, ordinary batch-1 decode: the weight stream
        dict(name="gemm_7b_row1", kind="gemm", m=22016, n=1, k=4096),
        # W_down of a 1B model, a ragged batch's step
        dict(name="gemm_1b_rows13", kind="gemm", m=2048, n=13, k=8192),
        # gate or up of a 7B model over a long prompt: the matrix units
        dict(name="gemm_7b_rows2047", kind="gemm", m=11008, n=2047, k=4096),
        # 24 sequences' new tokens of a grouped-query 1B model
        dict(name="write_1b_batch24", kind="write", seqs=24, rows=1, ctx=8191, kv=8, hd=64, page=64),
        # a 7B model's prompt
        dict(name="write_7b_prompt2047", kind="write", seqs=1, rows=2047, ctx=2047, kv=32, hd=128, page=64),
        # decode of the 135M-sized model early in a conversation: latency
        dict(name="attn_135m_ctx19", kind="attn", seqs=1, rows=1, ctx=19, heads=9, kv=3, hd=64, page=32, window=0),
        # one long document on a 7B model: the cache stream of a single token
        dict(name="attn_7b_ctx16001", kind="attn", seqs=1, rows=1, ctx=16001, heads=32, kv=32, hd=128, page=64,
             window=0),
        # 24 conversations of different lengths decoded together
        dict(name="attn_1b_batch24", kind="attn", seqs=24, rows=1, ctx=8191, heads=32, kv=8, hd=64, page=64, window=0),
        # three prompts of a 7B model packed together, the longest continuing a cached beginning
        dict(name="attn_7b_prompts3", kind="attn", seqs=3, rows=1023, ctx=1500, heads=32, kv=32, hd=128, page=64,
             window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant"] * 3 + ["gemm"] * 6 + ["write"] * 3 + ["attn"] * 8)
    if kind == "quant":
        cols = rng.choice([_log(rng, 32, 12288), 32 * _log(rng, 1, 384)])
        return dict(kind=kind, src=rng.choice(["f32", "bf16"]), rows=_log(rng, 1, min(32768, 45_000_000 // cols)), cols=cols)
    if kind == "gemm":
        k = rng.choice([_log(rng, 64, 12288), 32 * _log(rng, 4, 384), 128 * _log(rng, 2, 96)])
        m = _log(rng, 64, 22016)
        top = min(4096, 90_000_000_000 // (m * k))
        n = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 256), _log(rng, 17, top), _log(rng, 17, top)])
        return dict(kind=kind, m=m, n=n, k=k)
    hd = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8, 16, 32])
    page = rng.choice([32, 64, 64, 128, 256])
    prompt = rng.random() < 0.35
    if kind == "write":
        rows = _log(rng, 2, min(2048, 8_300_000 // (kv * hd))) if prompt else 1
        seqs = _log(rng, 1, min(64, 8_300_000 // (rows * kv * hd)))
        return dict(kind=kind, seqs=seqs, rows=rows, ctx=rows + _log(rng, 1, 4096) - 1, kv=kv, hd=hd, page=page)
    heads = kv * rng.choice([g for g in (1, 1, 2, 3, 4, 5, 7, 8, 16) if kv * g <= 64])
    rows = _log(rng, 2, 1024) if prompt else 1
    # 45 million cache elements; prompts: scores of all heads and rows as well
    seqs = _log(rng, 1, 8 if prompt else 64)
    ctx = rows + _log(rng, 1, max(1, min(2048 if prompt else 32768, 45_000_000 // (seqs * kv * hd)))) - 1
    if prompt:
        ctx = max(rows, min(ctx, 90_000_000 // (seqs * heads * rows)))
    return dict(kind=kind, seqs=seqs, rows=rows, ctx=ctx, heads=heads, kv=kv, hd=hd, page=page,
                window=rng.choice([0, 0, _log(rng, 16, 4096)]))


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


def _lens(c):
    """(rows, length) of each sequence: the first as the case says, the others spread below it."""
    r = random.Random("%d %d %d" % (c["seqs"], c["rows"], c["ctx"]))
    got = [(c["rows"], c["ctx"])]
    while len(got) < c["seqs"]:
        rows = r.randint(1, c["rows"])
        got.append((rows, r.randint(rows, c["ctx"])))
    return got


def _batch(c, seed):
    """The device arrays that describe a batch, and the pages' order."""
    lens, page = _lens(c), c["page"]
    width = -(-c["ctx"] // page)
    need = [-(-n // page) for _, n in lens]
    n_pages = sum(need) + 2
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed & 0x7FFFFFFF))
    table = torch.full((c["seqs"], width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n].int()
        at += n
    starts = [0]
    for rows, _ in lens:
        starts.append(starts[-1] + rows)
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(table=table.to(DEV), starts=torch.tensor(starts, **i32), lens=torch.tensor([n for _, n in lens], **i32),
                n_rows=starts[-1], n_pages=n_pages, width=width)


def _halves(codes):
    return codes[..., ::2] | codes[..., 1::2] << 4


def _keys(c, g, n):
    """K rows as they are after RoPE: channels of different size."""
    return _normal(g, (n, c["kv"], c["hd"])) * torch.exp(0.5 * _normal(g, (c["kv"], c["hd"])))


def _page_bytes(c, k, v):
    """Whole pages of K and V values [pages * page, kv, hd] as the cache holds them:
    for each page and KV head K's bytes [page][hd/2], its scales [page/8][hd/32][8],
    V's bytes [page/8][16][8][hd/32] (a group of hd/16 elements of eight tokens side
    by side) and its scales [page/8][hd/32][8]."""
    page, kv, hd = c["page"], c["kv"], c["hd"]
    out = []
    for x, apart in ((k, False), (v, True)):
        codes, scales = _encode(x)
        data = _halves(codes).view(-1, page // 8, 8, kv, 16, hd // 32)
        data = data.permute(0, 3, 1, 4, 2, 5) if apart else data.permute(0, 3, 1, 2, 4, 5)
        scales = scales.view(-1, page // 8, 8, kv, hd // 32).permute(0, 3, 1, 4, 2)
        out += [data.reshape(-1, kv, page * hd // 2), scales.reshape(-1, kv, page * hd // 32)]
    return torch.cat(out, -1).contiguous()


def _inputs(c, seed):
    kind = c["kind"]
    if kind == "quant":
        x = _acts(_gen(seed, 1), c["rows"], c["cols"])
        return dict(x=x.bfloat16() if c["src"] == "bf16" else x)
    if kind == "gemm":
        w, x = _normal(_gen(seed, 1), (c["m"], c["k"])).mul_(0.02), _acts(_gen(seed, 2), c["n"], c["k"])
        st = {}
        for name, v in (("w", w), ("x", x)):
            codes, scales = _encode(torch.nn.functional.pad(v, (0, -c["k"] % 32)))
            st[name], st[name + "_scales"] = _halves(codes).contiguous(), scales.contiguous()
        return st
    st = _batch(c, seed)
    if kind == "write":
        g = _gen(seed, 1)
        st["k"], st["v"] = _keys(c, g, st["n_rows"]), _normal(g, (st["n_rows"], c["kv"], c["hd"]))
        st["cache"] = torch.zeros((st["n_pages"], c["kv"], 17 * c["page"] * c["hd"] // 16), dtype=torch.uint8, device=DEV)
        return st
    n = st["n_pages"] * c["page"]
    st["cache"] = _page_bytes(c, _keys(c, _gen(seed, 1), n), _normal(_gen(seed, 2), (n, c["kv"], c["hd"])))
    st["q"] = _normal(_gen(seed, 3), (st["n_rows"], c["heads"], c["hd"]))
    return st


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=case)
    new = dict(device=DEV, dtype=torch.float32)
    kind = case["kind"]
    if kind == "quant":
        blocks = -(-case["cols"] // 32)
        st["data"] = torch.empty((case["rows"], 16 * blocks), dtype=torch.uint8, device=DEV)
        st["scales"] = torch.empty((case["rows"], blocks), dtype=torch.uint8, device=DEV)
        st["out"] = torch.empty((case["rows"], case["cols"]), **new)
    elif kind == "gemm":
        st["y"] = torch.empty((case["n"], case["m"]), **new)
    elif kind == "write":
        st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    else:
        st["out"] = torch.empty_like(st["q"])
    return st


# ---- the plain forms -------------------------------------------------------------


def _encode(v):
    """MXFP4 of the last dimension: element codes, and a scale byte for each 32."""
    b = v.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    byte = ((amax.view(torch.int32) >> 23) - 2).clamp_(min=0)
    byte = torch.where(amax == 0, 127, byte)
    x = b * ((254 - byte) << 23).view(torch.float32)[..., None]
    a = x.abs()
    code = (a > 0.25).byte()
    for edge, closed in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= edge) if closed else (a > edge)
    return (code | (x < 0).byte() << 3).flatten(-2), byte.byte()


def _table(dtype=torch.float32):
    t = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV, dtype=dtype)
    return torch.cat([t, -t])


def _values(codes, scales):
    x = _table()[codes.int()].unflatten(-1, (-1, 32))
    return (x * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _codes(data):
    return torch.stack([data & 15, data >> 4], -1).flatten(-2)


def _places(st, c):
    """Page and offset of each row's token."""
    row = torch.arange(st["n_rows"], device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(st["starts"], row, right=True) - 1
    pos = st["lens"][seq] - st["starts"][seq + 1] + row
    return st["table"][seq, pos // c["page"]].long(), (pos % c["page"]).long()


def _split(c, cache):
    """The four parts of a cache's pages, tokens first: bytes [pages, page, kv, hd/2], scales [pages, page, kv, hd/32]."""
    page, kv, hd = c["page"], c["kv"], c["hd"]
    d, s = page * hd // 2, page * hd // 32
    kd, ks, vd, vs = cache.split([d, s, d, s], -1)
    kd = kd.unflatten(-1, (page, hd // 2)).transpose(1, 2)
    vd = vd.unflatten(-1, (page // 8, 16, 8, hd // 32)).permute(0, 2, 4, 1, 3, 5)
    ks, vs = (x.unflatten(-1, (page // 8, hd // 32, 8)).permute(0, 2, 4, 1, 3) for x in (ks, vs))
    return kd, ks, vd, vs


def _plain_quant(st, c):
    x = torch.nn.functional.pad(st["x"], (0, -c["cols"] % 32))
    return _values(*_encode(x))[:, :c["cols"]]


def _plain_gemm(st, c):
    w, x = (_values(_codes(st[n]), st[n + "_scales"]) for n in ("w", "x"))
    return torch.matmul(x, w.t())


def _plain_write(st, c):
    page, at = _places(st, c)
    kd, ks, vd, vs = _split(c, st["cache"])
    out = []
    for x, data, scales in ((st["k"], kd, ks), (st["v"], vd, vs)):
        codes, byte = _encode(x)
        piece = _halves(codes)
        if data is vd:
            data[page, at // 8, at % 8] = piece.unflatten(-1, (16, -1))
            back = data[page, at // 8, at % 8].flatten(-2)
        else:
            data[page, at] = piece
            back = data[page, at]
        scales[page, at // 8, at % 8] = byte
        out.append(_values(_codes(back), scales[page, at // 8, at % 8]))
    return dict(k=out[0], v=out[1])


def _plain_attn(st, c):
    page, kv, hd, heads = c["page"], c["kv"], c["hd"], c["heads"]
    group, most, length = heads // kv, c["rows"], st["width"] * c["page"]
    pages = st["table"].clamp(min=0).long()
    kd, ks, vd, vs = _split(c, st["cache"][pages.flatten()])
    k = _values(_codes(kd), ks.flatten(1, 2)).view(c["seqs"], length, kv, hd)
    v = _values(_codes(vd.flatten(4).flatten(1, 2)), vs.flatten(1, 2)).view(c["seqs"], length, kv, hd)
    # the sequences' rows, padded to the longest
    rows = (st["starts"][1:] - st["starts"][:-1]).long()
    local = torch.arange(most, device=DEV)
    live = local < rows[:, None]
    at = torch.where(live, st["starts"][:-1].long()[:, None] + local, 0)
    q = st["q"][at].view(c["seqs"], most, kv, group, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) * hd ** -0.5
    pos = (st["lens"].long() - rows)[:, None] + local
    key = torch.arange(length, device=DEV)
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    s = s.view(c["seqs"], kv, group, most, length).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v.transpose(1, 2)).view(c["seqs"], kv, group, most, hd)
    return o.permute(0, 3, 1, 2, 4)[live].reshape(st["n_rows"], heads, hd)


PLAIN = {"quant": _plain_quant, "gemm": _plain_gemm, "write": _plain_write, "attn": _plain_attn}


# ---- the framework's calls -------------------------------------------------------


def _calls(st, c):
    """The entry points with the arguments that a program holds on to: device
    pointers, sizes, and the descriptions of its cache and batch."""
    from atlas_amd import _lib
    lib, p = _lib.load(), {n: t.data_ptr() for n, t in st.items() if isinstance(t, torch.Tensor)}
    if c["kind"] == "quant":
        rows, cols = c["rows"], c["cols"]
        return [(lib.atlas_quantize_mxfp4_dev, (p["x"], int(c["src"] == "bf16"), rows, cols, cols, p["data"], p["scales"])),
                (lib.atlas_dequantize_mxfp4_dev, (p["data"], p["scales"], rows, cols, p["out"], cols))]
    if c["kind"] == "gemm":
        return [(lib.atlas_gemm_mxfp4_f32, (p["w"], p["w_scales"], p["x"], p["x_scales"], p["y"], c["m"], c["n"], c["k"], c["m"]))]
    cache = _lib.Kv4CacheC(p["cache"], st["n_pages"], c["page"], c["kv"], c["hd"])
    # one row for each sequence needs no row starts
    batch = _lib.Kv4BatchC(p["starts"] if c["rows"] > 1 else None, p["lens"], p["table"], st["width"], c["seqs"],
                           st["n_rows"], c["ctx"])
    st["held"] = cache, batch
    args = C.byref(cache), C.byref(batch)
    wide = c["kv"] * c["hd"]
    if c["kind"] == "write":
        return [(lib.atlas_kv4_write_f32, args + (p["k"], p["v"], wide)),
                (lib.atlas_kv4_read_f32, args + (p["k_out"], p["v_out"], wide))]
    wide = c["heads"] * c["hd"]
    return [(lib.atlas_kv4_attention_f32, args + (p["q"], wide, c["heads"], c["hd"] ** -0.5, c["window"], p["out"], wide))]


def _run_own(st, c):
    calls = st.get("calls")
    if calls is None:
        from atlas_amd import _lib
        calls = st["calls"] = _calls(st, c)
        st["check"] = _lib.check
    check = st["check"]
    for fn, args in calls:
        check(fn(*args))
    if c["kind"] == "write":
        return dict(k=st["k_out"], v=st["v_out"])
    return st["y"] if c["kind"] == "gemm" else st["out"]


def run(state):
    c = state["case"]
    return _run_own(state, c) if own else PLAIN[c["kind"]](state, c)


# ---- 64 bits ---------------------------------------------------------------------


def _nearest(v):
    """The values that MXFP4 gives v, by distance to the eight magnitudes; v in whole blocks of 32."""
    b = v.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120))) - 2)
    x = b.abs() / scale
    mags = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    got = torch.zeros_like(x)
    for i in range(1, 8):
        mid = (mags[i - 1] + mags[i]) / 2
        # halfway goes to the magnitude of even place
        got = torch.where((x > mid) | ((x == mid) & (i % 2 == 0)), mags[i], got)
    return (got * scale * torch.sign(b)).flatten(-2)


def _read64(data, scales):
    lo, hi = (data % 16).long(), (data // 16).long()
    x = _table(torch.float64)[torch.stack([lo, hi], -1).flatten(-2)]
    return x * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _tokens64(c, st, s, n):
    """K and V [n, kv, hd] of a sequence's first n tokens."""
    page, kv, hd = c["page"], c["kv"], c["hd"]
    raw = st["cache"][st["table"][s, :-(-n // page)].long()]
    d, sc = page * hd // 2, page * hd // 32
    out = []
    for at, by_token in ((0, True), (d + sc, False)):
        data, scales = raw[..., at:at + d], raw[..., at + d:at + d + sc]
        if by_token:
            data = data.reshape(-1, kv, page, hd // 2)
        else:
            data = data.reshape(-1, kv, page // 8, 16, 8, hd // 32).transpose(3, 4).reshape(-1, kv, page, hd // 2)
        scales = scales.reshape(-1, kv, page // 8, hd // 32, 8).transpose(3, 4).reshape(-1, kv, page, hd // 32)
        out.append(_read64(data, scales).transpose(1, 2).reshape(-1, kv, hd)[:n])
    return out


def exact(case, seed):
    c, st = case, _inputs(case, seed)
    if c["kind"] == "quant":
        return _nearest(torch.nn.functional.pad(st["x"].double(), (0, -c["cols"] % 32)))[:, :c["cols"]]
    if c["kind"] == "gemm":
        return torch.matmul(_read64(st["x"], st["x_scales"]), _read64(st["w"], st["w_scales"]).t().contiguous())
    if c["kind"] == "write":
        return dict(k=_nearest(st["k"]), v=_nearest(st["v"]))
    group, outs, at = c["heads"] // c["kv"], [], 0
    for s, (rows, n) in enumerate(_lens(c)):
        k, v = _tokens64(c, st, s, n)
        q = st["q"][at:at + rows].double()
        at += rows
        pos, key = torch.arange(n - rows, n, device=DEV)[:, None], torch.arange(n, device=DEV)
        hidden = key > pos
        if c["window"]:
            hidden = hidden | (key <= pos - c["window"])
        heads = []
        for h in range(c["heads"]):
            x = torch.matmul(q[:, h], k[:, h // group].t().contiguous()) / math.sqrt(c["hd"])
            heads.append(torch.matmul(torch.softmax(x.masked_fill(hidden, -math.inf), -1), v[:, h // group].contiguous()))
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)


# ---- what a pass cannot do without -----------------------------------------------


def work(case):
    c = case
    if c["kind"] == "quant":
        n, blocks = c["rows"] * c["cols"], c["rows"] * -(-c["cols"] // 32)
        # the source, the encoded matrix, its values
        return {"bytes": n * (2 if c["src"] == "bf16" else 4) + 17 * blocks + 4 * n, "flops": n}
    if c["kind"] == "gemm":
        blocks = -(-c["k"] // 32)
        return {"bytes": 17 * blocks * (c["m"] + c["n"]) + 4 * c["m"] * c["n"], "flops": 2 * c["m"] * c["n"] * c["k"]}
    lens, wide = _lens(c), c["kv"] * c["hd"]
    if c["kind"] == "write":
        n = sum(rows for rows, _ in lens) * wide
        # both inputs, both parts of the cache, both outputs
        return {"bytes": 2 * (4 * n + 17 * n // 32 + 4 * n), "flops": 2 * n}
    w = c["window"] or c["ctx"] + 1
    seen = sum(min(p + 1, w) for rows, n in lens for p in range(n - rows, n))
    cached = sum(min(n, w + rows - 1) for rows, n in lens)
    n_rows = sum(rows for rows, _ in lens)
    return {"bytes": 17 * cached * wide // 16 + 8 * n_rows * c["heads"] * c["hd"], "flops": 4 * seen * c["heads"] * c["hd"]}

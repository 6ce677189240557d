"""Measured cases of the beam-search operators: attention over a prompt that several sequences share, choice of the
next beams, reordering of their paged caches, and the walk back through the chosen beams.

`run` computes an operator in its plain form (elementary torch operations) or, where `own` is set, through the
library's entry points.  The plain form works in 32 bits, or in 64 where candidates are ranked.
"""
import torch

own = False

QUANT_ID = {"none": 0, "int8": 1, "q4_0": 2}


def listed():
    return [
        # a short chat prompt, four beams, a few tokens in: nothing but launch latency
        dict(name="attn-4beams-p100", op="attn", groups=1, seqs=4, heads=16, kv_heads=8, dim=128, prefix=100, suffix=5, page=64,
             quant="none", ragged=False),
        # cross-attention of a speech decoder: the 1500 encoder frames of an utterance serve its five beams, no suffix
        dict(name="attn-cross-8x5-p1500", op="attn", groups=8, seqs=5, heads=20, kv_heads=20, dim=64, prefix=1500, suffix=0, page=64,
             quant="none", ragged=False),
        # a long system prompt under 64 conversations of different lengths
        dict(name="attn-64seqs-p32768", op="attn", groups=1, seqs=64, heads=32, kv_heads=8, dim=128, prefix=32768, suffix=256, page=64,
             quant="none", ragged=True),
        # four requests of eight beams over Int8 pages
        dict(name="attn-4x8-p4099-int8", op="attn", groups=4, seqs=8, heads=32, kv_heads=8, dim=128, prefix=4099, suffix=131, page=64,
             quant="int8", ragged=False),
        # two documents with sixteen continuations each over Q4_0 pages of 16 tokens
        dict(name="attn-2x16-p9001-q4_0", op="attn", groups=2, seqs=16, heads=16, kv_heads=8, dim=128, prefix=9001, suffix=77, page=16,
             quant="q4_0", ragged=True),
        # first step of one utterance (one live beam), odd vocabulary: rows that start off a 16-byte boundary
        dict(name="select-1x4-v51865-bf16", op="select", groups=1, beams=4, vocab=51865, dtype="bf16", n_out=4, first=True),
        # a few chat requests, twice as many candidates as beams
        dict(name="select-4x5-v151936-fp32", op="select", groups=4, beams=5, vocab=151936, dtype="fp32", n_out=10, first=False),
        # a full serving batch
        dict(name="select-32x8-v151936-bf16", op="select", groups=32, beams=8, vocab=151936, dtype="bf16", n_out=8, first=False),
        # one request on a small model, Int8 pages
        dict(name="reorder-1x4-l4-int8", op="reorder", groups=1, beams=4, layers=4, kv_heads=8, dim=128, page=16, pages=4, length=21,
             quant="int8"),
        # sixteen requests of eight beams through all the layers of a large decoder
        dict(name="reorder-16x8-l36-bf16", op="reorder", groups=16, beams=8, layers=36, kv_heads=8, dim=128, page=64, pages=3,
             length=173, quant="none"),
        # an utterance's transcript
        dict(name="trace-1x5-s37", op="trace", groups=1, beams=5, steps=37, picks=5),
        # long answers of a full batch
        dict(name="trace-32x8-s4096", op="trace", groups=32, beams=8, steps=4096, picks=8),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["attn", "attn", "select", "reorder", "trace"])
    if op == "attn":
        heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 8, 128), (20, 20, 64), (12, 4, 64), (8, 2, 128), (16, 1, 64)])
        groups, seqs = _log(rng, 1, 8), _log(rng, 1, 64)
        prefix = min(_log(rng, 1, 32768), 32768 // groups)
        while groups * seqs * heads * prefix > 64 * 32 * 32768 or groups * seqs > 128:
            seqs = max(1, seqs // 2)
        suffix = min(rng.choice([0, _log(rng, 1, 600)]), 8192 // (groups * seqs))
        return dict(op=op, groups=groups, seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, prefix=prefix, suffix=suffix,
                    page=rng.choice([5, 16, 64, 128]), quant=rng.choice(["none", "none", "int8", "q4_0"]), ragged=rng.random() < 0.5)
    if op == "select":
        groups, beams = _log(rng, 1, 32), rng.randint(1, 16)
        vocab = _log(rng, 60, 151936)
        while groups * beams * vocab > 32 * 8 * 151936:
            groups = max(1, groups // 2)
        return dict(op=op, groups=groups, beams=beams, vocab=vocab, dtype=rng.choice(["bf16", "fp32"]),
                    n_out=rng.choice([beams, 2 * beams]), first=rng.random() < 0.2)
    if op == "reorder":
        page = rng.choice([4, 16, 64])
        groups, beams, layers = _log(rng, 1, 16), rng.randint(2, 8), _log(rng, 1, 36)
        length = rng.randint(1, 4 * page)
        kv_heads, dim = rng.choice([(2, 64), (2, 128), (8, 64), (20, 64)] if layers > 18 else [(2, 64), (8, 64), (8, 128), (20, 64)])
        if layers > 18 and kv_heads == 20:
            layers = layers // 2
        return dict(op=op, groups=groups, beams=beams, layers=layers, kv_heads=kv_heads, dim=dim, page=page, pages=5, length=length,
                    quant=rng.choice(["none", "int8", "q4_0"]))
    beams = rng.randint(1, 16)
    return dict(op=op, groups=_log(rng, 1, 32), beams=beams, steps=_log(rng, 1, 4096), picks=rng.randint(1, min(beams, 8)))


# ---- inputs ------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lens(n, most, ragged):
    """n lengths up to `most`, the first of them `most`; ragged: down to about half of it."""
    return [most - (i * most) // (2 * n) if ragged else most for i in range(n)]


def _pages(g, rows, tokens, c, n_layers=1):
    """The pool, scales and page table of `rows` sequences of up to `tokens` tokens, pages in random order."""
    page, kvh, d, quant = c["page"], c["kv_heads"], c["dim"], c["quant"]
    per_row = max(1, -(-tokens // page)) if "pages" not in c else c["pages"]
    n = rows * per_row
    elems = page * kvh * d
    if quant == "none":
        vals = [torch.randn(n_layers, n * elems, device="cuda", generator=g).to(torch.bfloat16).view(torch.uint8) for _ in "kv"]
        scales = [None, None]
    elif quant == "int8":
        vals = [torch.randint(1, 256, (n_layers, n * elems), device="cuda", generator=g, dtype=torch.uint8) for _ in "kv"]
        scales = [torch.rand(n_layers, n, device="cuda", generator=g) * 0.01 + 0.01 for _ in "kv"]
    else:
        vals = []
        for _ in "kv":
            code = torch.randint(1, 16, (2, n_layers, n * elems // 2), device="cuda", generator=g, dtype=torch.uint8)
            vals.append(code[0] | (code[1] << 4))
        scales = [torch.rand(n_layers, n * elems // 32, device="cuda", generator=g) * 0.2 + 0.15 for _ in "kv"]
    table = torch.randperm(n, device="cuda", generator=g).to(torch.int32).reshape(rows, per_row)
    return dict(k=vals[0], v=vals[1], ks=scales[0], vs=scales[1], table=table)


def _parents(g, shape, beams):
    """Parents as a search chooses them: the better beams have more children."""
    return (torch.rand(shape, device="cuda", generator=g) ** 1.5 * beams).to(torch.int32).clamp_(max=beams - 1)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    if case["op"] == "attn":
        batch = case["groups"] * case["seqs"]
        s["q"] = (torch.randn(batch, case["heads"], case["dim"], device="cuda", generator=g) * 2).to(torch.bfloat16)
        s["prefix"] = _pages(g, case["groups"], case["prefix"], case)
        s["prefix"]["lens"] = torch.tensor(_lens(case["groups"], case["prefix"], case["ragged"]), dtype=torch.int32, device="cuda")
        if case["suffix"]:
            s["suffix"] = _pages(g, batch, case["suffix"], case)
            s["suffix"]["lens"] = torch.tensor(_lens(batch, case["suffix"], case["ragged"]), dtype=torch.int32, device="cuda")
    elif case["op"] == "select":
        n, k, v = case["groups"], case["beams"], case["vocab"]
        logits = torch.randn(n * k, v, device="cuda", generator=g) * 3
        s["logits"] = logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        s["scores"] = -torch.rand(n, k, device="cuda", generator=g) * 6 - 4
        s["finished"] = (torch.rand(n, k, device="cuda", generator=g) < 0.15).to(torch.uint8)
        s["eos"] = v // 3
        if case["first"]:  # one live beam for each request
            s["scores"] = torch.full((n, k), float("-inf"), device="cuda")
            s["scores"][:, 0] = 0
            s["finished"].zero_()
    elif case["op"] == "reorder":
        n, k = case["groups"], case["beams"]
        s["pool"] = _pages(g, n * k, 0, case, case["layers"])
        s["pool"]["lens"] = torch.full((n * k,), case["length"], dtype=torch.int32, device="cuda")
        s["parents"] = _parents(g, (n, k), k)
    else:
        shape = (case["steps"], case["groups"], case["beams"])
        s["parents"] = _parents(g, shape, case["beams"])
        s["tokens"] = torch.randint(0, 151936, shape, device="cuda", generator=g, dtype=torch.int32)
        s["last"] = torch.randint(0, case["beams"], (case["groups"], case["picks"]), device="cuda", generator=g, dtype=torch.int32)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _values(p, which, c, rows, dtype):
    """The pool's values as [pages, page, kv_heads, dim]: what the stored codes stand for."""
    raw, scale = (p["k"][0], p["ks"]) if which == "k" else (p["v"][0], p["vs"])
    shape = (-1, c["page"], c["kv_heads"], c["dim"])
    if c["quant"] == "none":
        return raw.view(torch.bfloat16).reshape(shape)[rows].to(dtype)
    if c["quant"] == "int8":
        code = raw.reshape(shape)[rows].float() - 128
        return (code * scale[0][rows].to(torch.bfloat16).float()[..., None, None, None]).to(torch.bfloat16).to(dtype)
    byte = raw.reshape(-1, c["page"] * c["kv_heads"] * c["dim"] // 2)[rows]
    code = torch.stack([byte & 15, byte >> 4], dim=-1).float() - 8
    code = code.reshape(*byte.shape[:-1], -1, 32) * scale[0].reshape(-1, c["page"] * c["kv_heads"] * c["dim"] // 32)[rows][..., None]
    return code.to(torch.bfloat16).reshape(*byte.shape[:-1], *shape[1:]).to(dtype)


def _dense(p, which, c, tokens):
    """[rows, tokens, kv_heads, dim] in 32 bits; zeros past each row's length."""
    rows = p["table"].shape[0]
    x = _values(p, which, c, p["table"].long(), torch.float32).reshape(rows, -1, c["kv_heads"], c["dim"])[:, :tokens]
    keep = torch.arange(tokens, device="cuda")[None, :] < p["lens"][:, None]
    return torch.where(keep[:, :, None, None], x, 0.0), keep


def _plain_attn(s):
    c = s["case"]
    n, k, kvh, d = c["groups"], c["seqs"], c["kv_heads"], c["dim"]
    gq = c["heads"] // kvh
    q = s["q"].float().reshape(n, k, kvh, gq, d) * d ** -0.5
    kp, keep = _dense(s["prefix"], "k", c, c["prefix"])
    vp, _ = _dense(s["prefix"], "v", c, c["prefix"])
    # the queries of a group meet its prefix in one product: [n, kvh, k * gq, d] x [n, kvh, d, prefix]
    qg = q.permute(0, 2, 1, 3, 4).reshape(n, kvh, k * gq, d)
    sp = torch.matmul(qg, kp.permute(0, 2, 3, 1))
    sp = torch.where(keep[:, None, None, :], sp, float("-inf")).reshape(n, kvh, k, gq, -1)
    scores = sp
    if c["suffix"]:
        ks, keep_s = _dense(s["suffix"], "k", c, c["suffix"])
        vs, _ = _dense(s["suffix"], "v", c, c["suffix"])
        qs = q.reshape(n * k, kvh, gq, d)
        ss = torch.matmul(qs, ks.permute(0, 2, 3, 1))
        ss = torch.where(keep_s[:, None, None, :], ss, float("-inf")).reshape(n, k, kvh, gq, -1).permute(0, 2, 1, 3, 4)
        scores = torch.cat([sp, ss], dim=-1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., :c["prefix"]].reshape(n, kvh, k * gq, -1), vp.permute(0, 2, 1, 3)).reshape(n, kvh, k, gq, d)
    if c["suffix"]:
        ps = p[..., c["prefix"]:].permute(0, 2, 1, 3, 4).reshape(n * k, kvh, gq, -1)
        out = out + torch.matmul(ps, vs.permute(0, 2, 1, 3)).reshape(n, k, kvh, gq, d).permute(0, 2, 1, 3, 4)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 2, 1, 3, 4).reshape(n * k, c["heads"], d).to(torch.bfloat16)


def _plain_select(s):
    c = s["case"]
    n, k, v = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].double().reshape(n, k, v)  # candidates are ranked: 64 bits
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    score = s["scores"].double()[..., None]
    done = s["finished"].bool()[..., None]
    at_eos = (torch.arange(v, device="cuda") == s["eos"])[None, None, :]
    total = torch.where(done, torch.where(at_eos, score, float("-inf")), score + (x - lse)).reshape(n, k * v)
    best, at = torch.sort(total, dim=-1, descending=True, stable=True)  # equal totals keep the lowest index in front
    best, at = best[:, :c["n_out"]], at[:, :c["n_out"]]
    live = best > float("-inf")
    parents = torch.where(live, at // v, 0).to(torch.int32)
    tokens = torch.where(live, at % v, s["eos"]).to(torch.int32)
    done = live & (torch.gather(s["finished"].bool(), 1, parents.long()) | (tokens == s["eos"]))
    if best.shape[1] < c["n_out"]:
        more = c["n_out"] - best.shape[1]
        best = torch.cat([best, torch.full((n, more), float("-inf"), device="cuda", dtype=best.dtype)], 1)
        parents = torch.cat([parents, parents.new_zeros(n, more)], 1)
        tokens = torch.cat([tokens, tokens.new_full((n, more), s["eos"])], 1)
        done = torch.cat([done, done.new_zeros(n, more)], 1)
    return dict(scores=best.float(), parents=parents, tokens=tokens, finished=done.to(torch.uint8))


def _plain_reorder(s):
    c, p = s["case"], s["pool"]
    n, k, page = c["groups"], c["beams"], c["page"]
    table = p["table"].reshape(n, k, -1)
    par = s["parents"].long()
    full, held = c["length"] // page, c["length"] % page
    new = table.clone()
    new[:, :, :full] = torch.gather(table, 1, par[..., None].expand(-1, -1, table.shape[2]))[:, :, :full]
    if held:
        same = par[:, :, None] == par[:, None, :]
        earlier = torch.ones(k, k, device="cuda", dtype=torch.bool).tril(-1)
        again = (same & earlier).any(-1)                                       # not its parent's first child
        chosen = (par[:, :, None] == torch.arange(k, device="cuda")).any(1)     # beams that have a child
        order = torch.sort(chosen.to(torch.int32), dim=-1, stable=True).indices   # the childless ones in front, ascending
        rank = again.to(torch.int64).cumsum(-1) - 1
        own_page = torch.where(again, torch.gather(order, 1, rank.clamp(min=0)), par)
        src = torch.gather(table[:, :, full], 1, par)
        dst = torch.gather(table[:, :, full], 1, own_page)
        new[:, :, full] = dst
        src, dst = src.reshape(-1).long(), dst.reshape(-1).long()
        row = c["kv_heads"] * c["dim"]
        unit = {"none": row * 2, "int8": row, "q4_0": row // 2}[c["quant"]]
        for name in ("k", "v"):
            pool = p[name].reshape(c["layers"], -1, page * unit)
            pool[:, dst, :held * unit] = pool[:, src, :held * unit]
            if c["quant"] != "none":
                sc = p[name + "s"].reshape(c["layers"], pool.shape[1], -1)
                m = 1 if c["quant"] == "int8" else held * row // 32
                sc[:, dst, :m] = sc[:, src, :m]
    return dict(table=new.reshape(n * k, -1), **{x: p[x] for x in ("k", "v", "ks", "vs") if p[x] is not None})


def _plain_trace(s):
    out = torch.empty(*s["last"].shape, s["case"]["steps"], device="cuda", dtype=torch.int32)
    at = s["last"].long()
    for i in range(s["case"]["steps"] - 1, -1, -1):  # each step's choice needs the one after it
        out[:, :, i] = torch.gather(s["tokens"][i], 1, at)
        at = torch.gather(s["parents"][i], 1, at).long()
    return out


# ---- the library's entry points --------------------------------------------------------------------------------------
def _cache(p, c, layer=0):
    from izwi_b200 import paged
    return paged.PagedKvCache.view(p["k"][layer], p["v"][layer], None if p["ks"] is None else p["ks"][layer],
                                   None if p["vs"] is None else p["vs"][layer], p["table"], p["lens"], c["kv_heads"], c["dim"], c["quant"], c["page"])


def _own(s):
    from izwi_b200 import ops, paged
    c = s["case"]
    if c["op"] == "attn":
        if "caches" not in s:  # the handles that a serving loop keeps
            s["caches"] = (_cache(s["prefix"], c), _cache(s["suffix"], c) if c["suffix"] else None)
        return paged.shared_prefix_attention(s["q"], *s["caches"])
    if c["op"] == "select":
        return dict(zip(("scores", "parents", "tokens", "finished"),
                        ops.beam_select(s["logits"], s["scores"], c["n_out"], finished=s["finished"], eos=s["eos"])))
    if c["op"] == "reorder":
        p = s["pool"]
        if "layers" not in s:
            s["layers"] = paged.PagedLayers([_cache(p, c, i) for i in range(c["layers"])])
        return dict(table=s["layers"].reorder(s["parents"]), **{x: p[x] for x in ("k", "v", "ks", "vs") if p[x] is not None})
    return ops.beam_trace(s["parents"], s["tokens"], s["last"])


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "select": _plain_select, "reorder": _plain_reorder, "trace": _plain_trace}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "attn":
        batch = c["groups"] * c["seqs"]
        per_value = {"none": 2, "int8": 1, "q4_0": 0.5 + 4 / 32}[c["quant"]]
        tokens_p, tokens_s = sum(_lens(c["groups"], c["prefix"], c["ragged"])), sum(_lens(batch, c["suffix"], c["ragged"]))
        kv = 2 * (tokens_p + tokens_s) * c["kv_heads"] * c["dim"] * per_value
        return dict(bytes=kv + 4 * batch * c["heads"] * c["dim"], flops=4 * c["heads"] * c["dim"] * (tokens_p * c["seqs"] + tokens_s))
    if c["op"] == "select":
        n = c["groups"] * c["beams"] * c["vocab"]
        if c["first"]:
            n //= c["beams"]  # the rows of beams that are not alive need no reading
        return dict(bytes=n * (2 if c["dtype"] == "bf16" else 4) + 13 * c["groups"] * c["n_out"], flops=3 * n)
    if c["op"] == "reorder":
        k = c["beams"]
        share = [((i + 1) / k) ** (1 / 1.5) - (i / k) ** (1 / 1.5) for i in range(k)]  # of _parents
        copies = k - sum(1 - (1 - x) ** k for x in share)
        per_value = {"none": 2, "int8": 1, "q4_0": 0.5 + 4 / 32}[c["quant"]]
        held = c["length"] % c["page"]
        moved = c["groups"] * copies * c["layers"] * 2 * held * c["kv_heads"] * c["dim"] * per_value
        return dict(bytes=2 * moved + 8 * c["groups"] * k * c["pages"], flops=0)
    return dict(bytes=4 * c["groups"] * c["steps"] * (2 * c["beams"] + c["picks"]), flops=0)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _stored(p, which, c, row, length):
    """[length, kv_heads, dim] in 64 bits: token by token from the row's pages."""
    t = torch.arange(length, device="cuda")
    pages = p["table"][row].long()[t // c["page"]]
    slot = t % c["page"]
    raw = p[which][0]
    n = c["kv_heads"] * c["dim"]
    first = (pages * c["page"] + slot)[:, None] * n + torch.arange(n, device="cuda")[None, :]
    if c["quant"] == "none":
        x = raw.view(torch.bfloat16)[first].double()
    elif c["quant"] == "int8":
        scale = p[which + "s"][0][pages].bfloat16().double()[:, None]
        x = ((raw[first].double() - 128) * scale).float().bfloat16().double()
    else:
        code = (raw[first // 2].int() >> (4 * (first % 2)).int()) & 15
        x = ((code.double() - 8) * p[which + "s"][0][first // 32].double()).float().bfloat16().double()
    return x.reshape(length, c["kv_heads"], c["dim"])


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "attn":
        out = torch.zeros(c["groups"] * c["seqs"], c["heads"], c["dim"], device="cuda", dtype=torch.float64)
        gq = c["heads"] // c["kv_heads"]
        lens_p = s["prefix"]["lens"].tolist()
        for g in range(c["groups"]):
            kp, vp = (_stored(s["prefix"], w, c, g, lens_p[g]) for w in "kv")
            for i in range(g * c["seqs"], (g + 1) * c["seqs"]):
                k, v = kp, vp
                if c["suffix"]:
                    m = int(s["suffix"]["lens"][i])
                    k, v = torch.cat([kp, _stored(s["suffix"], "k", c, i, m)]), torch.cat([vp, _stored(s["suffix"], "v", c, i, m)])
                q = s["q"][i].double().reshape(c["kv_heads"], gq, c["dim"])
                w = torch.softmax(torch.einsum("kgd,tkd->kgt", q, k) / c["dim"] ** 0.5, dim=-1)
                out[i] = torch.einsum("kgt,tkd->kgd", w, v).reshape(c["heads"], c["dim"])
        return out
    if c["op"] == "select":
        lp = torch.log_softmax(s["logits"].double(), dim=-1).reshape(c["groups"], c["beams"], -1) + s["scores"].double()[..., None]
        for g, b in s["finished"].nonzero().tolist():
            lp[g, b] = float("-inf")
            lp[g, b, s["eos"]] = s["scores"][g, b].double()
        lp = lp.reshape(c["groups"], -1)
        want = min(c["n_out"], lp.shape[1])
        best = torch.full((c["groups"], c["n_out"]), float("-inf"), device="cuda", dtype=torch.float64)
        best[:, :want] = torch.topk(lp, want, dim=-1).values
        return dict(scores=best, parents=None, tokens=None, finished=None)
    return None

"""Cases of the operators between the matmuls of a decode step and at its end: the norm and rotation of query and key heads,
the paged cache (written in f16, 8 or 4 bits a value, and read back), attention of drafted tokens over it, and the penalties,
biases and grammar masks of the logits.

Kinds of case
  rope     capi.qk_norm_rope: one token to a prompt, whole and partial rotation, both pair orders, with and without the norm
  cache    capi.kv_append of new tokens, then capi.kv_read of slots of the cache
  attn     capi.attention_tree: sequences of unlike lengths in pages, one token each or a tree of drafted ones
  logits   capi.logits_adjust: histories, sparse biases, grammar masks, one row to a batch

A cache's pages are [page][kv head][slot][row]: rows of f16 values, or of quants (8 bits: one signed byte a value; 4 bits: blocks of
32 values in 16 bytes, value j of a block in the low half of byte j, value j + 16 in the high half, 8 above its value) whose scales,
one f16 a block of 32 values, lie in a tensor of their own.
"""
import math

import torch

own = False


def listed():
    return [
        # one token of a decode step, rotation alone: the smallest call
        {"name": "rope_1", "kind": "rope", "tokens": 1, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128, "pairs": "adjacent", "norm": False, "far": 4096},
        # seven drafted tokens of a model that rotates a part of each head, far into a long context
        {"name": "rope_partial_7", "kind": "rope", "tokens": 7, "heads": 28, "kv_heads": 4, "d": 256, "rot": 64, "pairs": "halves", "norm": True, "far": 1000000},
        # a prompt of 2048 tokens with per-head norms
        {"name": "rope_2048", "kind": "rope", "tokens": 2048, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128, "pairs": "halves", "norm": True, "far": 131072},
        # drafted tokens of four sequences into an 8-bit cache
        {"name": "cache_q8_32", "kind": "cache", "ct": "q8", "append": 32, "read": 32, "kv_heads": 8, "d": 128, "page": 16, "pages": 2048},
        # a prompt into a 4-bit cache, and a whole context out of it
        {"name": "cache_q4_2048", "kind": "cache", "ct": "q4", "append": 2048, "read": 8191, "kv_heads": 8, "d": 128, "page": 64, "pages": 256},
        # the smallest attention: one token over a short context, f16
        {"name": "attn_f16_1", "kind": "attn", "ct": "f16", "seqs": 1, "most": 1, "heads": 32, "kv_heads": 8, "d": 128, "len": 300, "page": 16,
         "window": 0, "sinks": False, "softcap": 0.0},
        # one token over a very long context, 8-bit cache
        {"name": "attn_q8_long", "kind": "attn", "ct": "q8", "seqs": 1, "most": 1, "heads": 32, "kv_heads": 8, "d": 128, "len": 131072, "page": 64,
         "window": 0, "sinks": False, "softcap": 0.0},
        # a serving batch, one to eight drafted tokens each, unlike lengths
        {"name": "attn_q8_batch", "kind": "attn", "ct": "q8", "seqs": 48, "most": 8, "heads": 32, "kv_heads": 8, "d": 128, "len": 8000, "page": 16,
         "window": 0, "sinks": False, "softcap": 0.0},
        # large trees over long contexts, f16
        {"name": "attn_f16_trees", "kind": "attn", "ct": "f16", "seqs": 4, "most": 64, "heads": 32, "kv_heads": 8, "d": 128, "len": 16384, "page": 64,
         "window": 0, "sinks": False, "softcap": 0.0},
        # heads of 64 values, seven queries to a key head, a window and sinks, 4-bit cache
        {"name": "attn_q4_window", "kind": "attn", "ct": "q4", "seqs": 17, "most": 5, "heads": 56, "kv_heads": 8, "d": 64, "len": 5000, "page": 48,
         "window": 1024, "sinks": True, "softcap": 0.0},
        # one sampled row
        {"name": "logits_1", "kind": "logits", "rows": 1, "vocab": 128256, "history": 512, "biases": 16, "grammar": True},
        # a serving batch of rows, some of them under a grammar
        {"name": "logits_64", "kind": "logits", "rows": 64, "vocab": 128256, "history": 4096, "biases": 300, "grammar": True},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choices(["rope", "cache", "attn", "logits"], [20, 20, 40, 20])[0]
    heads, kv = rng.choice([(32, 8), (32, 32), (28, 4), (16, 1), (24, 3), (5, 5), (64, 8), (40, 8)])
    d = rng.choice([64, 64, 96, 128, 128, 128, 192, 256])
    if kind == "rope":
        return {"kind": kind, "tokens": min(_log(rng, 1, 2048), 2048 * 40 * 128 // ((heads + kv) * d)), "heads": heads, "kv_heads": kv, "d": d,
                "rot": rng.choice([d, d, d // 2, d // 4]), "pairs": rng.choice(["halves", "adjacent"]), "norm": rng.random() < 0.6, "far": _log(rng, 100, 1000000)}
    if kind == "cache":
        page = rng.choice([16, 32, 48, 64, 256])
        most = 8192 * 8 * 128 // (kv * d)
        return {"kind": kind, "ct": rng.choice(["f16", "q8", "q4"]), "append": min(_log(rng, 1, 2048), most // 4), "read": min(_log(rng, 1, 8192), most), "kv_heads": kv, "d": d,
                "page": page, "pages": 16384 // page}
    if kind == "attn":
        c = {"kind": kind, "ct": rng.choice(["f16", "q8", "q8", "q4"]), "seqs": _log(rng, 1, 64), "most": rng.choice([1, 1, 1, _log(rng, 1, 16), _log(rng, 1, 64)]),
             "heads": heads, "kv_heads": kv, "d": d, "len": _log(rng, 16, 131072), "page": rng.choice([16, 32, 48, 64, 256]),
             "window": rng.choice([0, 0, 0, _log(rng, 64, 2048)]), "sinks": rng.random() < 0.3, "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
        c["len"] = max(c["len"], c["most"])
        # at most the bytes of the longest listed context and the products of the listed trees
        while c["len"] > c["most"] and (work(c)["bytes"] > 285e6 or work(c)["flops"] > 20e9):
            c["len"] = max(c["most"], int(0.9 * c["len"]))
        if work(c)["flops"] > 20e9:
            c["seqs"] = max(1, int(c["seqs"] * 20e9 / work(c)["flops"]))
        return c
    rows = _log(rng, 1, 64)
    return {"kind": kind, "rows": rows, "vocab": min(_log(rng, 32000, 262144), 64 * 128256 // rows), "history": _log(rng, 1, 4096), "biases": rng.choice([0, _log(rng, 1, 300)]),
            "grammar": rng.random() < 0.6}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _cache(ct, pages, kv, page, d, gen):
    """Rows as a program left them: normal values, and their quants under scales of unlike size."""
    def one():
        if ct == "f16":
            return torch.randn((pages, kv, page, d), device="cuda", generator=gen).half(), None
        scale = (torch.rand((pages, kv, page, d // 32), device="cuda", generator=gen) + 0.5)
        if ct == "q8":
            return torch.randint(-127, 128, (pages, kv, page, d), dtype=torch.int8, device="cuda", generator=gen), (scale / 73).half()
        return torch.randint(0, 256, (pages, kv, page, d // 2), dtype=torch.uint8, device="cuda", generator=gen), (scale / -4.6).half()
    k, ks = one()
    v, vs = one()
    return {"ct": ct, "k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _batch(case):
    """Drafted tokens and lengths of the sequences: lengths from short ones up, with the drafted tokens among them; one sequence has the
    most of both, and in a larger batch one has drafted tokens alone."""
    n, most = case["seqs"], case["most"]
    count = [most] + [1 + int(0.618034 * i % 1 * most) for i in range(1, n)]
    u = [0.754878 * i % 1 for i in range(n)]
    length = [case["len"]] + [max(count[i], int(case["len"] * u[i] * max(u[i], 0.5))) for i in range(1, n)]
    if n > 3:
        length[1] = count[1]
    return count, length


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    kind, s = case["kind"], {"case": case}

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    if kind == "rope":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["d"]
        # the three outputs of the q/k/v projection lie in one row, as one product leaves them
        row = normal(t, (h + 2 * kv) * d)
        s["q"] = row[:, :h * d].unflatten(1, (h, d))
        s["k"] = row[:, h * d:(h + kv) * d].unflatten(1, (kv, d))
        start = torch.randint(0, max(1, case["far"] - t + 1), (1,), generator=host)
        s["pos"] = (start + torch.arange(t)).to(torch.int32).cuda()
        s["inv_freq"] = (500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).float().cuda()
        s["wq"], s["wk"] = (1 + 0.3 * normal(d), 1 + 0.3 * normal(d)) if case["norm"] else (None, None)
    elif kind == "cache":
        s |= _cache(case["ct"], case["pages"], case["kv_heads"], case["page"], case["d"], gen)
        slots = torch.randperm(case["pages"] * case["page"], device="cuda", generator=gen)
        s["to"] = slots[:case["append"]].contiguous()
        # what was just written is read back, and older tokens with it
        s["of"] = slots[:case["read"]].flip(0).contiguous()
        s["k_new"], s["v_new"] = (normal(case["append"], case["kv_heads"], case["d"]) for _ in range(2))
    elif kind == "attn":
        n, most, page = case["seqs"], case["most"], case["page"]
        count, length = (torch.tensor(x) for x in _batch(case))
        masks = []
        for c in count.tolist():
            r = torch.rand(c, generator=host).tolist()
            m = []
            for i in range(c):
                # chains mostly, branches here and there, now and then a second root
                parent = i - 1 if r[i] < 0.6 else int((r[i] - 0.6) / 0.4 * (i + 1)) - 1
                m.append((m[parent] if parent >= 0 else 0) | 1 << i)
            masks += m
        if n > 3 and count[1] > 1:
            masks[int(count[0]) + 1] = 0   # a row that sees nothing
        s["tree"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).cuda()
        s["q_start"] = torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)]).to(torch.int32).cuda()
        s["kv_len"] = length.to(torch.int32).cuda()
        used = (length + page - 1) // page
        table = torch.full((n, int(used.max())), -1, dtype=torch.int32)
        table[torch.arange(table.shape[1]) < used[:, None]] = torch.randperm(int(used.sum()), generator=host).to(torch.int32)
        s["table"] = table.cuda()
        s |= _cache(case["ct"], int(used.sum()), case["kv_heads"], page, case["d"], gen)
        s["q"] = 2 * normal(len(masks), case["heads"], case["d"])
        s["sinks"] = normal(case["heads"]) if case["sinks"] else None
        s["scale"] = case["d"] ** -0.5
        s["total"] = int(used.max()) * page
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = 3 * normal(rows, vocab)

        def ids(n):   # frequent tokens often, the same one many times
            return (vocab * torch.rand((rows, n), device="cuda", generator=gen) ** 6).to(torch.int32).clamp_(max=vocab - 1)
        s["hist"] = ids(case["history"])
        s["hist_len"] = (torch.rand(rows, generator=host) * (case["history"] + 1)).to(torch.int32).clamp_(max=case["history"]).cuda()
        s["hist_len"][0] = case["history"]
        s["rep"], s["freq"], s["pres"] = (a + b * torch.rand(rows, device="cuda", generator=gen) for a, b in ((1.0, 0.3), (0.0, 0.5), (0.0, 0.5)))
        if case["biases"]:
            s["bias_ids"], s["bias"] = ids(case["biases"]), 5 * normal(rows, case["biases"])
        if case["grammar"]:
            # half of the rows are under a grammar, which allows a few tokens or most of them
            share = torch.tensor([0.001, 0.1, 0.9], device="cuda").repeat((rows + 5) // 6 + 1)[:max(1, rows // 2)]
            ok = torch.rand((len(share), (vocab + 31) // 32 * 32), device="cuda", generator=gen) < share[:, None]
            s["mask"] = (ok.view(len(share), -1, 32).long() << torch.arange(32, device="cuda")).sum(2).to(torch.uint32).view(torch.int32)
            row = torch.full((rows,), -1, dtype=torch.int32)
            row[::2][:len(share)] = torch.arange(len(share), dtype=torch.int32)[:len(row[::2])]
            s["mask_row"] = row.cuda()
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def _decode(pool, scale, ct):
    """Rows of a cache as f32 values."""
    if ct == "f16":
        return pool.float()
    if ct == "q4":
        b = pool.unflatten(-1, (-1, 16))
        q = torch.cat([b & 15, b >> 4], -1).float() - 8
    else:
        q = pool.unflatten(-1, (-1, 32)).float()
    return (q * scale.float()[..., None]).flatten(-2)


def _encode(x, ct):
    """f32 rows as a cache holds them."""
    if ct == "f16":
        return x.half(), None
    b = x.unflatten(-1, (-1, 32))
    if ct == "q8":
        d = (b.abs().amax(-1) / 127).half()
        q = torch.round(b / d.float()[..., None]).clamp(-127, 127)
        return torch.where(d[..., None] != 0, q, 0).to(torch.int8).flatten(-2), d
    hi, lo = b.amax(-1), b.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) / -8).half()
    q = torch.where(d[..., None] != 0, torch.round(b / d.float()[..., None]) + 8, 8).clamp(0, 15).to(torch.uint8)
    return (q[..., :16] | q[..., 16:] << 4).flatten(-2), d


def _plain_rope(s):
    case = s["case"]
    rot = case["rot"]
    # the angle of a far position keeps its fraction of a turn only in 64 bits
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def one(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        r = x[..., :rot]
        if case["pairs"] == "halves":
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = r[..., ::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([r, x[..., rot:]], -1)
    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _plain_cache(s):
    ct, page = s["ct"], s["case"]["page"]
    out = []
    for new, pool, scale in ((s["k_new"], s["k"], s["k_scale"]), (s["v_new"], s["v"], s["v_scale"])):
        q, d = _encode(new, ct)
        pool[s["to"] // page, :, s["to"] % page] = q
        if d is not None:
            scale[s["to"] // page, :, s["to"] % page] = d
        of = (s["of"] // page, slice(None), s["of"] % page)
        out.append(_decode(pool[of], None if d is None else scale[of], ct))
    return out


def _seen(s, device="cuda"):
    """[seqs][most][positions]: what a drafted token sees, and which rows there are."""
    case = s["case"]
    start, length = s["q_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(case["most"], device=device)
    there = i < count[:, None]
    row = (start[:-1, None] + i).clamp(max=len(s["tree"]) - 1)
    bits = (s["tree"][row][..., None] >> torch.arange(64, device=device)) & 1
    before = length - count
    p = torch.arange(s["total"], device=device)
    j = p - before[:, None]
    drafted = torch.gather(bits, 2, j.clamp(0, 63)[:, None].expand(-1, case["most"], -1)).bool() & ((j >= 0) & (p < length[:, None]))[:, None]
    context = (p < before[:, None])[:, None]
    if case["window"]:
        context = context & (before[:, None] + bits.sum(-1) - 1)[..., None].sub(p).lt(case["window"])
    return (drafted | context) & there[..., None], row, there


def _plain_attn(s):
    case = s["case"]
    n, most, h, kv, d = case["seqs"], case["most"], case["heads"], case["kv_heads"], case["d"]
    seen, row, there = _seen(s)
    pages = s["table"].long().clamp(min=0)
    k, v = (_decode(s[x][pages], None if s[x + "_scale"] is None else s[x + "_scale"][pages], s["ct"]).transpose(2, 1).flatten(2, 3) for x in ("k", "v"))
    q = s["q"][row].view(n, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    score = (q @ k.transpose(2, 3)).mul_(s["scale"])
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    score = score.view(n, kv, h // kv, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    sink = None
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, kv, h // kv, 1, 1)
        top = torch.maximum(top, sink)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    o = (p.view(n, kv, -1, s["total"]) @ v).view(n, kv, h // kv, most, d) / torch.where(total > 0, total, 1)
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, h, d)[there]


def _plain_logits(s):
    x = s["logits"]
    rows, vocab = x.shape
    at = torch.arange(s["hist"].shape[1], device="cuda")
    count = torch.zeros_like(x).scatter_add_(1, s["hist"].long(), (at < s["hist_len"][:, None]).float())
    if "bias" in s:
        # of an id that is listed twice the last one holds
        last = torch.full((rows, vocab), -1, device="cuda").scatter_reduce_(1, s["bias_ids"].long(), torch.arange(s["bias"].shape[1], device="cuda").expand(rows, -1), "amax")
        x = x + torch.where(last >= 0, s["bias"].gather(1, last.clamp(min=0)), 0)
    rep, freq, pres = (s[n][:, None] for n in ("rep", "freq", "pres"))
    x = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep) - (freq * count + pres), x)
    if "mask" in s:
        ok = ((s["mask"].long()[..., None] >> torch.arange(32, device="cuda")) & 1).flatten(1)[:, :vocab].bool()
        x = torch.where((s["mask_row"] < 0)[:, None] | ok[s["mask_row"].long().clamp(min=0)], x, -math.inf)
    return x


def _own(s):
    from kraken_b200 import capi
    case, kind = s["case"], s["case"]["kind"]
    if kind == "rope":
        return capi.qk_norm_rope(s["q"], s["k"], s["pos"], s["inv_freq"], s["wq"], s["wk"], norm=case["norm"], eps=1e-6, interleaved=case["pairs"] == "adjacent")
    if kind == "logits":
        return capi.logits_adjust(s["logits"], s["hist"], s["hist_len"], s["rep"], s["freq"], s["pres"], s.get("bias_ids"), s.get("bias"), s.get("mask"), s.get("mask_row"))
    if "cache" not in s:   # the handle that a program keeps
        s["cache"] = capi.KvCache({"f16": capi.KV_F16, "q8": capi.KV_Q8, "q4": capi.KV_Q4}[s["ct"]], s["k"], s["v"], s["k_scale"], s["v_scale"])
    if kind == "cache":
        capi.kv_append(s["cache"], s["k_new"], s["v_new"], s["to"])
        return capi.kv_read(s["cache"], s["of"])
    return capi.attention_tree(s["q"], s["cache"], s["q_start"], s["kv_len"], s["table"], case["most"], s["tree"], scale=s["scale"], softcap=case["softcap"],
                               window=case["window"], sinks=s["sinks"])


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "cache": _plain_cache, "attn": _plain_attn, "logits": _plain_logits}[state["case"]["kind"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _values(s, name, page, slot):
    """[n][kv heads][d] in 64 bits of the cache's rows at (page, slot)."""
    x = s[name][page, :, slot]
    if s["ct"] == "f16":
        return x.double()
    d = s[name + "_scale"][page, :, slot].double().repeat_interleave(32, -1)
    if s["ct"] == "q8":
        return x.double() * d
    j = torch.arange(s["case"]["d"], device="cuda")
    byte = x[..., j // 32 * 16 + j % 16].long()
    return (torch.where(j % 32 < 16, byte % 16, byte // 16) - 8).double() * d


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        rot, out = case["rot"], []
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * s["inv_freq"].double())[:, None]
        for x, w in ((s["q"].double(), s["wq"]), (s["k"].double(), s["wk"])):
            if w is not None:
                x = w.double() * x / ((x ** 2).sum(-1, keepdim=True) / case["d"] + 1e-6).sqrt()
            y = x.clone()
            a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if case["pairs"] == "halves" else (slice(0, rot, 2), slice(1, rot, 2))
            z = torch.complex(x[..., a], x[..., b]) * turn
            y[..., a], y[..., b] = z.real, z.imag
            out.append(y)
        return tuple(out)
    if kind == "cache":
        page, out = case["page"], []
        at = torch.full((case["pages"] * page,), -1, device="cuda")
        at[s["to"]] = torch.arange(case["append"], device="cuda")
        new_at = at[s["of"]]
        for name in ("k", "v"):
            x = s[name + "_new"].double()
            if case["ct"] == "f16":
                y = x.half().double()
            else:
                b = x.view(*x.shape[:2], -1, 32)
                if case["ct"] == "q8":
                    d = (b.abs().max(-1).values / 127).float().half().double()[..., None]
                    y = (b / d).round().clamp(-127, 127) * d
                else:
                    top = b.gather(-1, b.abs().max(-1).indices[..., None])
                    d = (top / -8).float().half().double()
                    y = (b / d).round().clamp(-8, 7) * d
                y = y.view(x.shape)
            old = _values(s, name, s["of"] // page, s["of"] % page)
            out.append(torch.where((new_at >= 0)[:, None, None], y[new_at.clamp(min=0)], old))
        return out
    if kind == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        start, length, tree = s["q_start"].tolist(), s["kv_len"].tolist(), s["tree"].tolist()
        group = case["heads"] // case["kv_heads"]
        for i, n in enumerate(length):
            rows = range(start[i], start[i + 1])
            before = n - len(rows)
            ok = torch.zeros((len(rows), n), dtype=torch.bool)
            for a, r in enumerate(rows):
                m = tree[r] & (1 << 64) - 1
                first = max(0, before + bin(m).count("1") - case["window"]) if case["window"] else 0
                ok[a, first:before] = True
                for b in range(len(rows)):
                    ok[a, before + b] = bool(m >> b & 1)
            ok = ok.cuda()
            p = torch.arange(n, device="cuda")
            page, slot = s["table"][i].long()[p // case["page"]], p % case["page"]
            k, v = _values(s, "k", page, slot), _values(s, "v", page, slot)
            for h in range(case["heads"]):
                z = s["q"][start[i]:start[i + 1], h].double() @ k[:, h // group].T * s["scale"]
                if case["softcap"]:
                    z = torch.tanh(z / case["softcap"]) * case["softcap"]
                z = torch.where(ok, z, -math.inf)
                if s["sinks"] is not None:
                    z = torch.cat([z, s["sinks"][h].double().expand(len(rows), 1)], 1)
                w = torch.softmax(z, 1).nan_to_num(0.0)[:, :n]
                out[start[i]:start[i + 1], h] = w @ v[:, h // group]
        return out
    x = s["logits"].double()
    for r in range(case["rows"]):
        y = x[r]
        if "bias" in s:
            pairs = dict(zip(s["bias_ids"][r].tolist(), s["bias"][r].double().tolist()))
            y[torch.tensor(list(pairs), device="cuda")] += torch.tensor(list(pairs.values()), dtype=torch.float64, device="cuda")
        ids, times = torch.unique(s["hist"][r, :int(s["hist_len"][r])].long(), return_counts=True)
        z, rep = y[ids], s["rep"][r].double()
        y[ids] = torch.where(z > 0, z / rep, z * rep) - s["freq"][r].double() * times - s["pres"][r].double()
        if "mask" in s and s["mask_row"][r] >= 0:
            i = torch.arange(case["vocab"], device="cuda")
            y[(s["mask"][int(s["mask_row"][r])].long()[i // 32] >> i % 32) % 2 == 0] = -math.inf
    return x


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rope":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["d"]
        return {"bytes": 8 * values + 4 * case["tokens"], "flops": (3 + 4 * case["norm"]) * values}
    if kind in ("cache", "attn"):
        row = case["kv_heads"] * {"f16": 2 * case["d"], "q8": case["d"] + case["d"] // 16, "q4": case["d"] // 2 + case["d"] // 16}[case["ct"]]
    if kind == "cache":
        return {"bytes": 2 * (case["append"] + case["read"]) * (4 * case["kv_heads"] * case["d"] + row), "flops": 0}
    if kind == "attn":
        count, length = _batch(case)
        seen = [min(n, case["window"] + c - 1) if case["window"] else n for c, n in zip(count, length)]
        positions, pairs, tokens = sum(seen), sum(c * (min(n, case["window"]) if case["window"] else n) for c, n in zip(count, length)), sum(count)
        return {"bytes": 2 * positions * row + 8 * tokens * case["heads"] * case["d"], "flops": 4 * pairs * case["heads"] * case["d"]}
    rows = case["rows"]
    lists = 4 * case["history"] + 8 * case["biases"]
    return {"bytes": rows * (8 * case["vocab"] + lists) + (max(1, rows // 2) * case["vocab"] // 8 if case["grammar"] else 0), "flops": rows * case["vocab"]}

"""Cases of the operators of a step that mixes prompts and drafted tokens: the plan of the step (pages, slots, positions from the
requests' lengths), the norms either side of a block with its gate and residual, attention of chunks of prompts over the paged cache,
and the verification of drafted tokens against the target's probabilities.

Kinds of case
  plan    capi.step_plan: new tokens of each request get pages, slots and positions
  norm    capi.block_norm: norm of a block's output, gate, residual, and the norm before the next block
  chunk   capi.attention_chunk: chunks of prompts, of one token to thousands, behind contexts of unlike lengths
  verify  capi.verify_draft: drafted tokens are accepted or refused by given random numbers, one more token is drawn, and
          the logarithms of the target's probabilities of what came out

A cache's pages are [page][kv head][slot][row]: rows of f16 values, or of quants (8 bits: one signed byte a value; 4 bits: blocks of
32 values in 16 bytes, value j of a block in the low half of byte j, value j + 16 in the high half, 8 above its value) whose scales,
one f16 a block of 32 values, lie in a tensor of their own.
"""
import math

import torch

own = False


def listed():
    return [
        # a decode step of a few requests: the smallest plan
        {"name": "plan_8", "kind": "plan", "seqs": 8, "most": 4, "context": 2000, "page": 16, "tokens": 32},
        # a long step of prompts: hundreds of requests, some of them decoding, all of them short of the buffer's end
        {"name": "plan_512", "kind": "plan", "seqs": 512, "most": 600, "context": 8000, "page": 64, "tokens": 131072},
        # one token between two blocks
        {"name": "norm_1", "kind": "norm", "rows": 1, "n": 4096, "post": False, "gate": "none", "out": "f32"},
        # a prompt between two blocks with norms on both sides and a learned gate; the result is the f16 input of the next products
        {"name": "norm_2048", "kind": "norm", "rows": 2048, "n": 4096, "post": True, "gate": "vector", "out": "f16"},
        # a short prompt with nothing before it: the smallest attention
        {"name": "chunk_33", "kind": "chunk", "ct": "f16", "act": "f32", "seqs": 1, "most": 33, "context": 0, "heads": 32, "kv_heads": 8, "d": 128, "page": 16,
         "window": 0, "sinks": False, "softcap": 0.0},
        # a prompt at once, in f32 as the matmuls of this path give and take it
        {"name": "chunk_2048", "kind": "chunk", "ct": "f16", "act": "f32", "seqs": 1, "most": 2048, "context": 0, "heads": 32, "kv_heads": 8, "d": 128, "page": 64,
         "window": 0, "sinks": False, "softcap": 0.0},
        # the third chunk of a long prompt, in f16
        {"name": "chunk_long", "kind": "chunk", "ct": "f16", "act": "f16", "seqs": 1, "most": 4096, "context": 8192, "heads": 32, "kv_heads": 8, "d": 128, "page": 64,
         "window": 0, "sinks": False, "softcap": 0.0},
        # a serving batch of unlike chunks, single tokens among them, over an 8-bit cache
        {"name": "chunk_q8_batch", "kind": "chunk", "ct": "q8", "act": "f16", "seqs": 24, "most": 512, "context": 8000, "heads": 32, "kv_heads": 8, "d": 128, "page": 16,
         "window": 0, "sinks": False, "softcap": 0.0},
        # the same cache with f32 activations
        {"name": "chunk_q8_f32", "kind": "chunk", "ct": "q8", "act": "f32", "seqs": 2, "most": 700, "context": 5000, "heads": 32, "kv_heads": 8, "d": 128, "page": 32,
         "window": 0, "sinks": False, "softcap": 0.0},
        # heads of 64 values, seven queries to a key head, a window and sinks, 4-bit cache
        {"name": "chunk_q4_window", "kind": "chunk", "ct": "q4", "act": "f16", "seqs": 5, "most": 1500, "context": 4000, "heads": 56, "kv_heads": 8, "d": 64, "page": 48,
         "window": 1024, "sinks": True, "softcap": 0.0},
        # drafts of one request that were looked up, not drawn
        {"name": "verify_1", "kind": "verify", "seqs": 1, "most": 5, "vocab": 128256, "drafter": False},
        # a serving batch of requests with up to seven drafted tokens of a small model
        {"name": "verify_64", "kind": "verify", "seqs": 64, "most": 7, "vocab": 128256, "drafter": True},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choices(["plan", "norm", "chunk", "verify"], [15, 20, 45, 20])[0]
    if kind == "plan":
        seqs = _log(rng, 1, 2048)
        most = _log(rng, 1, min(8192, 131072 // seqs))
        return {"kind": kind, "seqs": seqs, "most": most, "context": _log(rng, 1, 131072), "page": rng.choice([16, 32, 48, 64, 256]),
                "tokens": rng.choice([seqs * most, _log(rng, 1, seqs * most)])}
    if kind == "norm":
        n = rng.choice([4096, 11008, 8 * _log(rng, 1, 2048), 8 * _log(rng, 1, 2048)])
        return {"kind": kind, "rows": min(_log(rng, 1, 2048), 2048 * 4096 // n), "n": n, "post": rng.random() < 0.5, "gate": rng.choice(["none", "vector", "rows"]),
                "out": rng.choice(["f32", "f16"])}
    if kind == "verify":
        seqs = _log(rng, 1, 64)
        vocab = _log(rng, 32000, 262144)
        most = min(_log(rng, 1, 15), 64 * 8 * 128256 // (seqs * vocab) - 1)
        return {"kind": kind, "seqs": seqs, "most": max(0, most), "vocab": vocab, "drafter": rng.random() < 0.6}
    heads, kv = rng.choice([(32, 8), (32, 32), (28, 4), (16, 1), (24, 3), (5, 5), (64, 8), (40, 8)])
    c = {"kind": kind, "ct": rng.choice(["f16", "f16", "q8", "q4"]), "act": rng.choice(["f32", "f16"]), "seqs": _log(rng, 1, 32), "most": _log(rng, 1, 4096),
         "context": rng.choice([0, _log(rng, 16, 32768), _log(rng, 16, 32768)]), "heads": heads, "kv_heads": kv, "d": rng.choice([64, 64, 96, 128, 128, 128, 192, 256]),
         "page": rng.choice([16, 32, 48, 64, 256]), "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]), "sinks": rng.random() < 0.3, "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
    # a quarter of the products of the longest listed chunk, at most the bytes of its cache ten times
    while c["seqs"] > 1 and (work(c)["bytes"] > 1e9 or work(c)["flops"] > 150e9):
        c["seqs"] = max(1, c["seqs"] * 3 // 4)
    while c["most"] > 1 and work(c)["flops"] > 150e9:
        c["most"] = max(1, c["most"] * 3 // 4)
    return c


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
    """New tokens of the sequences and positions before them. One has the most of both; of a larger batch some bring one token, and one
    has nothing before it."""
    n, most = case["seqs"], case["most"]
    count = [most] + [1 if i % 3 == 2 else 1 + int(0.618034 * i % 1 * most) for i in range(1, n)]
    before = [case["context"]] + [int(case["context"] * max(0.754878 * i % 1, 0.1)) for i in range(1, n)]
    if n > 3:
        before[1] = 0
    return count, before


def _drafted(case):
    """Drafted tokens of each request, from none up; the first has the most."""
    return [case["most"]] + [int(0.618034 * i % 1 * (case["most"] + 1)) for i in range(1, case["seqs"])]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    kind, s = case["kind"], {"case": case}

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    if kind == "plan":
        n, page = case["seqs"], case["page"]
        new = torch.randint(0, case["most"] + 1, (n,), generator=host)
        new[0] = case["most"]
        before = torch.randint(0, case["context"] + 1, (n,), generator=host)
        new[(new == 0) & (torch.rand(n, generator=host) < 0.7)] = 1
        have, need = (before + page - 1) // page, (before + new + page - 1) // page
        width = (case["context"] + case["most"] + page - 1) // page
        order = torch.randperm(int(need.sum()) + 16, generator=host).to(torch.int32)
        s["table"] = torch.full((n, width), -1, dtype=torch.int32)
        s["table"][torch.arange(width) < have[:, None]] = order[:int(have.sum())]
        s["table"] = s["table"].cuda()
        # the pages that no request has, as a stack; a few more than are taken
        s["free"] = order[int(have.sum()):].cuda()
        s["n_free"] = torch.tensor([len(s["free"])], dtype=torch.int32).cuda()
        s["before"], s["new"] = before.to(torch.int32).cuda(), new.to(torch.int32).cuda()
    elif kind == "norm":
        rows, n = case["rows"], case["n"]
        s["x"], s["residual"] = 0.7 * normal(rows, n), 2 * normal(rows, n)
        s["weight"] = 1 + 0.3 * normal(n)
        s["post"] = 1 + 0.3 * normal(n) if case["post"] else None
        s["gate"] = {"none": None, "vector": 0.5 * normal(n), "rows": 0.5 * normal(rows, n)}[case["gate"]]
    elif kind == "chunk":
        n, page = case["seqs"], case["page"]
        count, before = (torch.tensor(x) for x in _batch(case))
        s["q_start"] = torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)]).to(torch.int32).cuda()
        s["kv_len"] = (before + count).to(torch.int32).cuda()
        used = (before + count + page - 1) // page
        table = torch.full((n, int(used.max())), -1, dtype=torch.int32)
        table[torch.arange(table.shape[1]) < used[:, None]] = torch.randperm(int(used.sum()), generator=host).to(torch.int32)
        s["table"] = table.cuda()
        s |= _cache(case["ct"], int(used.sum()), case["kv_heads"], page, case["d"], gen)
        s["q"] = (2 * normal(int(count.sum()), case["heads"], case["d"])).to(torch.float16 if case["act"] == "f16" else torch.float32)
        s["sinks"] = normal(case["heads"]) if case["sinks"] else None
        s["scale"] = case["d"] ** -0.5
    else:
        n, vocab = case["seqs"], case["vocab"]
        count = torch.tensor(_drafted(case))
        rows = int((count + 1).sum())
        s["start"] = torch.cat([torch.zeros(1, dtype=torch.long), (count + 1).cumsum(0)]).to(torch.int32).cuda()
        s["logits"] = 3.5 * normal(rows, vocab)
        s["accept_u"] = torch.rand(rows, device="cuda", generator=gen)
        s["sample_u"] = torch.rand(n, device="cuda", generator=gen)
        # every seventh request is greedy
        temp = 0.5 + 0.7 * torch.rand(n, generator=host)
        temp[6::7] = 0.0
        s["temp"] = temp.cuda()
        if case["drafter"]:
            # a small model's logits, near the target's; its tokens are drawn from them (a greedy request's are its greatest)
            s["draft_logits"] = s["logits"] + 0.7 * normal(rows, vocab)
            t = s["temp"].repeat_interleave((count + 1).cuda(), output_size=rows)[:, None]
            noise = -torch.log(-torch.log(torch.rand((rows, vocab), device="cuda", generator=gen).clamp(1e-9, 1 - 1e-7)))
            s["draft"] = torch.where(t > 0, s["draft_logits"] / t.clamp(min=1e-3) + noise, s["draft_logits"]).argmax(1).to(torch.int32)
        else:
            # tokens that were looked up: mostly the target's likeliest, now and then one of the next
            top = s["logits"].topk(4, 1).indices
            s["draft_logits"] = None
            s["draft"] = top.gather(1, (4 * torch.rand((rows, 1), device="cuda", generator=gen) ** 4).long().clamp(max=3))[:, 0].to(torch.int32).contiguous()
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def _plain_plan(s):
    case = s["case"]
    n, page, room = case["seqs"], case["page"], case["tokens"]
    table, (_, width) = s["table"].long(), s["table"].shape
    before, new = s["before"].long().clamp(min=0), s["new"].long().clamp(min=0)
    end = new.cumsum(0).clamp(max=room)
    start = torch.cat([end.new_zeros(1), end])
    new = start[1:] - start[:-1]
    length = before + new
    # pages wanted: those from the first without a position on
    have, need = (before + page - 1) // page, (length + page - 1) // page
    first = torch.cat([need.new_zeros(1), (need - have).clamp(min=0).cumsum(0)])
    i = torch.arange(width, device="cuda")
    k = first[:-1, None] + i - have[:, None]
    n_free = s["n_free"].long().clamp(min=0)
    fresh = (i >= have[:, None]) & (i < need[:, None])
    got = fresh & (k < n_free)
    page_of = torch.where(got, s["free"].long()[torch.where(got, n_free - 1 - k, 0)], -1)
    table = torch.where(fresh, page_of, table)
    t = torch.arange(room, device="cuda")
    seq = torch.searchsorted(end, t, right=True).clamp(max=n - 1)
    there = t < end[-1]
    position = torch.where(there, before[seq] + t - start[seq], 0)
    at = table[seq, (position // page).clamp(max=width - 1)]
    slot = torch.where(there & (at >= 0) & (position // page < width), at * page + position % page, -1)
    taken = got.sum()
    counts = torch.cat([n_free - taken, (first[-1] - taken).view(1), end[-1:], s["new"].long().clamp(min=0).sum().view(1) - end[-1:]])
    last = torch.where(new > 0, start[1:] - 1, -1)
    return tuple(x.int() for x in (start, length, position)) + (slot,) + tuple(x.int() for x in (last, counts, table))


def _plain_norm(s):
    x, case = s["x"], s["case"]
    if s["post"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s["post"]
    if s["gate"] is not None:
        x = x * s["gate"]
    h = s["residual"] + 0.5 * x
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * s["weight"]
    return (y.half() if case["out"] == "f16" else y), h


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


def _plain_chunk(s):
    case = s["case"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    out, row = torch.empty_like(s["q"]), 0
    for i, (count, before) in enumerate(zip(*_batch(case))):
        n = before + count
        pages = s["table"][i, :(n + page - 1) // page].long()
        k, v = (_decode(s[x][pages], None if s[x + "_scale"] is None else s[x + "_scale"][pages], s["ct"]).transpose(1, 0).flatten(1, 2)[:, :n] for x in ("k", "v"))
        q = s["q"][row:row + count].float().view(count, kv, h // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
        score = (q @ k.transpose(1, 2)).mul_(s["scale"])
        if case["softcap"]:
            score = case["softcap"] * torch.tanh(score / case["softcap"])
        own_place = before + torch.arange(count, device="cuda")[:, None]
        p = torch.arange(n, device="cuda")
        hidden = p > own_place
        if case["window"]:
            hidden = hidden | (p <= own_place - case["window"])
        score = score.view(kv, h // kv, count, n).masked_fill_(hidden, -math.inf)
        top = score.amax(-1, keepdim=True)
        sink = None
        if s["sinks"] is not None:
            sink = s["sinks"].view(kv, h // kv, 1, 1)
            top = torch.maximum(top, sink)
        w = score.sub_(top).exp_()
        total = w.sum(-1, keepdim=True)
        if sink is not None:
            total = total + torch.exp(sink - top)
        o = (w.view(kv, -1, n) @ v).view(kv, h // kv, count, d) / total
        out[row:row + count] = o.permute(2, 0, 1, 3).reshape(count, h, d).to(out.dtype)
        row += count
    return out


def _plain_verify(s):
    case = s["case"]
    n, vocab, rows = case["seqs"], case["vocab"], len(s["logits"])
    start = s["start"].long()
    count = start[1:] - start[:-1]
    seq = torch.searchsorted(start[1:], torch.arange(rows, device="cuda"), right=True)
    # sums of a hundred thousand weights, and where a random number falls among them, in 64 bits
    temp = s["temp"].double()[seq, None]
    safe = torch.where(temp > 0, temp, 1)

    def softmax(x):
        x = x.double()
        x = (x - x.amax(-1, keepdim=True)) / safe
        e = torch.exp(x)
        total = e.sum(-1, keepdim=True)
        return e / total, x - torch.log(total)
    p, log_p = softmax(s["logits"])
    token = s["draft"].long()[:, None]
    q = softmax(s["draft_logits"])[0] if s["draft_logits"] is not None else torch.zeros_like(p).scatter_(1, token, 1.0)
    index = torch.arange(vocab, device="cuda")
    best = torch.where(s["logits"] == s["logits"].amax(-1, keepdim=True), index, vocab).amin(-1)
    ok = torch.where(temp[:, 0] > 0, s["accept_u"].double() * q.gather(1, token)[:, 0] < p.gather(1, token)[:, 0], best == token[:, 0])
    place = torch.arange(rows, device="cuda") - start[seq]
    last = place == count[seq] - 1
    # the first row of each request that is refused, or its last one
    stop = torch.full((n,), rows, device="cuda").scatter_reduce_(0, seq, torch.where(ok & ~last, rows, place), "amin")
    at = start[:-1] + stop
    w = torch.where(last[at, None], p[at], (p[at] - q[at]).clamp(min=0))
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[at])
    upto = w.cumsum(-1)
    drawn = torch.where((upto > s["sample_u"].double()[:, None] * upto[:, -1:]) & (w > 0), index, vocab).amin(-1)
    final = torch.where(s["temp"] > 0, drawn, best[at])
    tokens = torch.where(place < stop[seq], token[:, 0], torch.where(place == stop[seq], final[seq], -1))
    log_p = torch.where(tokens >= 0, log_p.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0)
    return tokens.int(), stop.int(), log_p.float()


def _own(s):
    from kraken_b200 import capi
    case, kind = s["case"], s["case"]["kind"]
    if kind == "plan":
        return tuple(capi.step_plan(s["before"], s["new"], s["table"], s["free"], s["n_free"], case["page"], case["tokens"]))
    if kind == "norm":
        return capi.block_norm(s["x"], s["weight"], residual=s["residual"], post_weight=s["post"], gate=s["gate"], alpha=0.5, eps=1e-6,
                               dtype=torch.float16 if case["out"] == "f16" else torch.float32)
    if kind == "verify":
        return capi.verify_draft(s["logits"], s["start"], s["draft"], s["accept_u"], s["sample_u"], draft_logits=s["draft_logits"], temp=s["temp"])
    if "cache" not in s:   # the handle that a program keeps
        s["cache"] = capi.KvCache({"f16": capi.KV_F16, "q8": capi.KV_Q8, "q4": capi.KV_Q4}[s["ct"]], s["k"], s["v"], s["k_scale"], s["v_scale"])
    return capi.attention_chunk(s["q"], s["cache"], s["q_start"], s["kv_len"], s["table"], case["most"], scale=s["scale"], softcap=case["softcap"], window=case["window"],
                                sinks=s["sinks"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plain_plan, "norm": _plain_norm, "chunk": _plain_chunk, "verify": _plain_verify}[state["case"]["kind"]](state)


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


def _exact_plan(s, case):
    page, room = case["page"], case["tokens"]
    table, stack = s["table"].tolist(), s["free"].tolist()[:int(s["n_free"])]
    width, missing, position, slot, start, length, last = len(table[0]), 0, [], [], [0], [], []
    for r, b, c in zip(table, s["before"].tolist(), s["new"].tolist()):
        c = min(c, room - len(position))
        for i in range(-(-b // page), -(-(b + c) // page)):
            missing += not stack
            r[i] = stack.pop() if stack else -1
        for p in range(b, b + c):
            position.append(p)
            slot.append(r[p // page] * page + p % page if p // page < width and r[p // page] >= 0 else -1)
        start.append(len(position))
        length.append(b + c)
        last.append(len(position) - 1 if c > 0 else -1)
    counts = [len(stack), missing, len(position), int(s["new"].long().sum()) - len(position)]
    tail = room - len(position)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    return i32(start), i32(length), i32(position + [0] * tail), torch.tensor(slot + [-1] * tail, device="cuda"), i32(last), i32(counts), i32(table)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return _exact_plan(s, case)
    if kind == "norm":
        def unit(x, w):
            return w.double() * x / ((x ** 2).sum(-1, keepdim=True) / case["n"] + 1e-6).sqrt()
        x = s["x"].double() if s["post"] is None else unit(s["x"].double(), s["post"])
        h = s["residual"].double() + x / 2 * (1.0 if s["gate"] is None else s["gate"].double())
        return unit(h, s["weight"]), h
    if kind == "chunk":
        out, row, group = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, case["heads"] // case["kv_heads"]
        for i, (count, before) in enumerate(zip(*_batch(case))):
            p = torch.arange(before + count, device="cuda")
            page, slot = s["table"][i].long()[p // case["page"]], p % case["page"]
            k, v = _values(s, "k", page, slot), _values(s, "v", page, slot)
            ago = torch.arange(before, before + count, device="cuda")[:, None] - p
            seen = (ago >= 0) & (ago < (case["window"] or before + count))
            for head in range(case["heads"]):
                z = s["q"][row:row + count, head].double() @ k[:, head // group].T * s["scale"]
                if case["softcap"]:
                    z = torch.tanh(z / case["softcap"]) * case["softcap"]
                z = torch.where(seen, z, -math.inf)
                if s["sinks"] is not None:
                    z = torch.cat([z, s["sinks"][head].double().expand(count, 1)], 1)
                out[row:row + count, head] = torch.softmax(z, 1)[:, :before + count] @ v[:, head // group]
            row += count
        return out
    tokens, accepted = [], []
    start, draft, temp = s["start"].tolist(), s["draft"].tolist(), s["temp"].double().tolist()
    for i in range(case["seqs"]):
        rows = range(start[i], start[i + 1])
        for j, r in enumerate(rows):
            x = s["logits"][r].double()
            token = draft[r]
            if temp[i] <= 0:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0, 0])] = 1.0
                q = torch.zeros_like(p)
                q[token] = 1.0
            else:
                p = torch.softmax(x / temp[i], 0)
                q = torch.zeros_like(p)
                if s["draft_logits"] is None:
                    q[token] = 1.0
                else:
                    q = torch.softmax(s["draft_logits"][r].double() / temp[i], 0)
            bonus = r == rows[-1]
            if not bonus and float(s["accept_u"][r]) * float(q[token]) < float(p[token]):
                tokens.append(token)
                continue
            w = p if bonus else torch.relu(p - q)
            if temp[i] <= 0:
                w = p
            sums = torch.cumsum(w, 0)
            tokens.append(int((sums > float(s["sample_u"][i]) * float(sums[-1])).nonzero()[0, 0]))
            tokens += [-1] * (len(rows) - j - 1)
            accepted.append(j)
            break
    # the target's probabilities of what came out, at the request's temperature (a greedy one's: 1)
    log_p = [0.0 if t < 0 else float(torch.log_softmax(s["logits"][r].double() / (temp[i] if temp[i] > 0 else 1.0), 0)[t])
             for i in range(case["seqs"]) for r, t in zip(range(start[i], start[i + 1]), tokens[start[i]:start[i + 1]])]
    return (torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.tensor(accepted, dtype=torch.int32, device="cuda"),
            torch.tensor(log_p, dtype=torch.float64, device="cuda"))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        # a position and a slot for each place of the buffer, a page number a page of new tokens, the requests' numbers
        return {"bytes": 12 * case["tokens"] + 8 * min(case["tokens"], case["seqs"] * case["most"]) // case["page"] + 20 * case["seqs"], "flops": 0}
    if kind == "norm":
        values = case["rows"] * case["n"]
        return {"bytes": values * (12 + (4 if case["out"] == "f32" else 2) + 4 * (case["gate"] == "rows")) + 4 * case["n"] * (1 + case["post"] + (case["gate"] == "vector")),
                "flops": values * (6 + 4 * case["post"])}
    if kind == "verify":
        rows = sum(_drafted(case)) + case["seqs"]
        return {"bytes": 4 * case["vocab"] * (rows + (rows - case["seqs"]) * case["drafter"]) + 16 * rows + 16 * case["seqs"], "flops": 3 * rows * case["vocab"] * (1 + case["drafter"])}
    row = case["kv_heads"] * {"f16": 2 * case["d"], "q8": case["d"] + case["d"] // 16, "q4": case["d"] // 2 + case["d"] // 16}[case["ct"]]
    positions = pairs = tokens = 0
    for c, b in zip(*_batch(case)):
        w = case["window"] or b + c
        positions += min(b + c, w + c - 1)
        # token i sees min(b + i + 1, w) positions
        rising = max(0, min(c, w - b))
        pairs += rising * b + rising * (rising + 1) // 2 + (c - rising) * w
        tokens += c
    return {"bytes": 2 * positions * row + (8 if case["act"] == "f32" else 4) * tokens * case["heads"] * case["d"], "flops": 4 * pairs * case["heads"] * case["d"]}

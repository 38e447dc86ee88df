"""Prompts in chunks and then a verifying step, through the library: the step's plan, projections, head norm and rotation, cache, attention of the chunks, what lies
between blocks, head, verification; against the same in 64 bits. The new calls through the backend object, and their refusals by the binding on a GPU."""
import numpy as np
import pytest

from attn_plain import attention, decode, encode
from test_gpu_verify_draft import plain as plain_verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,graph", [(0, False), (1, False), (2, False), (0, True)])
def test_chunks_and_a_verifying_step(cuda, oracle, kind, graph):
    """Three requests, prompts of 130, 5 and 61 tokens in three unlike steps, two layers, and a step of drafted tokens. graph: the steps are replays of one graph, whose
    batch has as many tokens as the largest."""
    import torch
    from kraken_b200 import synth
    hid, heads, kv, d, page, vocab, wt, eps = 512, 8, 2, 64, 16, 2000, synth.Q8_0, 1e-6
    steps = [(50, 5, 9), (63, 0, 1), (17, 0, 51), (4, 1, 3)]
    room, lens = 68, np.sum(steps, 0)
    rng = np.random.default_rng(kind)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    sizes = {"q": (heads * d, hid), "k": (kv * d, hid), "v": (kv * d, hid), "o": (hid, heads * d), "head": (vocab, hid)}
    w = [{n: synth.weights(wt, *s, synth.BASE_SEED, stream=10 * layer + i) for i, (n, s) in enumerate(sizes.items())} for layer in range(2)]
    full = [{n: oracle.dequant_rows(a[n], wt, *s).astype(np.float64) for n, s in sizes.items()} for a in w]
    wd = [{n: dev(a[n]) for n in sizes} for a in w]
    w_in, w_post, w_next = ([rng.uniform(0.5, 1.5, hid).astype(np.float32) for _ in range(2)] for _ in range(3))
    freq = (10000.0 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    x = [rng.standard_normal((n, hid)).astype(np.float32) for n in lens]   # of the requests' tokens

    caches = [cuda.KvCache.empty(kind, 30, kv, page, d) for _ in range(2)]
    table = torch.full((3, 10), -1, dtype=torch.int32, device="cuda")
    free, n_free = i32(rng.permutation(30)), i32([30])
    before, new, xd = i32([0, 0, 0]), i32([0, 0, 0]), torch.zeros((room, hid), device="cuda")
    freq_d, norms = dev(freq), [[dev(a) for a in b] for b in (w_in, w_post, w_next)]

    def mat(y, layer, n):
        return torch.cat([cuda.gemv(y[i:i + 8], wd[layer][n], wt, *sizes[n]) for i in range(0, len(y), 8)])

    def step():
        plan = cuda.step_plan(before, new, table, free, n_free, page, room)
        y, h = cuda.block_norm(xd, norms[0][0], eps=eps)
        kept = []
        for layer in range(2):
            q, k, v = (mat(y, layer, n).view(room, -1, d) for n in "qkv")
            q, k = cuda.qk_norm_rope(q, k, plan.positions, freq_d, eps=eps)
            cuda.kv_append(caches[layer], k, v, plan.slots)
            o = torch.zeros_like(q)
            cuda.attention_chunk(q, caches[layer], plan.q_start, plan.kv_len, plan.page_table, 64, out=o)
            y, h = cuda.block_norm(mat(o.view(room, -1), layer, "o"), norms[2][layer], residual=h, post_weight=norms[1][layer], eps=eps)
            kept.append((k, v, h))
        return plan, mat(y, 1, "head"), kept

    def inputs(c):
        new.copy_(i32(c))
        n_free.fill_(left)
        xd.zero_()
        xd[:sum(c)] = dev(np.concatenate([x[s][at[s]:at[s] + c[s]] for s in range(3)]))

    captured, left, at, done = None, 30, np.zeros(3, int), []
    for c in steps:
        inputs(c)
        if not graph:
            got = step()
        else:
            if captured is None:
                keep = [t.clone() for t in (table, n_free)]
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                torch.cuda.current_stream().wait_stream(side)
                table.copy_(keep[0]), n_free.copy_(keep[1])
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    outs = step()
            captured.replay()
            got = outs
        torch.cuda.synchronize()
        plan, logits, kept = got
        counts = plan.counts.tolist()
        left = counts[0]
        assert counts[1:] == [0, sum(c), 0] and left == 30 - sum(-(-int(n) // page) for n in at + c)
        rows = np.cumsum((0,) + c)
        assert plan.q_start.tolist() == rows.tolist() and plan.kv_len.tolist() == (at + c).tolist()
        done.append((rows, [t.cpu().numpy().astype(np.float64) for t in (logits, *(t for layer in kept for t in layer))]))
        at += c
        before.copy_(i32(at))

    # ---- in 64 bits, a request at a time, over what the caches were given
    norm = lambda z, g: z / np.sqrt((z ** 2).mean(-1, keepdims=True) + eps) * g  # noqa: E731
    for s in range(3):
        got = [np.concatenate([t[i][r[s]:r[s + 1]] for r, t in done]) for i in range(7)]
        h = x[s].astype(np.float64)
        y = norm(h, w_in[0])
        turn = np.exp(1j * np.arange(lens[s])[:, None] * freq.astype(np.float64))[:, None]
        for layer in range(2):
            q, k, v = ((y @ full[layer][n].T).reshape(lens[s], -1, d) for n in "qkv")

            def rope(z):
                z = norm(z, 1.0)
                z = (z[..., :d // 2] + 1j * z[..., d // 2:]) * turn
                return np.concatenate([z.real, z.imag], -1)
            mine = got[1 + 3 * layer:4 + 3 * layer]
            for a, b in ((mine[0], rope(k)), (mine[1], v)):
                assert np.linalg.norm(a - b) <= (1 + layer) * 2e-5 * np.linalg.norm(b)
            rows = [decode(*encode(a.astype(np.float32), kind), kind) for a in mine[:2]]
            o, _ = attention(rope(q).astype(np.float32), *rows, np.tril(np.ones((lens[s], lens[s]), bool)), d ** -0.5)
            h = h + norm(o.reshape(lens[s], -1) @ full[layer]["o"].T, w_post[layer])
            y = norm(h, w_next[layer])
            assert np.linalg.norm(mine[2] - h) <= (1 + layer) * 2e-5 * np.linalg.norm(h)
        fl = y @ full[1]["head"].T
        assert np.linalg.norm(got[0] - fl) <= 4e-5 * np.linalg.norm(fl)

    # ---- the drafted tokens of the last step: requests' rows, the last of each for the token behind them
    n = sum(steps[-1])
    start, z = np.cumsum((0,) + steps[-1]), done[-1][1][0][:n].astype(np.float32)
    draft = z.argmax(1).astype(np.int32)
    draft[1] = (draft[1] + 1) % vocab
    au, su, temp = rng.random(n).astype(np.float32) * 1e-3, rng.random(3).astype(np.float32), np.array([0.7, 0.0, 1.3], np.float32)
    out = cuda.verify_draft(dev(z), plan.q_start, dev(draft), dev(au), dev(su), temp=dev(temp))
    want = plain_verify(z, start, draft, au, su, temp=temp)
    assert (out[0].cpu().numpy() == want[0]).all() and (out[1].cpu().numpy() == want[1]).all()
    assert np.abs(out[2].cpu().numpy() - want[2]).max() <= 1e-5 * (1 + np.abs(want[2]).max())
    assert cuda.device_status() == 0


def test_through_the_backend_object(cuda):
    """The members of the backend, on its own stream and workspace, give what the functions give."""
    import torch
    torch.manual_seed(1)
    heads, kv, d, page, total, n_q = 8, 2, 64, 16, 3000, 300
    f = lambda *s: torch.randn(s, device="cuda")  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    p = lambda t: t.data_ptr()  # noqa: E731
    cache = cuda.KvCache.empty(cuda.KV_F16, total // page + 1, kv, page, d)
    quants = cuda.KvCache.empty(cuda.KV_Q8, total // page + 1, kv, page, d)
    fill = f(2, total, kv, d)
    for c in (cache, quants):
        cuda.kv_append(c, fill[0], fill[1], torch.arange(total, device="cuda"))
    q, table = f(n_q, heads, d), torch.arange(total // page + 1, dtype=torch.int32, device="cuda").view(1, -1)
    start, length = i32(0, n_q), i32(total)
    a_want = [cuda.attention_chunk(q, c, start, length, table, n_q) for c in (cache, quants)] + [cuda.attention_chunk(q.half(), quants, start, length, table, n_q)]
    free = torch.arange(50, dtype=torch.int32, device="cuda").flip(0).contiguous()
    lens = i32(5, 0, 40), i32(20, 1, 0)
    tables = [torch.full((3, 5), -1, dtype=torch.int32, device="cuda") for _ in range(2)]
    n_free = [i32(50), i32(50)]
    plan = cuda.step_plan(*lens, tables[0], free, n_free[0], page, 30)
    x, r, gain = f(7, 500), f(7, 500), f(500)
    n_want = cuda.block_norm(x, gain, residual=r)
    z, draft, au, su = f(6, 1000), i32(1, 2, 3, 4, 5, 6), torch.rand(6, device="cuda"), torch.rand(2, device="cuda")
    rows = i32(0, 4, 6)
    v_want = cuda.verify_draft(z, rows, draft, au, su)

    be = cuda.Backend(0)
    torch.cuda.synchronize()
    a_got = [torch.zeros_like(t) for t in a_want]
    half = q.half()
    torch.cuda.synchronize()
    att = cuda.Attention(q_start=p(start), kv_len=p(length), page_table=p(table), q_stride=heads * d, out_stride=heads * d, n_seq=1, n_heads=heads, max_q=n_q,
                         table_width=table.shape[1], scale=d ** -0.5)
    be.attention_chunk(p(a_got[0]), 0, p(q), 0, cache.struct, att)
    be.attention_chunk(p(a_got[1]), 0, p(q), 0, quants.struct, att)
    be.attention_chunk(p(a_got[2]), 1, p(half), 1, quants.struct, att)
    got = cuda.StepPlan(*(torch.zeros_like(t) for t in plan[:6]), tables[1])
    n_got, v_got = [torch.zeros_like(t) for t in n_want], [torch.zeros_like(t) for t in v_want]
    torch.cuda.synchronize()
    be.step_plan(cuda.Step(kv_before=p(lens[0]), n_new=p(lens[1]), page_table=p(tables[1]), free_pages=p(free), n_free=p(n_free[1]), q_start=p(got.q_start), kv_len=p(got.kv_len),
                           positions=p(got.positions), slots=p(got.slots), last=p(got.last), counts=p(got.counts), n_seq=3, table_width=5, page_size=page, free_cap=50, max_tok=30))
    be.block_norm(p(n_got[0]), p(n_got[1]), p(x), cuda.Norm(residual=p(r), weight=p(gain), rows=7, n=500, x_stride=500, residual_stride=500, h_stride=500, y_stride=500, alpha=1.0,
                                                            eps=1e-6))
    be.verify_draft(p(v_got[0]), p(v_got[1]), p(v_got[2]), p(z), cuda.Verify(row_start=p(rows), draft=p(draft), accept_u=p(au), sample_u=p(su), n_rows=6, n_vocab=1000, stride=1000,
                                                                             n_seq=2))
    be.sync()
    for got_all, want_all in ((a_got, a_want), (got, plan), (n_got, n_want), (v_got, v_want)):
        for g, want in zip(got_all, want_all):
            assert (g == want).all()
    be.close()


def test_bindings_check_shapes(cuda):
    import torch
    f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = cuda.KvCache.empty(cuda.KV_Q8, 4, 2, 16, 64)
    ok = dict(q=f(1, 4, 64), cache=c, q_start=i32(0, 1), kv_len=i32(3), page_table=i32(0).view(1, 1), max_q=1)
    refused = (ValueError, TypeError, cuda.KrkCudaError)
    before = cuda.launch_count()
    for bad in (dict(q=f(1, 3, 64)), dict(q=f(1, 4, 32)), dict(q=f(1, 64, 4).transpose(1, 2)), dict(q=f(1, 4, 64).double()), dict(q=f(1, 4, 64).bfloat16()),
                dict(q=f(1, 4, 64).half(), out=f(1, 4, 64)), dict(q_start=i32(0, 1, 2)), dict(kv_len=i32(3, 3)), dict(kv_len=torch.tensor([3], device="cuda")), dict(page_table=i32(0)),
                dict(sinks=f(3)), dict(out=f(2, 4, 64)), dict(max_q=-1), dict(window=-1), dict(max_kv_len=17), dict(workspace=f(3)), dict(kv_len=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(refused):
            cuda.attention_chunk(**{**ok, **bad})
    ok = dict(kv_before=i32(1, 2), n_new=i32(3, 4), page_table=torch.zeros((2, 3), dtype=torch.int32, device="cuda"), free_pages=i32(1, 2, 3), n_free=i32(3), page_size=16, max_tok=9)
    for bad in (dict(kv_before=i32(1)), dict(n_new=i32(1, 2, 3)), dict(n_new=torch.zeros(2, dtype=torch.long, device="cuda")), dict(page_table=i32(1, 2)), dict(n_free=i32(1, 2)),
                dict(page_size=0), dict(max_tok=-1), dict(free_pages=f(3)), dict(n_free=torch.zeros(1, dtype=torch.int32)), dict(out=(i32(1), i32(1)))):
        with pytest.raises(refused):
            cuda.step_plan(**{**ok, **bad})
    ok = dict(x=f(2, 8), weight=f(8), residual=f(2, 8))
    for bad in (dict(x=f(8)), dict(x=f(2, 8).half()), dict(weight=f(7)), dict(residual=f(2, 9)), dict(residual=f(3, 8)), dict(gate=f(9)), dict(gate=f(3, 8)), dict(post_weight=f(7)),
                dict(eps=-1.0), dict(h_out=f(2, 9)), dict(out=f(1, 8)), dict(dtype=torch.float16, out=f(2, 8)), dict(dtype=torch.bfloat16), dict(x=f(2, 16)[:, ::2]), dict(residual=torch.zeros(2, 8))):
        with pytest.raises(refused):
            cuda.block_norm(**{**ok, **bad})
    ok = dict(logits=f(4, 10), row_start=i32(0, 2, 4), draft=i32(1, 2, 3, 4), accept_u=f(4), sample_u=f(2))
    for bad in (dict(logits=f(4, 10).half()), dict(logits=f(40)), dict(row_start=f(3)), dict(draft=i32(1, 2, 3)), dict(accept_u=f(3)), dict(sample_u=f(3)), dict(temp=f(3)),
                dict(draft_logits=f(4, 11)), dict(draft_logits=f(3, 10)), dict(draft_temp=f(1)), dict(tokens=f(4)), dict(n_accepted=i32(1)), dict(logprob=f(3)),
                dict(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda")), dict(sample_u=torch.zeros(2))):
        with pytest.raises(refused):
            cuda.verify_draft(**{**ok, **bad})
    assert cuda.launch_count() == before

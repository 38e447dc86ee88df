"""A verifying step of drafted tokens through the library, end to end: projections, head norm and rotation, cache, attention, output
projection, head, penalties, ranking; against the same step in 64 bits. And the binding's refusals on a GPU."""
import numpy as np
import pytest

from attn_plain import attention, decode, encode, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_verifying_step(cuda, oracle, kind):
    import torch
    from kraken_b200 import synth
    hid, heads, kv, d, page, vocab, wt = 512, 8, 2, 64, 16, 2000, synth.Q8_0
    n_q, context = 5, 203   # five drafted tokens after a context of 203
    rng = np.random.default_rng(kind)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    sizes = {"q": (heads * d, hid), "k": (kv * d, hid), "v": (kv * d, hid), "o": (hid, heads * d), "head": (vocab, hid)}
    w = {n: synth.weights(wt, *s, synth.BASE_SEED, stream=i) for i, (n, s) in enumerate(sizes.items())}
    full = {n: oracle.dequant_rows(w[n], wt, *s).astype(np.float64) for n, s in sizes.items()}
    x = rng.standard_normal((n_q, hid)).astype(np.float32)
    wq, wk = (rng.uniform(0.5, 1.5, d).astype(np.float32) for _ in range(2))
    freq = (10000.0 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    masks = [1, 3, 5, 11, 21]
    pos = np.array([context + bin(m).count("1") - 1 for m in masks], np.int32)
    total = context + n_q
    pages = (total + page - 1) // page
    table = rng.permutation(pages + 3)[:pages].astype(np.int32)
    at = np.arange(total)
    slots = table[at // page].astype(np.int64) * page + at % page
    old = [rng.standard_normal((context, kv, d)).astype(np.float32) for _ in range(2)]

    cache = cuda.KvCache.empty(kind, pages + 3, kv, page, d)
    cuda.kv_append(cache, dev(old[0]), dev(old[1]), dev(slots[:context]))
    xd = dev(x)
    q, k, v = (cuda.gemv(xd, dev(w[n]), wt, *sizes[n]).view(n_q, -1, d) for n in "qkv")
    q, k = cuda.qk_norm_rope(q, k, dev(pos), dev(freq), dev(wq), dev(wk), eps=1e-6)
    cuda.kv_append(cache, k, v, dev(slots[context:]))
    o = cuda.attention_tree(q, cache, dev(np.array([0, n_q], np.int32)), dev(np.array([total], np.int32)), dev(table[None]), n_q,
                            dev(np.array(masks, np.int64)))
    y = xd.clone()
    cuda.gemv(o.view(n_q, -1), dev(w["o"]), wt, *sizes["o"], out=y, accumulate=True)
    logits = cuda.gemv(y, dev(w["head"]), wt, *sizes["head"])
    hist = rng.integers(0, vocab, (n_q, 30)).astype(np.int32)
    rep = np.full(n_q, 1.3, np.float32)
    adjusted = cuda.logits_adjust(logits, hist=dev(hist), rep=dev(rep))
    ids = [cuda.logits_topk(adjusted[i], 4)[0].cpu().numpy() for i in range(n_q)]

    def rope(z, wz):
        z = z / np.sqrt((z ** 2).mean(-1, keepdims=True) + 1e-6) * wz
        t = np.exp(1j * pos.astype(np.float64)[:, None] * freq.astype(np.float64))[:, None]
        c = (z[..., :d // 2] + 1j * z[..., d // 2:]) * t
        return np.concatenate([c.real, c.imag], -1)
    x64 = x.astype(np.float64)
    fq, fk, fv = ((x64 @ full[n].T).reshape(n_q, -1, d) for n in "qkv")
    fq, fk = rope(fq, wq), rope(fk, wk)
    # what the cache holds of the new keys and values is the quants of the library's own (a rounding may fall either way)
    rows = [np.concatenate([decode(*encode(a, kind), kind), decode(*encode(b.cpu().numpy(), kind), kind)]) for a, b in ((old[0], k), (old[1], v))]
    for got, want in ((q, fq), (k, fk), (v, fv)):
        assert np.linalg.norm(got.cpu().numpy() - want) <= 1e-5 * np.linalg.norm(want)
    fo, _ = attention(fq.astype(np.float32), *rows, visible(masks, n_q, total), d ** -0.5)
    fy = x64 + fo.reshape(n_q, -1) @ full["o"].T
    fl = fy @ full["head"].T
    for got, want in ((o, fo), (y, fy), (logits, fl)):
        assert np.linalg.norm(got.cpu().numpy() - want) <= 2e-5 * np.linalg.norm(want)
    for i in range(n_q):
        z = fl[i].copy()
        once = np.unique(hist[i])
        z[once] = np.where(z[once] > 0, z[once] / 1.3, z[once] * 1.3)
        best = np.argsort(-z)[:5]
        if np.min(-np.diff(z[best])) > 1e-3 * np.abs(z).max():   # (no near tie)
            assert (ids[i] == best[:4]).all()


def test_bindings_check_shapes(cuda):
    import torch
    f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = cuda.KvCache.empty(cuda.KV_Q8, 4, 2, 16, 64)
    ok = dict(q_start=i32(0, 1), kv_len=i32(3), page_table=i32(0).view(1, 1), max_q=1)
    before = cuda.launch_count()
    for bad in (dict(q=f(1, 3, 64)), dict(q=f(1, 4, 32)), dict(q=f(1, 64, 4).transpose(1, 2)), dict(q=f(1, 4, 64).half()), dict(q_start=i32(0, 1, 2)), dict(kv_len=i32(3, 3)),
                dict(kv_len=torch.tensor([3], device="cuda")), dict(page_table=i32(0)), dict(tree=i32(1)), dict(tree=torch.zeros(2, dtype=torch.long, device="cuda")),
                dict(sinks=f(3)), dict(out=f(2, 4, 64)), dict(max_q=65), dict(window=10), dict(max_kv_len=17), dict(workspace=f(3)), dict(kv_len=torch.zeros(1, dtype=torch.int32))):
        a = {**dict(q=f(1, 4, 64), cache=c), **ok, **bad}
        with pytest.raises((ValueError, cuda.KrkCudaError)):
            cuda.attention_tree(**a)
    big = cuda.KvCache.empty(cuda.KV_Q8, 100, 2, 16, 64)
    with pytest.raises(cuda.KrkCudaError, match="workspace"):
        cuda.attention_tree(f(1, 4, 64), big, **{**ok, "page_table": torch.zeros((1, 100), dtype=torch.int32, device="cuda")},
                            workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    k = f(3, 2, 64)
    slots = torch.zeros(3, dtype=torch.long, device="cuda")
    for a in ((f(3, 2, 32), k, slots), (k, f(2, 2, 64), slots), (k, k, slots[:2]), (k, k, slots.int()), (k, k.half(), slots), (k.transpose(0, 1), k, slots)):
        with pytest.raises(ValueError):
            cuda.kv_append(c, *a)
    for a in (dict(k=f(2, 2, 64)), dict(k=f(3, 2, 32)), dict(pos=i32(1)), dict(inv_freq=f(33)), dict(inv_freq=f(3)), dict(q_weight=f(63)), dict(q_out=f(3, 2, 65)[..., 1:]), dict(eps=-1.0)):
        with pytest.raises((ValueError, cuda.KrkCudaError)):
            cuda.qk_norm_rope(**{**dict(q=f(3, 2, 64), k=f(3, 2, 64), pos=i32(1, 2, 3), inv_freq=f(32)), **a})
    for a in (dict(hist=i32(1, 2)), dict(hist=i32(1, 2).view(1, 2)), dict(rep=f(3)), dict(bias=f(2, 1)), dict(bias=f(2, 1), bias_ids=i32(1, 2, 3, 4).view(2, 2)),
              dict(mask=i32(1, 1).view(2, 1)), dict(out=f(2, 99)), dict(mask_row=i32(0))):
        with pytest.raises((ValueError, cuda.KrkCudaError)):
            cuda.logits_adjust(f(2, 100), **a)
    assert cuda.launch_count() == before


def test_through_the_backend_object(cuda):
    """The members of the backend, on its own stream and workspace, give what the functions give."""
    import torch
    rng = np.random.default_rng(4)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    heads, kv, d, page, n_q, total = 8, 2, 64, 16, 4, 2000
    q, k, v = (dev(rng.standard_normal((n, h, d)).astype(np.float32)) for n, h in ((n_q, heads), (total, kv), (total, kv)))
    pos, freq = dev(np.arange(n_q, dtype=np.int32) + total - n_q), dev(rng.random(d // 2).astype(np.float32))
    slots = torch.randperm(total // page * page, device="cuda")
    table = torch.arange(total // page, dtype=torch.int32, device="cuda").view(1, -1)
    start, length = dev(np.array([0, n_q], np.int32)), dev(np.array([total], np.int32))
    hist, rep = dev(rng.integers(0, 500, (n_q, 20)).astype(np.int32)), dev(np.full(n_q, 1.2, np.float32))
    logits = dev(rng.standard_normal((n_q, 500)).astype(np.float32))
    want_cache, cache = (cuda.KvCache.empty(cuda.KV_Q8, total // page, kv, page, d) for _ in range(2))
    q_want, _ = cuda.qk_norm_rope(q, None, pos, freq)
    cuda.kv_append(want_cache, k, v, slots)
    want = cuda.attention_tree(q_want, want_cache, start, length, table, n_q)
    k_want, v_want = cuda.kv_read(want_cache, slots[:50])
    l_want = cuda.logits_adjust(logits, hist, rep=rep)

    be = cuda.Backend(0)
    torch.cuda.synchronize()
    q_got, got, k_got, v_got, l_got = (torch.zeros_like(t) for t in (q_want, want, k_want, v_want, l_want))
    p = lambda t: t.data_ptr()  # noqa: E731
    rope = cuda.Rope(pos=p(pos), inv_freq=p(freq), n_tok=n_q, q_stride=heads * d, q_out_stride=heads * d, n_heads=heads, head_dim=d, rot_dim=d, norm=1, eps=1e-6)
    be.qk_norm_rope(p(q_got), None, p(q), None, rope)
    be.kv_append(cache.struct, p(k), p(v), kv * d, kv * d, p(slots), total)
    be.attention_tree(p(got), p(q_got), cache.struct, cuda.Attention(q_start=p(start), kv_len=p(length), page_table=p(table), q_stride=heads * d, out_stride=heads * d,
                                                                     n_seq=1, n_heads=heads, max_q=n_q, table_width=total // page, scale=d ** -0.5))
    be.kv_read(cache.struct, p(k_got), p(v_got), p(slots), 50)
    be.logits_adjust(p(l_got), p(logits), cuda.Adjust(n_rows=n_q, n_vocab=500, stride=500, out_stride=500, hist=p(hist), hist_n=20, hist_stride=20, rep=p(rep)))
    be.sync()
    for a, b in ((q_got, q_want), (got, want), (k_got, k_want), (v_got, v_want), (l_got, l_want)):
        assert (a == b).all()
    be.close()

"""Norm and rotation of query and key heads, and the paged cache: against plain forms in 64 bits."""
import numpy as np
import pytest

from attn_plain import decode, encode

pytestmark = pytest.mark.gpu
KINDS = {"f16": 0, "q8": 1, "q4": 2}


def rope_plain(x, pos, inv_freq, w, norm, eps, interleaved):
    x = x.astype(np.float64)
    if norm:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * (1.0 if w is None else w.astype(np.float64))
    size = np.abs(x)
    rot = 0 if inv_freq is None else 2 * len(inv_freq)
    if rot:
        z = np.exp(1j * (pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)))[:, None]
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        y = (x[..., a] + 1j * x[..., b]) * z
        both = np.abs(x[..., a]) + np.abs(x[..., b])
        x, size = x.copy(), size.copy()
        x[..., a], x[..., b], size[..., a], size[..., b] = y.real, y.imag, both, both
    # the sum of squares, its root and quotient, two products: 16 halves of a step; the angle is rounded to 24 bits of half a turn, its sine
    # and cosine are good to 2^-22, two products and a sum: 2^-21 of the pair's sizes
    return x, size * (16 * 2.0 ** -24 + (2.0 ** -21 + np.pi * 2.0 ** -24 if rot else 0.0))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,d,rot,norm,far", [
    (1, 32, 8, 128, 128, True, 10), (1, 1, 1, 8, 8, True, 5), (7, 28, 4, 256, 64, True, 1000000), (3, 5, 5, 64, 64, False, 2000), (300, 14, 2, 96, 48, True, 131072),
    (65, 3, 1, 80, 0, True, 9), (2, 4, 0, 128, 32, True, 2 ** 31 - 5), (700, 32, 8, 128, 128, True, 40000), (5, 2, 2, 24, 16, False, 77)])
def test_norm_and_rotation(cuda, interleaved, tokens, heads, kv, d, rot, norm, far):
    import torch
    rng = np.random.default_rng(tokens + d)
    q, k = (rng.standard_normal((tokens, h, d)).astype(np.float32) * 3 for h in (heads, kv))
    pos = (far - rng.integers(0, min(far, 1000) + 1, tokens)).astype(np.int32)
    freq = (10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1))).astype(np.float32) if rot else None
    wq, wk = (rng.uniform(0.5, 1.5, d).astype(np.float32) for _ in range(2))
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    # rows inside a wider tensor
    wide = torch.zeros((tokens, (heads + kv) * d + 12), device="cuda")
    qd, kd = wide[:, :heads * d].unflatten(1, (heads, d)), wide[:, heads * d:(heads + kv) * d].unflatten(1, (kv, d)) if kv else None
    qd.copy_(dev(q))
    if kv:
        kd.copy_(dev(k))
    got = cuda.qk_norm_rope(qd, kd, dev(pos), dev(freq), dev(wq), None, norm=norm, eps=1e-5, interleaved=interleaved)
    for y, x, w in ((got[0], q, wq), (got[1], k, None)):
        if y is None:
            assert kv == 0
            continue
        want, tol = rope_plain(x, pos, freq, w, norm, 1e-5, interleaved)
        assert (np.abs(y.cpu().numpy() - want) <= tol + 1e-30).all()
    # in place, with the keys' weights
    cuda.qk_norm_rope(qd, kd, dev(pos), dev(freq), dev(wq), dev(wk), norm=norm, eps=1e-5, interleaved=interleaved, q_out=qd, k_out=kd)
    assert (qd == got[0]).all() and (wide[:, (heads + kv) * d:] == 0).all()
    if kv:
        want, tol = rope_plain(k, pos, freq, wk, norm, 1e-5, interleaved)
        assert (np.abs(kd.cpu().numpy() - want) <= tol + 1e-30).all()


@pytest.mark.parametrize("tokens,heads,kv,d", [(475, 32, 8, 128), (592, 32, 8, 128), (600, 28, 4, 128), (1024, 32, 8, 128), (1500, 32, 8, 128), (1500, 28, 4, 64), (300, 28, 4, 256), (700, 27, 0, 96)])
def test_norm_over_runs_of_unlike_length(cuda, tokens, heads, kv, d):
    """Token counts at which the groups of lanes of one warp walk runs of heads that differ by one (148 SMs: 2 and 3 heads at 475 and 592 tokens of 40
    heads, 4 and 5 at 1024), so that one of them is through a trip of the loop earlier."""
    import torch
    rng = np.random.default_rng(tokens)
    q, k = (rng.standard_normal((tokens, h, d)).astype(np.float32) for h in (heads, kv))
    pos = np.arange(tokens, dtype=np.int32)
    freq = (10000.0 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    wq, wk = (rng.uniform(0.5, 1.5, d).astype(np.float32) for _ in range(2))
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    got = cuda.qk_norm_rope(dev(q), dev(k) if kv else None, dev(pos), dev(freq), dev(wq), dev(wk))
    for y, x, w in ((got[0], q, wq), (got[1], k, wk)):
        if y is not None:
            want, tol = rope_plain(x, pos, freq, w, True, 1e-6, False)
            assert (np.abs(y.cpu().numpy() - want) <= tol + 1e-30).all()


def test_norm_of_zeros_and_negative_positions(cuda):
    import torch
    q = torch.zeros((2, 1, 64), device="cuda")
    pos = torch.tensor([-3, 4], dtype=torch.int32, device="cuda")
    freq = torch.rand(32, device="cuda")
    assert (cuda.qk_norm_rope(q, None, pos, freq)[0] == 0).all()
    q = torch.randn((2, 1, 64), device="cuda")
    want, tol = rope_plain(q.cpu().numpy(), pos.cpu().numpy(), freq.cpu().numpy(), None, True, 1e-6, False)
    assert (np.abs(cuda.qk_norm_rope(q, None, pos, freq)[0].cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("far", [2000, 1 << 30])
def test_sines_and_cosines(cuda, far):
    """Of pairs (1, 0) nothing else is left: the f32 sine and cosine of a half turn's fraction are off by a unit in the last place at most, 2^-24 below 1;
    the angle's rest is put right with one rounding, 2^-25."""
    import torch
    rng = np.random.default_rng(far)
    pos = rng.integers(-far, far, 4096).astype(np.int32)
    freq = rng.uniform(0.0, 1.0, 64).astype(np.float32)
    q = torch.zeros((4096, 1, 128), device="cuda")
    q[..., :64] = 1
    got = cuda.qk_norm_rope(q, None, torch.from_numpy(pos).cuda(), torch.from_numpy(freq).cuda(), norm=False)[0].cpu().numpy()[:, 0]
    # (64 bits: the product of 31 and 24 bits rounds 2^-53 of it, the division by a turn, on either side, twice that)
    angle = pos.astype(np.float64)[:, None] * freq.astype(np.float64)
    tol = 1.5 * 2.0 ** -24 + np.abs(angle).max() * 2.0 ** -52
    assert np.abs(got[:, :64] - np.cos(angle)).max() <= tol and np.abs(got[:, 64:] - np.sin(angle)).max() <= tol


@pytest.mark.parametrize("heads", [1, 5])
def test_weights_of_keys_that_are_not_there(cuda, heads):
    """Heads are worked on in pairs: of an odd number of query heads the last one's partner would be the first key head."""
    import torch
    q = torch.randn((3, heads, 64), device="cuda")
    pos, freq = torch.arange(3, dtype=torch.int32, device="cuda"), torch.rand(32, device="cuda")
    want = cuda.qk_norm_rope(q, None, pos, freq)[0]
    assert torch.equal(cuda.qk_norm_rope(q, None, pos, freq, None, torch.full((64,), float("nan"), device="cuda"))[0], want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,kv,d,page", [(1, 8, 128, 16), (5, 3, 32, 48), (37, 2, 96, 16), (130, 1, 256, 64), (2500, 2, 64, 32)])
def test_append_and_read(cuda, kind, tokens, kv, d, page):
    import torch
    rng = np.random.default_rng(tokens)
    kd = KINDS[kind]
    pages = (tokens + page - 1) // page + 2
    cache = cuda.KvCache.empty(kd, pages, kv, page, d)
    k, v = (rng.standard_normal((tokens, kv, d)).astype(np.float32) * np.exp2(rng.uniform(-20, 12, (tokens, kv, 1))).astype(np.float32) for _ in range(2))
    k[0, 0, :32], v[-1, -1, -32:] = 0, 1e-9                    # a block of zeros, one whose scale is none
    k[-1, 0, :32] = 3e38 if kd else 1e6                        # beyond the scales (f16: beyond the type)
    v[0, 0, :32] = np.resize([2.0, -2.0], 32)                  # equal magnitudes of either sign
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[tokens // 2] = -1 if tokens > 2 else slots[tokens // 2]
    wide = torch.zeros((tokens, 2 * kv * d + 4), device="cuda")
    kt, vt = wide[:, :kv * d].unflatten(1, (kv, d)), wide[:, kv * d:2 * kv * d].unflatten(1, (kv, d))
    kt.copy_(torch.from_numpy(k))
    vt.copy_(torch.from_numpy(v))
    st = torch.from_numpy(slots).cuda()
    cuda.kv_append(cache, kt, vt, st)
    ok = slots >= 0
    for x, pool, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        rows, d16 = encode(x[ok], kd)
        at = slots[ok] // page, slice(None), slots[ok] % page
        got = pool.cpu().numpy()
        assert got[at].tobytes() == rows.tobytes()
        left = np.ones((pages, page), bool)
        left[at[0], at[2]] = False
        assert (got.transpose(0, 2, 1, 3)[left] == 0).all(), "rows that nobody wrote"
        if kd:
            assert np.array_equal(scale.cpu().numpy()[at], d16)   # (a block of zeros: the scale is 0 or -0, which are the same)
    gk, gv = cuda.kv_read(cache, st)
    for got, x in ((gk, k), (gv, v)):
        rows, d16 = encode(x, kd)
        want = decode(rows, d16, kd).astype(np.float32)
        want[~ok] = 0
        assert (got.cpu().numpy() == want).all()


@pytest.mark.parametrize("kind", KINDS)
def test_slots_that_are_none_or_come_twice(cuda, kind):
    import torch
    for tokens in (9, 4000):
        cache = cuda.KvCache.empty(KINDS[kind], 300, 2, 16, 64)
        k = torch.randn((tokens, 2, 64), device="cuda")
        slots = torch.randint(0, 4, (tokens,), device="cuda") * 1000 + torch.randint(0, 2 if tokens < 10 else 200, (tokens,), device="cuda")
        slots[tokens // 3], slots[tokens // 2] = 4800, -7
        cuda.kv_append(cache, k, -k, slots)
        last = {int(s): i for i, s in enumerate(slots.tolist())}
        ids = torch.tensor(sorted(s for s in last if 0 <= s < 4800), device="cuda")
        gk, gv = cuda.kv_read(cache, ids)
        want = k[[last[int(s)] for s in ids.tolist()]].cpu().numpy()
        for got, x in ((gk, want), (gv, -want)):
            assert (got.cpu().numpy() == decode(*encode(x, KINDS[kind]), KINDS[kind]).astype(np.float32)).all()
    gk, gv = cuda.kv_read(cache, torch.tensor([-1, 4800, 1 << 62, -(1 << 62)], device="cuda"))
    assert (gk == 0).all() and (gv == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [8191, 8192, 13001, 40000])
def test_long_appends_go_in_pieces(cuda, kind, tokens):
    """Whose number grows with the tokens (each piece is looked through for its own slots); of tokens of different pieces with one slot the last stays."""
    import torch
    gen = torch.Generator("cuda").manual_seed(tokens)
    cache = cuda.KvCache.empty(KINDS[kind], 700, 1, 16, 32)
    k = torch.randn((tokens, 1, 32), device="cuda", generator=gen)
    slots = torch.randint(-300, 11500, (tokens,), device="cuda", generator=gen)
    slots[0], slots[tokens // 2], slots[-1] = 77, 77, 77
    before = cuda.launch_count()
    cuda.kv_append(cache, k, -k, slots)
    assert cuda.launch_count() - before == {8191: 1, 8192: 2, 13001: 3, 40000: 10}[tokens]
    last = {s: i for i, s in enumerate(slots.tolist()) if 0 <= s < 11200}
    gk, gv = (x.cpu().numpy() for x in cuda.kv_read(cache, torch.arange(11200, device="cuda")))
    at = np.array(sorted(last))
    x = k.cpu().numpy()[[last[s] for s in at.tolist()]]
    for got, want in ((gk, x), (gv, -x)):
        assert (got[at] == decode(*encode(want, KINDS[kind]), KINDS[kind]).astype(np.float32)).all()
        assert (np.delete(got, at, 0) == 0).all()


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_infinities_and_nan_stay_in_their_block(cuda, kind):
    import torch
    cache = cuda.KvCache.empty(KINDS[kind], 1, 1, 16, 64)
    k = torch.ones((2, 1, 64), device="cuda")
    k[0, 0, 3], k[1, 0, 40] = float("nan"), float("-inf")
    cuda.kv_append(cache, k, k, torch.tensor([0, 5], device="cuda"))
    gk, gv = (x.cpu().numpy() for x in cuda.kv_read(cache, torch.tensor([0, 5], device="cuda")))
    # (127 f16(1 / 127) and -8 f16(1 / -8): the scale is rounded to 11 bits, half a step is 2^-11 of it)
    for g in (gk, gv):
        assert np.isnan(g[0, 0, :32]).all() and (abs(g[0, 0, 32:] - 1) <= 2.0 ** -11).all()
        assert (abs(g[1, 0, :32] - 1) <= 2.0 ** -11).all() and np.isnan(g[1, 0, 32:]).all()


def test_f16_keeps_infinities(cuda):
    import torch
    cache = cuda.KvCache.empty(cuda.KV_F16, 1, 1, 16, 32)
    k = torch.full((1, 1, 32), 1e30, device="cuda")
    k[0, 0, 1], k[0, 0, 2], k[0, 0, 3] = float("inf"), float("nan"), -1e30
    cuda.kv_append(cache, k, k, torch.tensor([2], device="cuda"))
    g = cuda.kv_read(cache, torch.tensor([2], device="cuda"))[0].cpu().numpy()[0, 0]
    assert g[0] == 65504 and np.isposinf(g[1]) and np.isnan(g[2]) and g[3] == -65504


def test_cache_past_32_bit_offsets(cuda):
    """Pools of more than 2^32 bytes: the last slots are where they should be, and attention reads them there."""
    import torch
    page, d, kv = 256, 256, 8
    pages = (1 << 32) // (page * d * kv * 2) + 3
    cache = cuda.KvCache.empty(cuda.KV_F16, pages, kv, page, d)
    slots = torch.tensor([pages * page - 1 - i for i in range(20)], device="cuda")
    k, v = torch.randn((20, kv, d), device="cuda"), torch.randn((20, kv, d), device="cuda")
    cuda.kv_append(cache, k, v, slots)
    gk, gv = cuda.kv_read(cache, slots)
    assert (gk == k.half().float()).all() and (gv == v.half().float()).all()
    assert int(cache.k[:-1].count_nonzero()) == 0
    one = dict(q_start=torch.tensor([0, 1], dtype=torch.int32, device="cuda"), kv_len=torch.tensor([page], dtype=torch.int32, device="cuda"),
               page_table=torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda"), max_q=1)
    q = torch.randn((1, kv, d), device="cuda")
    got = cuda.attention_tree(q, cache, **one)
    w = torch.softmax(torch.einsum("hd,hpd->hp", q[0].double(), cache.k[-1].double()) * d ** -0.5, 1)
    want = torch.einsum("hp,hpd->hd", w, cache.v[-1].double())
    assert (got[0] - want).abs().max() < 1e-5

"""Attention of chunks of prompts over a paged cache, against a plain form in 64 bits: types, head layouts, chunks from one token to hundreds, windows,
pages in any order and missing ones, rows that see nothing, infinities at positions that are not seen, strides, streams, graphs."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
KINDS = {"f16": 0, "q8": 1, "q4": 2}
ACTS = ("f32", "f16", "f32>f16")   # of q and out


class Batch:
    """Sequences over a cache whose pages lie in no order, with unused pages and rows of q behind the last sequence."""

    def __init__(self, cuda, seed, kind, d, kv, group, page, counts, lens, act="f32", q_size=2.0, spread=True):
        import torch
        self.torch, self.cuda, self.kind, self.d, self.kv, self.page, self.counts, self.lens = torch, cuda, kind, d, kv, page, counts, lens
        gen = torch.Generator("cuda").manual_seed(seed)
        used = [max(0, n + page - 1) // page for n in lens]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.table = torch.full((len(lens), max(max(used), 1) + 1), -1, dtype=torch.int32)
        at = 0
        for s, u in enumerate(used):
            self.table[s, :u] = order[at:at + u]
            at += u
        self.cache = cuda.KvCache.empty(kind, pages, kv, page, d)
        x = torch.randn((2, pages * page, kv, d), device="cuda", generator=gen)
        if spread:
            x *= 0.2 + 2.8 * torch.rand((2, pages * page, kv, 1), device="cuda", generator=gen)
        cuda.kv_append(self.cache, x[0], x[1], torch.arange(pages * page, device="cuda"))
        self.q_half, self.half = act == "f16", act.endswith("f16")
        self.q = (q_size * torch.randn((sum(counts) + 2, kv * group, d), device="cuda", generator=gen)).to(torch.float16 if self.q_half else torch.float32)

    def args(self):
        i32 = lambda x: self.torch.tensor(x, dtype=self.torch.int32, device="cuda")  # noqa: E731
        return dict(q_start=i32([0] + np.cumsum(self.counts).tolist()), kv_len=i32(self.lens), page_table=self.table.cuda(), max_q=max(max(self.counts), 1))

    def want(self, scale, softcap=0.0, window=0, sinks=None, max_kv_len=0):
        from chunk_plain import attention, decoded, seen_of
        torch = self.torch
        out, tol = (torch.zeros(self.q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
        row = 0
        for s, (c, n) in enumerate(zip(self.counts, self.lens)):
            p = torch.arange(max(n, 0), device="cuda")
            page = self.table.cuda()[s, (p // self.page).clamp(max=self.table.shape[1] - 1)].long()
            there = (page >= 0) & (page < self.cache.n_pages) & ((p < max_kv_len) if max_kv_len else True)
            at = page.clamp(0, self.cache.n_pages - 1), slice(None), p % self.page
            k, v = (decoded(a[at], None if b is None else b[at], self.kind) for a, b in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)))
            rows = slice(row, row + c)
            out[rows], tol[rows] = attention(self.q[rows].double(), k, v, seen_of(c, n, window, there), scale, softcap, sinks, self.half, self.kind != 0, self.q_half)
            row += c
        return out, tol, row

    def check(self, scale=None, softcap=0.0, window=0, sinks=None, max_kv_len=0, **more):
        torch = self.torch
        scale = self.d ** -0.5 if scale is None else scale
        out = torch.full(self.q.shape, 7.0, device="cuda", dtype=torch.float16 if self.half else torch.float32)
        self.cuda.attention_chunk(self.q, self.cache, scale=scale, softcap=softcap, window=window, sinks=sinks, max_kv_len=max_kv_len, out=out, **{**self.args(), **more})
        want, tol, rows = self.want(scale, softcap, window, sinks, max_kv_len)
        assert (out[rows:] == 7.0).all(), "rows behind the last sequence"
        got, want, tol = out[:rows].double(), want[:rows], tol[:rows]
        finite = torch.isfinite(want)
        assert (torch.isfinite(got) == finite).all(), "where results are numbers"
        ratio = torch.where(finite, (got - want).abs() / (tol + 1e-30), 0)
        if ratio.numel():
            assert float(ratio.max()) <= 1.0, f"worst {float(ratio.max()):.3g} of the tolerance at {np.unravel_index(int(ratio.argmax()), tuple(ratio.shape))}"
        assert self.cuda.device_status() == 0
        return out[:rows]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("d,kv,group,page", [(64, 2, 7, 16), (96, 1, 3, 48), (128, 2, 4, 16), (128, 1, 1, 64), (192, 1, 5, 32), (256, 2, 2, 16), (128, 1, 20, 256)])
def test_types_and_head_layouts(cuda, kind, act, d, kv, group, page):
    Batch(cuda, d + group, KINDS[kind], d, kv, group, page, [1, 40, 0, 130, 7], [1, 40, 30, 700, 66], act).check()


@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("f16", "f16"), ("q8", "f16"), ("q4", "f32")])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 600])
@pytest.mark.parametrize("before", [0, 5, 700])
def test_lengths(cuda, kind, act, n, before):
    Batch(cuda, n, KINDS[kind], 128, 1, 4, 16, [n], [before + n], act).check()


@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("f16", "f16"), ("q8", "f32>f16"), ("q4", "f16"), ("q8", "f32")])
def test_long_contexts(cuda, kind, act):
    """A few tokens behind many positions, which several blocks of threads share; a long chunk beside them."""
    b = Batch(cuda, 3, KINDS[kind], 128, 2, 4, 64, [1, 5, 300, 1, 64], [20001, 9000, 3000, 700, 12345], act)
    first = b.check()
    assert (b.check() == first).all(), "the same bits every time"
    b.check(max_kv_len=20001)
    b.check(max_kv_len=8000)


@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("q8", "f16")])
@pytest.mark.parametrize("counts,context", [([900], 0), ([2, 1, 3, 1, 1, 2, 1, 4] * 12, 100), ([257, 1, 1, 513, 64, 3], 900)])
def test_batches(cuda, kind, act, counts, context):
    lens = [c + (context * (i % 4)) // 3 for i, c in enumerate(counts)]
    Batch(cuda, 5, KINDS[kind], 64, 2, 2, 32, counts, lens, act).check()


@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("f16", "f16"), ("q8", "f16"), ("q4", "f32")])
@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 1000])
def test_windows(cuda, kind, act, window):
    Batch(cuda, window, KINDS[kind], 64, 1, 4, 16, [1, 150, 300, 40], [800, 950, 300, 40], act).check(window=window)


@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("f16", "f16"), ("q8", "f16"), ("q4", "f32")])
def test_softcap_and_sinks(cuda, kind, act):
    b = Batch(cuda, 7, KINDS[kind], 128, 2, 4, 16, [140, 1], [900, 30], act, q_size=8.0)
    sinks = 5 * b.torch.randn(8, device="cuda", generator=b.torch.Generator("cuda").manual_seed(1))
    sinks[1], sinks[2] = -np.inf, 80.0
    b.check(softcap=20.0)
    b.check(sinks=sinks)
    b.check(softcap=50.0, sinks=sinks, window=128)
    b.check(scale=-0.05)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_rows_that_see_nothing(cuda, kind, act):
    """More rows than positions, sequences without positions, pages that are none."""
    b = Batch(cuda, 9, KINDS[kind], 64, 1, 2, 16, [5, 3, 200, 40], [2, 0, 130, 40], act)
    got = b.check()
    assert (got[:3] == 0).all() and (got[5:8] == 0).all() and (got[8:78] == 0).all() and (got[3:5] != 0).any()
    sinks = b.torch.randn(2, device="cuda")
    assert (b.check(sinks=sinks)[:3] == 0).all()
    b.lens[1] = -7
    b.check()
    b = Batch(cuda, 10, KINDS[kind], 128, 1, 2, 16, [150, 20], [600, 20], act)
    b.table[0, :5], b.table[0, 9], b.table[0, 20], b.table[1, 0] = -1, 1 << 30, b.cache.n_pages, -5
    assert (b.check()[150:150 + 16] == 0).all()
    b.check(window=40)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_what_is_not_seen_does_not_matter(cuda, kind, act):
    """Infinities and NaN behind the last position, in unused pages, before the window, and in tokens of the chunk that come later."""
    b = Batch(cuda, 11, KINDS[kind], 64, 1, 2, 16, [150, 1], [405, 1003], act)
    torch = b.torch
    clean = b.check(window=200)
    keep = torch.zeros((b.cache.n_pages, 16), dtype=torch.bool)
    for s, (c, n) in enumerate(zip(b.counts, b.lens)):
        p = torch.arange(max(0, n - c + 1 - 200), n)
        keep[b.table[s, p // 16].long(), p % 16] = True
    keep = keep.cuda()[:, None, :, None]
    odd = torch.tensor([np.nan, np.inf, -np.inf, 65504], dtype=torch.float16, device="cuda")
    for a in (b.cache.k, b.cache.v) if KINDS[kind] == 0 else (b.cache.k_scale, b.cache.v_scale):
        a.copy_(torch.where(keep, a, odd[torch.randint(0, 4, a.shape, device="cuda")]))
    assert (b.check(window=200) == clean).all()
    # the chunk's 70th token has values that are no numbers, its 100th a key
    for name, i in (("v", 70), ("k", 100)):
        a = getattr(b.cache, name if KINDS[kind] == 0 else name + "_scale")
        p = 405 - 150 + i
        a[b.table[0, p // 16].long(), 0, p % 16, 0] = np.inf if name == "v" else np.nan
    out = torch.full(b.q.shape, 7.0, device="cuda", dtype=torch.float16 if b.half else torch.float32)
    cuda.attention_chunk(b.q, b.cache, scale=0.125, window=200, out=out, **b.args())
    assert (out[:70] == clean[:70]).all() and (out[150] == clean[150]).all()
    assert (~torch.isfinite(out[70:100])).any(-1).all() and (~torch.isfinite(out[100:150])).all()
    if KINDS[kind] == 0:
        assert torch.isfinite(out[70:100, :, 1:]).all() and not torch.isfinite(out[70:100, :, 0]).any()


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_values_of_unlike_size(cuda, act):
    b = Batch(cuda, 13, 0, 64, 1, 4, 16, [130], [1300], act)
    torch = b.torch
    size = torch.exp2(torch.linspace(-12, 9, 1300, device="cuda"))
    p = torch.arange(1300, device="cuda")
    b.cache.v[b.table[0].cuda()[p // 16].long(), 0, p % 16] *= size[:, None].half()
    b.check()
    for q_size in (1e-20, 1e-4, 1e4) if act == "f32" else (1e-4, 1e4):
        b.q = (q_size * torch.randn(b.q.shape, device="cuda")).to(b.q.dtype)
        b.check(scale=1.0 / q_size / 8)


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_scales_beyond_the_range_of_f16_values(cuda, kind):
    """f32 results over quants times scales that pass 65504: what no two f16 terms hold."""
    b = Batch(cuda, 14, KINDS[kind], 128, 2, 4, 16, [90, 40], [700, 300], "f32")
    clean = b.check()
    for name, p in (("v", 3), ("k", 200), ("v", 695)):
        scale = getattr(b.cache, name + "_scale")
        was = scale.clone()
        scale[b.table[0, p // 16].long(), 1, p % 16] = 60000.0
        if name == "k":
            b.q *= 2.0 ** -16
        b.check()
        if name == "k":
            b.q *= 2.0 ** 16
        scale.copy_(was)
    assert (b.check() == clean).all()
    b.cache.v_scale[b.table[0, 2].long(), :, 5] = 60000.0   # a position before the window
    b.check(window=300)


@pytest.mark.parametrize("kind,d", [("f16", 128), ("f16", 64), ("f16", 256), ("q8", 128), ("q4", 96)])
def test_sums_over_many_positions(cuda, kind, d):
    """f32: products' sums are cut off at 2^-23 of what they have come to, which a run of 256 steps' worth of positions bounds at 256 / 2 * 2^-23 (sums that grow evenly,
    of values of one sign), however many positions there are; 5 * 2^-20 beside that (weights and values in two terms, exponentials of scores below 2)."""
    b = Batch(cuda, 21, KINDS[kind], d, 1, 4, 64, [200, 64], [20000, 9000], "f32", q_size=0.1, spread=False)
    torch = b.torch
    x = torch.randn((2, b.cache.n_pages * 64, 1, d), device="cuda")
    cuda.kv_append(b.cache, x[0], x[1].abs() + 2, torch.arange(b.cache.n_pages * 64, device="cuda"))
    got = b.check().double()
    want, _, rows = b.want(d ** -0.5)
    assert float(((got - want[:rows]).abs() / want[:rows]).max()) <= 128 * 2.0 ** -23 + 5 * 2.0 ** -20


def test_strides_streams_and_graphs(cuda):
    """Rows of q and out apart, another stream, two captured graphs that share a workspace and replay on other lengths."""
    import torch
    b = Batch(cuda, 15, 1, 128, 2, 2, 16, [70, 3], [400, 2000], "f16")
    args = b.args()
    rows = 73
    want = b.check()
    wide = torch.zeros((rows, 6, 128), dtype=torch.float16, device="cuda")
    wide[:, 1:5] = b.q[:rows]
    to = torch.full((rows, 7, 128), 3.0, dtype=torch.float16, device="cuda")
    cuda.attention_chunk(wide[:, 1:5], b.cache, out=to[:, 2:6], **args)
    assert (to[:, 2:6] == want).all() and (to[:, :2] == 3).all() and (to[:, 6:] == 3).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    on_side = cuda.attention_chunk(b.q, b.cache, stream=side, **args)
    side.synchronize()
    assert (on_side[:rows] == want).all()
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    outs, graphs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(cuda.attention_chunk(b.q, b.cache, workspace=ws, **args))
        graphs.append(graph)
    for o, graph in zip(outs, graphs):
        o.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert all((o[:rows] == want).all() for o in outs)
    args["kv_len"].copy_(torch.tensor([300, 1500], dtype=torch.int32))
    args["q_start"].copy_(torch.tensor([0, 20, 21], dtype=torch.int32))
    graphs[0].replay()
    b.counts, b.lens = [20, 1], [300, 1500]
    want = b.check(max_q=70)
    assert (outs[0][:21] == want).all()


def test_far_pages(cuda):
    """Rows of the pool more than 2^31 values and 2^32 bytes in."""
    import torch
    pages, kv, page, d = 150000, 2, 64, 128
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 10 GB")
    cache = cuda.KvCache(0, *(torch.empty((pages, kv, page, d), dtype=torch.float16, device="cuda") for _ in range(2)))
    b = Batch(cuda, 17, 0, d, kv, 2, page, [100], [300], "f32")
    far = torch.arange(pages - b.cache.n_pages, pages, device="cuda")
    cache.k[far], cache.v[far] = b.cache.k, b.cache.v
    want = b.check()
    args = b.args()
    args["page_table"] = torch.where(args["page_table"] >= 0, args["page_table"] + pages - b.cache.n_pages, -1)
    assert (cuda.attention_chunk(b.q, cache, **args)[:100] == want).all()


def test_through_the_c_call(cuda):
    """No sequences, no rows; more rows than max_q (those beyond are not touched); a workspace of the size that is asked for."""
    import torch
    b = Batch(cuda, 19, 0, 64, 1, 2, 16, [40], [1000], "f32")
    a = b.args()
    out = torch.full(b.q.shape, 7.0, device="cuda")
    p = lambda t: t.data_ptr()  # noqa: E731
    s = cuda.Attention(q_start=p(a["q_start"]), kv_len=p(a["kv_len"]), page_table=p(a["page_table"]), q_stride=128, out_stride=128, n_seq=1, n_heads=2, max_q=40,
                       table_width=a["page_table"].shape[1], scale=0.125)
    size = cuda.lib.krk_cuda_attention_chunk_workspace_bytes(C.byref(b.cache.struct), C.byref(s), 0)
    ws = torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    assert cuda.lib.krk_cuda_attention_chunk(p(out), 0, p(b.q), 0, C.byref(b.cache.struct), C.byref(s), p(ws), size, st) == 0
    want = b.check()
    assert (out[:40] == want).all() and (ws[size:] == 0xFF).all()
    before = cuda.launch_count()
    for n_seq, max_q in ((0, 40), (1, 0)):
        s.n_seq, s.max_q = n_seq, max_q
        assert cuda.lib.krk_cuda_attention_chunk(p(out), 0, p(b.q), 0, C.byref(b.cache.struct), C.byref(s), None, 0, st) == 0
    assert cuda.launch_count() == before

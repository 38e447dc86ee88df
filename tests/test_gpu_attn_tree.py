"""Attention of drafted tokens over a paged cache, against a plain form in 64 bits: types, head sizes and groups, lengths from none to long
ones, pages, trees, windows, sinks, masks that leave rows empty, infinities and NaN at positions that are not seen."""
import numpy as np
import pytest

from attn_plain import attention, decode, encode, visible

pytestmark = pytest.mark.gpu
KINDS = {"f16": 0, "q8": 1, "q4": 2}
ALL = (1 << 64) - 1


def tree_masks(rng, n, shape="tree"):
    if shape == "chain":
        return [(2 << i) - 1 for i in range(n)]
    out = []
    for i in range(n):
        parent = int(rng.integers(-1, i)) if i else -1
        out.append((out[parent] if parent >= 0 else 0) | 1 << i)
    return out


class Batch:
    """Sequences over a cache whose pages lie in no order; `extra` unused pages, and rows of q behind the last sequence."""

    def __init__(self, cuda, rng, kind, d, kv, group, page, counts, lens, masks, extra_rows=2, q_size=2.0):
        import torch
        self.cuda, self.kind, self.d, self.kv, self.group, self.page = cuda, kind, d, kv, group, page
        self.counts, self.lens, self.masks = counts, lens, masks
        used = [(n + page - 1) // page for n in lens]
        self.width = max(max(used), 1) + 1
        order = rng.permutation(sum(used) + 2)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for s, u in enumerate(used):
            self.table[s, :u] = order[at:at + u]
            at += u
        shape = (sum(used) + 2, kv, page, d)
        self.raw = []
        for _ in range(2):
            x = rng.standard_normal(shape).astype(np.float32) * rng.uniform(0.2, 3.0, (*shape[:3], 1)).astype(np.float32)
            self.raw.append([a if a is None else np.array(a) for a in encode(x, kind)])
        self.q = (q_size * rng.standard_normal((sum(counts) + extra_rows, kv * group, d))).astype(np.float32)
        self.torch = torch

    def dev(self, a):
        return None if a is None else self.torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def cache(self):
        (k, ks), (v, vs) = self.raw
        return self.cuda.KvCache(self.kind, self.dev(k), self.dev(v), self.dev(ks), self.dev(vs))

    def args(self):
        start = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        tree = None if self.masks is None else self.dev(np.array([m for ms in self.masks for m in ms] + [0] * (len(self.q) - sum(self.counts)), np.uint64).view(np.int64))
        return dict(q_start=self.dev(start), kv_len=self.dev(np.array(self.lens, np.int32)), page_table=self.dev(self.table), max_q=max(max(self.counts), 1), tree=tree)

    def want(self, scale, softcap=0.0, window=0, sinks=None):
        out, tol, row = np.zeros(self.q.shape), np.zeros(self.q.shape), 0
        for s, (c, n) in enumerate(zip(self.counts, self.lens)):
            p = np.arange(n)
            page = self.table[s, p // self.page]
            at = np.clip(page, 0, len(self.raw[0][0]) - 1), slice(None), p % self.page   # (a page that is none is masked below)
            k, v = (decode(np.asarray(a)[at], None if b is None else np.asarray(b)[at], self.kind) for a, b in self.raw)
            seen = visible(None if self.masks is None else self.masks[s], c, n, window) & (page >= 0) & (page < len(self.raw[0][0]))
            out[row:row + c], tol[row:row + c] = attention(self.q[row:row + c], k, v, seen, scale, softcap, sinks)
            row += c
        return out, tol, row

    def check(self, scale=None, softcap=0.0, window=0, sinks=None, **more):
        scale = self.d ** -0.5 if scale is None else scale
        out = self.torch.full(self.q.shape, 7.0, device="cuda")
        self.cuda.attention_tree(self.dev(self.q), self.cache(), scale=scale, softcap=softcap, window=window, sinks=self.dev(sinks), out=out, **{**self.args(), **more})
        got = out.cpu().numpy().astype(np.float64)
        want, tol, rows = self.want(scale, softcap, window, sinks)
        assert (got[rows:] == 7.0).all(), "rows behind the last sequence"
        finite = np.isfinite(want[:rows])
        assert (np.isfinite(got[:rows]) == finite).all()
        off = np.abs(got[:rows] - want[:rows])[finite]
        lim = tol[:rows][finite] + 1e-30
        assert (off <= lim).all(), f"worst {float((off / lim).max()):.3g} of the tolerance at {np.argmax(off / lim)}"
        return got[:rows]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,kv,group,page", [(64, 2, 7, 16), (96, 1, 3, 48), (128, 2, 4, 16), (128, 1, 1, 64), (192, 1, 5, 32), (256, 2, 2, 16), (128, 1, 20, 32)])
def test_types_and_head_layouts(cuda, kind, d, kv, group, page):
    rng = np.random.default_rng(d + group)
    counts, lens = [1, 3, 0, 8, 1], [1, 3, 40, 700, 65]
    masks = [tree_masks(rng, c) for c in counts]
    Batch(cuda, rng, KINDS[kind], d, kv, group, page, counts, lens, masks).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 63, 64, 65, 511, 512, 513, 4099])
def test_one_token_over_lengths(cuda, kind, n):
    rng = np.random.default_rng(n)
    Batch(cuda, rng, KINDS[kind], 128, 2, 4, 16, [1], [n], None).check()


@pytest.mark.parametrize("kind,n_q,group,shape", [("f16", 64, 4, "tree"), ("f16", 64, 1, "chain"), ("q8", 33, 8, "tree"), ("q4", 17, 3, "tree"), ("q8", 64, 7, "chain"), ("f16", 16, 1, "tree")])
def test_trees(cuda, kind, n_q, group, shape):
    """The last mask bits of 64 rows, chains that cross chunks, a context that ends inside a chunk."""
    rng = np.random.default_rng(n_q)
    counts = [n_q, max(1, n_q // 2), n_q]
    lens = [n_q + 1000, counts[1] + 7, n_q]
    Batch(cuda, rng, KINDS[kind], 64, 1, group, 16, counts, lens, [tree_masks(rng, c, shape) for c in counts]).check()


def test_no_tree_is_causal(cuda):
    rng = np.random.default_rng(3)
    b = Batch(cuda, rng, 0, 128, 1, 2, 32, [64, 5], [300, 5], None)
    got = b.check()
    b.masks = [tree_masks(rng, 64, "chain"), tree_masks(rng, 5, "chain")]
    assert (b.check() == got).all()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_see_nothing(cuda, kind):
    """Empty masks without a context, bits that point at no row, sequences without positions, shorter than their rows."""
    rng = np.random.default_rng(5)
    masks = [[0, 2, 4], [0], [1 << 63, ALL], [3, 2], [0, 1]]
    b = Batch(cuda, rng, KINDS[kind], 64, 2, 3, 16, [3, 1, 2, 2, 2], [3, 1, 2, 0, 600], masks)
    got = b.check()
    assert (got[0] == 0).all() and (got[3] == 0).all() and (got[6] == 0).all() and (got[1] != 0).any()
    sinks = rng.standard_normal(6).astype(np.float32)
    assert (b.check(sinks=sinks)[0] == 0).all()
    # more rows than positions: those at positions before the first see what there is
    b = Batch(cuda, rng, KINDS[kind], 64, 1, 2, 16, [5], [2], None)
    assert (b.check()[:3] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,n", [(64, 63), (64, 64), (64, 65), (64, 200), (127, 900), (100, 4000), (2000, 700)])
def test_windows(cuda, kind, window, n):
    rng = np.random.default_rng(window + n)
    counts, lens = [1, 6], [n, n + 6]
    b = Batch(cuda, rng, KINDS[kind], 64, 1, 4, 16, counts, lens, [[1], tree_masks(rng, 6)])
    b.check(window=window)
    b.masks[1][3] = 0   # its position is one before the first drafted token
    b.check(window=window)


@pytest.mark.parametrize("kind", KINDS)
def test_softcap_and_sinks(cuda, kind):
    rng = np.random.default_rng(7)
    b = Batch(cuda, rng, KINDS[kind], 128, 2, 4, 16, [4, 1], [900, 30], [tree_masks(rng, 4), [1]], q_size=8.0)
    sinks = (5 * rng.standard_normal(8)).astype(np.float32)
    sinks[1], sinks[2] = -np.inf, 80.0
    b.check(softcap=20.0)
    b.check(sinks=sinks)
    b.check(softcap=50.0, sinks=sinks, window=128)
    b.check(scale=-0.05)


@pytest.mark.parametrize("kind", KINDS)
def test_values_of_unlike_size(cuda, kind):
    """Scales over many powers of two, the greatest met late; queries far from one; scores far apart."""
    rng = np.random.default_rng(9)
    b = Batch(cuda, rng, KINDS[kind], 64, 1, 4, 16, [2], [1300], None)
    size = np.exp2(np.linspace(-12, 9, b.raw[1][0].shape[0] * 16)).reshape(-1, 1, 16, 1)
    order = np.argsort(np.concatenate([b.table[0][b.table[0] >= 0], np.setdiff1d(np.arange(len(size)), b.table[0])]))
    x = rng.standard_normal(b.raw[1][0].shape[:3] + (64,)).astype(np.float32) * size[order]
    b.raw[1] = list(encode(x, KINDS[kind]))
    b.check()
    for q_size in (1e-20, 1e-4, 1e4):
        b.q = (q_size * rng.standard_normal(b.q.shape)).astype(np.float32)
        b.check(scale=1.0 / q_size / 8)


@pytest.mark.parametrize("kind", KINDS)
def test_what_is_not_seen_does_not_matter(cuda, kind):
    """Infinities and NaN behind the last position, in unused pages, before the window, and at drafted tokens of other branches."""
    rng = np.random.default_rng(11)
    counts, lens = [5, 1], [405, 1003]
    masks = [[1, 2 | 1, 4 | 1, 8, 16 | 8], [1]]
    b = Batch(cuda, rng, KINDS[kind], 64, 1, 2, 16, counts, lens, masks)
    clean = b.check(window=200)
    for a, scale in b.raw:
        bad = np.array(a if KINDS[kind] == 0 else scale)
        flat = bad.copy()
        keep = np.zeros(bad.shape[:1] + bad.shape[2:3], bool)   # [page][place]
        for s, (c, n) in enumerate(zip(counts, lens)):
            for p in range(max(0, n - c - 200), n):
                keep[b.table[s, p // 16], p % 16] = True
        vals = np.array([np.nan, np.inf, -np.inf, 65504], np.float16)
        flat[:] = vals[rng.integers(0, 4, bad.shape)]
        target = a if KINDS[kind] == 0 else scale
        target[...] = np.where(keep[:, None, :, None], bad, flat)
    assert (b.check(window=200) == clean).all()
    # drafted tokens 1 (seen by row 1 alone) and 3 (by rows 3 and 4)
    for a, scale in b.raw:
        target = a if KINDS[kind] == 0 else scale
        p = lens[0] - 5 + np.array([1, 3])
        target[b.table[0, p // 16], 0, p % 16, 0] = [np.nan, np.inf]
    got = b.check(window=200)
    assert (got[[0, 2]] == clean[[0, 2]]).all() and (got[5] == clean[5]).all()
    assert np.isnan(got[1]).any() and not np.isfinite(got[3:5]).all()


def test_infinite_values_reach_the_rows_that_see_them(cuda):
    """f16: an infinite value at one place of a drafted token's row gives that place alone."""
    rng = np.random.default_rng(12)
    b = Batch(cuda, rng, 0, 128, 1, 1, 16, [3], [50], [[1, 3, 5]])
    p = 50 - 2
    b.raw[1][0][b.table[0, p // 16], 0, p % 16, 77] = -np.inf
    got = b.check()
    assert np.isneginf(got[1, 0, 77]) and np.isfinite(got[[0, 2]]).all() and np.isfinite(np.delete(got[1, 0], 77)).all()


def test_bad_pages_are_not_seen(cuda):
    rng = np.random.default_rng(13)
    for kind in KINDS.values():
        b = Batch(cuda, rng, kind, 64, 1, 2, 16, [1, 2], [700, 100], None)
        b.table[0, 3], b.table[0, 20], b.table[1, 2], b.table[1, 6] = -1, 1 << 30, len(b.raw[0][0]), -(1 << 31)
        b.check()


def test_max_kv_len_is_a_limit(cuda):
    rng = np.random.default_rng(14)
    b = Batch(cuda, rng, 0, 64, 1, 2, 16, [1, 1], [100, 40], None)
    got = b.check()
    assert (b.check(max_kv_len=100) == got).all()


@pytest.mark.parametrize("kind", KINDS)
def test_ragged_batch_and_the_same_bits(cuda, kind):
    """Many sequences of unlike lengths: items divided among CTAs, several to a CTA, and the same bits from every call."""
    rng = np.random.default_rng(15)
    lens = [int(x) for x in np.concatenate([rng.integers(1, 200, 140), rng.integers(600, 4000, 6), [0, 1, 64]])]
    counts = [int(min(c, max(n, 1))) for c, n in zip(rng.integers(0, 6, len(lens)), lens)]
    counts[-3:] = [1, 1, 1]
    b = Batch(cuda, rng, KINDS[kind], 64, 2, 3, 16, counts, lens, [tree_masks(rng, c) for c in counts])
    assert (b.check() == b.check()).all()


def test_strides_streams_and_graphs(cuda):
    """q and out inside wider rows; another stream; a captured call replayed on new lengths and inputs; two graphs with a workspace each."""
    import torch
    rng = np.random.default_rng(16)
    b = Batch(cuda, rng, 1, 128, 2, 4, 16, [2, 3], [1500, 700], [tree_masks(rng, 2), tree_masks(rng, 3)], extra_rows=0)
    want = b.check()
    cache, args = b.cache(), b.args()
    wide = torch.zeros((5, 8 * 128 + 2 * 256 + 4), device="cuda")
    q = wide[:, :1024].unflatten(1, (8, 128))
    q.copy_(b.dev(b.q))
    wide_out = torch.full((5, 1100), 3.0, device="cuda")
    out = wide_out[:, 4:1028].unflatten(1, (8, 128))
    cuda.attention_tree(q, cache, out=out, **args)
    assert (out.cpu().numpy() == want).all() and (wide_out[:, :4] == 3.0).all() and (wide_out[:, 1028:] == 3.0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    on_side = cuda.attention_tree(q, cache, stream=side, **args)
    side.synchronize()
    assert (on_side.cpu().numpy() == want).all()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cuda.attention_tree(q, cache, **args))
        graphs.append(g)
    for g, o in zip(graphs, outs):
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert (o.cpu().numpy() == want).all()
    b.lens, b.counts, b.masks = [900, 303], [1, 4], [[1], tree_masks(rng, 4)]
    b.q = rng.standard_normal(b.q.shape).astype(np.float32)
    new = b.args()
    for name in ("q_start", "kv_len", "tree"):
        args[name].copy_(new[name])
    q.copy_(b.dev(b.q))
    graphs[0].replay()   # captured for three rows a sequence, which the second one has more than: its rows that are there are right
    torch.cuda.synchronize()
    assert (outs[0][0].cpu().numpy() == b.check()[0]).all()
    b.lens, b.counts, b.masks = [900, 303], [2, 3], [[1, 3], tree_masks(rng, 3)]
    for name, new in b.args().items():
        if name in ("q_start", "kv_len", "tree"):
            args[name].copy_(new)
    graphs[1].replay()
    torch.cuda.synchronize()
    assert (outs[1].cpu().numpy() == b.check()).all()


# ---- more than 32 rows to a key head over an f16 cache, heads of 96 and 128 values, contexts that are divided: the form on tcgen05


@pytest.mark.parametrize("d,group,n_q,page", [(128, 4, 9, 16), (128, 1, 33, 48), (96, 8, 8, 16), (96, 5, 13, 64), (128, 7, 64, 32), (128, 16, 4, 16), (96, 2, 64, 16), (128, 3, 17, 272)])
def test_many_rows(cuda, d, group, n_q, page):
    rng = np.random.default_rng(d + n_q)
    counts = [n_q, 1, n_q - 1, 0, n_q, 3]
    lens = [n_q + 2100, 900, n_q - 1, 40, n_q + 131, 129]
    Batch(cuda, rng, 0, d, 2, group, page, counts, lens, [tree_masks(rng, c) for c in counts]).check()


@pytest.mark.parametrize("n", [1, 40, 127, 128, 129, 255, 257, 1000, 5000])
def test_many_rows_over_lengths(cuda, n):
    rng = np.random.default_rng(n)
    Batch(cuda, rng, 0, 128, 1, 4, 16, [min(n, 40), 12], [n, 600], None).check()


def test_many_rows_windows_sinks_and_limits(cuda):
    rng = np.random.default_rng(21)
    b = Batch(cuda, rng, 0, 128, 2, 4, 16, [12, 30, 1], [1500, 130, 700], [tree_masks(rng, 12), tree_masks(rng, 30), [1]], q_size=6.0)
    sinks = (5 * rng.standard_normal(8)).astype(np.float32)
    sinks[0], sinks[3] = -np.inf, 60.0
    for window in (0, 64, 100, 513, 1400):
        b.check(window=window)
        b.check(window=window, sinks=sinks, softcap=25.0)
    b.check(scale=-0.1)
    b.masks[1][4] = b.masks[1][9] = 0
    b.lens[1] = 30
    got = b.check()
    assert (got[12 + 4] == 0).all() and (got[12 + 9] == 0).all()


def test_many_rows_values_of_unlike_size(cuda):
    """The greatest scores late, and far above the first ones: references that have to follow."""
    rng = np.random.default_rng(22)
    b = Batch(cuda, rng, 0, 128, 1, 4, 16, [10], [3000], None, q_size=3.0)
    for t in range(0, 2900, 97):
        page = b.table[0, t // 16]
        b.raw[0][0][page, 0, t % 16] *= np.float16(1 + t / 300)
    got = b.check()
    assert (got == b.check()).all()
    for q_size in (1e-20, 1e4):
        b.q = (q_size * rng.standard_normal(b.q.shape)).astype(np.float32)
        b.check(scale=1.0 / q_size / 11)


def test_many_rows_what_is_not_seen(cuda):
    rng = np.random.default_rng(23)
    counts, lens = [12, 1], [905, 1003]
    masks = [[1, 3, 5, 9, 24 | 1, 1 << 5, 3 << 5, 1 << 7, 1 << 8, 1 << 9, 1 << 10, 1 << 11], [1]]
    b = Batch(cuda, rng, 0, 128, 1, 4, 16, counts, lens, masks)
    clean = b.check(window=200)
    vals = np.array([np.nan, np.inf, -np.inf, 65504], np.float16)
    for a, _ in b.raw:
        keep = np.zeros((len(a), 16), bool)
        for s, (c, n) in enumerate(zip(counts, lens)):
            for p in range(max(0, n - c - 200), n):
                keep[b.table[s, p // 16], p % 16] = True
        a[...] = np.where(keep[:, None, :, None], a, vals[rng.integers(0, 4, a.shape)])
    assert (b.check(window=200) == clean).all()
    p = lens[0] - 12 + np.array([1, 6])   # seen by row 1, by row 6
    for a, _ in b.raw:
        a[b.table[0, p // 16], 0, p % 16, 5] = np.nan
    got = b.check(window=200)
    assert np.isnan(got[1]).any() and np.isnan(got[6]).any() and np.isfinite(np.delete(got, [1, 6], 0)).all()
    b.raw[0][0][b.table[0, p // 16], 0, p % 16, 5] = 0     # the values alone
    got = b.check(window=200)
    assert np.isnan(got[[1, 6], :, 5]).all() and np.isnan(got).sum() == 8


def test_many_rows_bad_pages_graphs_and_limits(cuda):
    import torch
    rng = np.random.default_rng(24)
    b = Batch(cuda, rng, 0, 128, 2, 4, 16, [10, 16], [1700, 100], [tree_masks(rng, 10), tree_masks(rng, 16)])
    b.table[0, 3], b.table[0, 20], b.table[0, 106], b.table[1, 2] = -1, 1 << 30, len(b.raw[0][0]), -5
    want = b.check()
    cache, args, q = b.cache(), b.args(), b.dev(b.q)
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cuda.attention_tree(q, cache, out=out, **args)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert (out.cpu().numpy()[:26] == want).all()
    assert cuda.device_status() == 0


@pytest.mark.parametrize("kind,n_q", [("f16", 3), ("q8", 3), ("f16", 40)])
def test_positions_behind_max_kv_len(cuda, kind, n_q):
    """The drafted tokens stay the last of kv_len; what lies behind the limit is not seen."""
    rng = np.random.default_rng(25)
    b = Batch(cuda, rng, KINDS[kind], 128, 1, 2, 16, [n_q, 1], [1200, 300], [tree_masks(rng, n_q), [1]])
    for limit in (1190, 900, 299, 3):
        out = b.dev(np.zeros_like(b.q))
        cuda.attention_tree(b.dev(b.q), b.cache(), scale=0.1, max_kv_len=limit, out=out, **b.args())
        got, row = out.cpu().numpy(), 0
        for s, (c, n) in enumerate(zip(b.counts, b.lens)):
            p = np.arange(n)
            at = b.table[s, p // 16], slice(None), p % 16
            k, v = (decode(np.asarray(a)[at], None if x is None else np.asarray(x)[at], b.kind) for a, x in b.raw)
            want, tol = attention(b.q[row:row + c], k, v, visible(b.masks[s], c, n) & (p < limit), 0.1)
            assert (np.abs(got[row:row + c] - want) <= tol + 1e-30).all()
            row += c


def test_no_rows_and_infinite_sinks(cuda):
    import torch
    rng = np.random.default_rng(26)
    b = Batch(cuda, rng, 0, 64, 1, 2, 16, [0, 0], [50, 0], None, extra_rows=0)
    assert cuda.attention_tree(b.dev(b.q), b.cache(), **b.args()).shape == (0, 2, 64)
    b = Batch(cuda, rng, 0, 64, 1, 2, 16, [2], [50], None, extra_rows=0)
    sinks = torch.tensor([float("inf"), 0.0], device="cuda")
    got = cuda.attention_tree(b.dev(b.q), b.cache(), sinks=sinks, **b.args())
    assert (got[:, 0] == 0).all() and (got[:, 1] != 0).all()


@pytest.mark.parametrize("kind,n_q,width", [(0, 3, 4), (0, 40, 100), (1, 3, 100), (2, 40, 4)])
def test_a_cache_without_pages(cuda, kind, n_q, width):
    """No memory behind it: nothing is seen."""
    import ctypes as C

    import torch
    q = torch.ones((n_q, 2, 128), device="cuda")
    out = torch.full_like(q, 7.0)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    start, length, table = i32(0, n_q), i32(1500), torch.zeros((1, width), dtype=torch.int32, device="cuda")
    cache = cuda.KvCacheStruct(type=kind, head_dim=128, n_kv_heads=1, page_size=16, n_pages=0)
    a = cuda.Attention(q_start=start.data_ptr(), kv_len=length.data_ptr(), page_table=table.data_ptr(), q_stride=256, out_stride=256, n_seq=1, n_heads=2,
                       max_q=n_q, table_width=width, scale=0.1)
    size = cuda.lib.krk_cuda_attention_tree_workspace_bytes(C.byref(cache), C.byref(a))
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    assert cuda.lib.krk_cuda_attention_tree(out.data_ptr(), q.data_ptr(), C.byref(cache), C.byref(a), ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
    assert (out == 0).all()


@pytest.mark.parametrize("kind,n_q", [("f16", 3), ("q8", 3), ("q4", 3), ("f16", 20)])
@pytest.mark.parametrize("softcap", [1e30, 3e38])
def test_soft_limits_far_above_the_scores(cuda, kind, n_q, softcap):
    """The formula is the one without a limit there. A score over such a limit lies below the normal numbers: half a step of the quotient and
    two of the tangent, 2.5 2^-149, come back times the limit (3e38 is below 2^128) as 1.25 2^-20 at most, two products as 2^-23 of the score each;
    attention()'s tolerance counts 2^-22 and 2^-23 of the score beside others, so that six of it hold both."""
    rng = np.random.default_rng(27)
    b = Batch(cuda, rng, KINDS[kind], 128, 1, 4, 16, [n_q, 1], [900, 30], [tree_masks(rng, n_q), [1]])
    want, tol, rows = b.want(0.1)
    got = cuda.attention_tree(b.dev(b.q), b.cache(), scale=0.1, softcap=softcap, **b.args()).cpu().numpy()
    assert (np.abs(got[:rows] - want[:rows]) <= 6 * tol[:rows] + 1e-30).all()


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("group,n_q,bad", [(1, 4, np.inf), (2, 4, np.inf), (4, 4, np.inf), (1, 40, np.inf), (1, 40, 65504.0), (1, 40, 100.0), (4, 13, 65504.0)])
def test_scales_that_a_row_does_not_see(cuda, kind, group, n_q, bad):
    """Small values, and at a drafted token of another branch a scale many powers of two above theirs (an infinite one, or one that no row of the same
    block of 16 sees): the rows that do not see it are as near to the formula as without it."""
    rng = np.random.default_rng(28)
    # the last token is the first one's sibling, all others are below the first one
    masks = [[1] + [1 | 1 << i for i in range(1, n_q - 1)] + [1 << n_q - 1], [1]]
    b = Batch(cuda, rng, KINDS[kind], 64, 1, group, 16, [n_q, 1], [n_q + 21, 700], masks)
    x = rng.standard_normal(b.raw[1][0].shape[:3] + (64,)).astype(np.float32) * 2.0 ** -8
    b.raw[1] = [np.array(a) for a in encode(x, KINDS[kind])]
    b.check()
    want, tol, rows = b.want(64 ** -0.5)
    p = 21 + n_q - 1
    block = [i for i in range(n_q - 1) if np.isinf(bad) or i * group // 16 < (n_q - 1) * group // 16]
    for which in (slice(0, 1), slice(0, 2)):
        keep = b.raw[1][1].copy()
        b.raw[1][1][b.table[0, p // 16], 0, p % 16, which] = bad
        got = cuda.attention_tree(b.dev(b.q), b.cache(), **b.args()).cpu().numpy()[:rows]
        with np.errstate(invalid="ignore"):
            ok = np.abs(got - want[:rows]) <= tol[:rows]
        assert ok[block].all() and ok[n_q].all()
        assert np.isfinite(got[n_q - 1]).all() == np.isfinite(bad)
        if np.isinf(bad) and which == slice(0, 1):   # an infinite scale of one block leaves the other one's values
            assert ok[:n_q, :, 32:].all()
        b.raw[1][1] = keep


def test_many_rows_holes_beside_infinite_values(cuda):
    """Pages that are not there inside tiles that all rows see (of 128 positions), and an infinite value in such a tile: its place is no number, all
    others are as they should be; a tile without a page."""
    rng = np.random.default_rng(30)
    b = Batch(cuda, rng, 0, 128, 2, 4, 16, [10, 16], [1700, 1100], [tree_masks(rng, 10), tree_masks(rng, 16)])
    b.table[0, 20], b.table[0, 22], b.table[1, 16:24], b.table[1, 40] = -1, len(b.raw[0][0]), -1, 1 << 30
    b.check()
    p = 300   # (page 18, in the tile of pages 16 to 23)
    b.raw[1][0][b.table[0, p // 16], :, p % 16, 77] = np.inf
    got = b.check()
    assert not np.isfinite(got[:10, :, 77]).any() and np.isfinite(np.delete(got, 77, 2)).all() and np.isfinite(got[10:]).all()
    assert cuda.device_status() == 0

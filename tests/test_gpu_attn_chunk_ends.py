"""Attention of chunks at the ends of its numbers: soft limits up to the largest f32, scales of zero and near it, windows up to the largest int, and values that are no numbers over
8 and 4 bits in calls whose rows do not go to the kernel of trees. Against the definition in 64 bits; which rows go where is that of krk_attn_chunk.cu (max_q * group * head_dim above
256 * 128)."""
import numpy as np
import pytest

from test_gpu_attn_chunk import ACTS, KINDS, Batch

pytestmark = pytest.mark.gpu


def limited(b, s, rows, softcap, scale):
    """(out, tolerance) of sequence s of a Batch, all of whose pages and numbers are there.

    Per unit of a = sum(w |v|) / sum(w), as tests/chunk_plain.py derives them, but for the soft limit, whose error is counted against the score y = s / softcap that goes
    in and not against the limit: below |y| = 1/4 an odd series of five terms (the next one, 1382 / 155925 y^11, is 1e-8 of y at 1/4) with its rounding, 2^-22; from there on 1 - 2 / (1 + e), e off by
    2^-22 and its argument's rounding: 2^-22 of a tangent of 1, of one of 0.245 less than 2^-20. So 2^-20 of the greatest score."""
    from chunk_plain import decoded, seen_of
    torch = b.torch
    n, c = b.lens[s], b.counts[s]
    p = torch.arange(n, device="cuda")
    at = b.table.cuda()[s, p // b.page].long(), slice(None), p % b.page
    k, v = (decoded(a[at], None if x is None else x[at], b.kind) for a, x in ((b.cache.k, b.cache.k_scale), (b.cache.v, b.cache.v_scale)))
    seen, q, quants, d = seen_of(c, n), b.q[rows].double(), b.kind != 0, b.d
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(q.shape[1]):
        kk, vv, qq = k[:, h // (q.shape[1] // b.kv)], v[:, h // (q.shape[1] // b.kv)], q[:, h]
        x = torch.where(seen, qq @ kk.T, 0) * scale
        size = (torch.where(seen, qq.abs() @ kk.abs().T, 0) * abs(scale)).amax(1, keepdim=True)
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        most = x.abs().amax(1, keepdim=True)
        z = torch.where(seen, x, -torch.inf)
        w = torch.exp(z - z.amax(1, keepdim=True))
        total = w.sum(1, keepdim=True)
        o, a = w @ vv / total, w @ vv.abs() / total
        seen_n = seen.sum(1).double()[:, None]
        off = (2.0 ** -11 * ((not b.q_half) + quants) if b.half else 2.0 ** -22 * (1 + quants)) * size + (d / 16 + 4) * (1 if b.half else 3 if quants else 2) * 2.0 ** -23 * size
        if b.half and quants:
            off = off + 2.0 ** -25 * qq.abs().sum(1, keepdim=True) * abs(scale)
        off = off + 2.0 ** -22 * most + 2.0 ** -21 + (2.0 ** -20 * most if softcap else 0.0)
        t = a * (2 * off + (2.0 ** -11 * (1 + quants) + 2.0 ** -12 if b.half else 2.0 ** -22 * (2 + quants)) + (seen_n / 16 + 300) * 2.0 ** -23) + seen_n * 2.0 ** -32 * vv.abs().amax() / total.clamp(min=1.0)
        out[:, h], tol[:, h] = o, t + (2.0 ** -11 * o.abs() + 2.0 ** -25 * (2 + quants) if b.half else 0.0)
    return out, tol


def check(b, softcap=0.0, scale=None):
    torch = b.torch
    scale = b.d ** -0.5 if scale is None else scale
    out = torch.full(b.q.shape, 7.0, device="cuda", dtype=torch.float16 if b.half else torch.float32)
    b.cuda.attention_chunk(b.q, b.cache, scale=scale, softcap=softcap, out=out, **b.args())
    row = 0
    for s, c in enumerate(b.counts):
        rows = slice(row, row + c)
        want, tol = limited(b, s, rows, float(np.float32(softcap)), float(np.float32(scale)))
        ratio = (out[rows].double() - want).abs() / tol
        assert torch.isfinite(out[rows]).all() and float(ratio.max()) <= 1.0, f"softcap {softcap}, scale {scale}, sequence {s}: worst {float(ratio.max()):.3g} of the tolerance"
        row += c
    assert (out[row:] == 7.0).all()
    return out[:row]


# (rows * d above and below the border to the kernel of trees, which over 8 and 4 bits has the f32 results of the smaller one; a head that no two tiles of rows have room for)
SHAPES = [(128, 2, 4, [140, 1], [900, 30]), (64, 1, 2, [40, 3], [300, 700]), (256, 1, 2, [130], [400])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES)
def test_soft_limits(cuda, kind, act, shape):
    d, kv, group, counts, lens = shape
    b = Batch(cuda, 31, KINDS[kind], d, kv, group, 16, counts, lens, act, q_size=4.0)
    for limit in (1e-40, 1e-3, 1.0, 30.0, 300.0, 1e4, 1e6, 1e8, 1e30, 3e38, 3.4028234e38):
        check(b, limit)
    free = check(b).double()
    huge = check(b, 1e30).double()
    bound = sum(limited(b, 0, slice(0, counts[0]), c, d ** -0.5)[1] for c in (0.0, 1e30))
    assert ((free - huge).abs()[:counts[0]] <= bound).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES)
def test_scales_of_nothing(cuda, kind, act, shape):
    """A scale of zero is the mean of what a row sees; so is one that f32 does not hold beside the queries' powers of two, and one that holds but adds nothing to any score."""
    d, kv, group, counts, lens = shape
    b = Batch(cuda, 32, KINDS[kind], d, kv, group, 16, counts, lens, act)
    rows = sum(counts)
    for q_size, scale in ((1.0, 0.0), (1.0, -0.0), (1.0, 1e-30), (1e-6, 1e-37), (1e-6, 1e-42), (2.0 ** -20, -1e-40)):
        was = b.q
        b.q = (b.q * q_size).to(b.q.dtype)
        for softcap in (0.0, 5.0):
            check(b, softcap, scale)
        b.q = was
    mean = check(b, 0.0, 0.0)
    b.q = b.q * 0
    assert (check(b, 0.0, 1.0) == mean).all() and mean.shape[0] == rows
    # windows, sinks, missing pages: the mean of what is left
    b.table[0, 1] = -1
    for more in (dict(window=20), dict(sinks=b.torch.randn(kv * group, device="cuda"))):
        b.check(scale=0.0, **more)
    # a key that is no number: 0 times it is none either, for the rows that see it
    if KINDS[kind] == 0:
        for odd in (np.inf, -np.inf, np.nan):
            b.cache.k[b.table[0, 0].long(), 0, 3, 0] = odd
            assert not b.torch.isfinite(b.cuda.attention_chunk(b.q, b.cache, scale=0.0, **b.args())[:counts[0], :group]).any()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("d", [64, 128])
def test_two_tiles_of_rows_over_values_that_are_no_numbers(cuda, act, d):
    """f16 caches: values that are no numbers at later tokens of a long chunk, in every tile that only some rows of a block see. Both tiles of rows look for them in the same memory;
    rows that do not see them come out as from a clean cache, time after time."""
    b = Batch(cuda, 33, 0, d, 2, 4, 16, [700, 90], [900, 90], act)
    torch = b.torch
    clean = torch.empty(b.q.shape, device="cuda", dtype=torch.float16 if b.half else torch.float32)
    args = dict(scale=d ** -0.5, **b.args())
    cuda.attention_chunk(b.q, b.cache, out=clean, **args)
    odd = 200 + 64 * 5 + 3   # tokens before the 323rd of the first chunk do not see them
    p = torch.arange(odd, 900, 2, device="cuda")
    page = b.table[0].cuda()[p // 16].long()
    values = torch.tensor([np.inf, -np.inf, np.nan], device="cuda", dtype=torch.float16)
    b.cache.v[page, :, p % 16, 1::3] = values[torch.arange(len(p), device="cuda") % 3][:, None, None]
    out = torch.empty_like(clean)
    for _ in range(40):
        cuda.attention_chunk(b.q, b.cache, out=out, **args)
        assert (out[:odd - 200] == clean[:odd - 200]).all() and (out[700:790] == clean[700:790]).all()
        assert not torch.isfinite(out[odd - 200:700, :, 1::3]).any() and (out[odd - 200:700, :, 0::3] == clean[odd - 200:700, :, 0::3]).all()


@pytest.mark.parametrize("kind,act,d", [("f16", "f32", 128), ("f16", "f16", 64), ("q8", "f16", 128), ("q8", "f32", 128), ("q4", "f32", 64)])
def test_windows_wider_than_any_context(cuda, kind, act, d):
    """Up to the largest int, also where a sequence has more rows than positions, whose first rows lie before position 0."""
    for group in (1, 4):
        b = Batch(cuda, 34, KINDS[kind], d, 1, group, 16, [250, 300, 40, 1], [240, 20, 700, 300], act)
        free = b.check()
        for window in (2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30 + 1, 2 ** 30, 100000):
            got = b.check(window=window)
            assert ((got == 0) == (free == 0)).all()   # (the division of the work may be another one)
    few = Batch(cuda, 35, KINDS[kind], d, 1, 4, 16, [60, 5], [50, 300], "f32")
    tree = [cuda.attention_tree(few.q, few.cache, window=w, **few.args())[:65] for w in (0, 2 ** 31 - 1, 2 ** 30)]
    want, tol, _ = few.want(d ** -0.5)
    assert all(((t.double() - want[:65]).abs() <= tol[:65]).all() for t in tree)


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("d,group", [(64, 7), (96, 4), (128, 4), (128, 1)])
@pytest.mark.parametrize("window", [0, 200])
def test_scales_that_are_no_numbers(cuda, kind, d, group, window):
    """f32 results over 8 and 4 bits, more rows than go to the kernel of trees. Scales that are no numbers, and ones that take values beyond f16, where no row sees them (behind the last
    position, in unused pages, before the window, at later tokens of the chunk): the same bits as without them. Values that are no numbers reach the rows that see them, in their block
    of 32 alone."""
    b = Batch(cuda, 41, KINDS[kind], d, 2, group, 16, [301, 7, 1], [805, 500, 1003], "f32")
    torch = b.torch
    clean = b.check(window=window)
    first = 805 - 301
    keep = torch.zeros((b.cache.n_pages, 16), dtype=torch.bool)
    for s, (c, n) in enumerate(zip(b.counts, b.lens)):
        p = torch.arange(max(0, n - c + 1 - window) if window else 0, n)
        keep[b.table[s, p // 16].long(), p % 16] = True
    keep = keep.cuda()[:, None, :, None]
    odd = torch.tensor([np.nan, np.inf, -np.inf, 65504], dtype=torch.float16, device="cuda")
    for a in (b.cache.k_scale, b.cache.v_scale):
        a.copy_(torch.where(keep, a, odd[torch.randint(0, 4, a.shape, device="cuda")]))
    assert (b.check(window=window) == clean).all()

    def at(p):
        return b.table[0, p // 16].long(), 1, p % 16
    was_k, was_v = b.cache.k_scale.clone(), b.cache.v_scale.clone()
    heads = slice(group, 2 * group)   # of key head 1
    args = dict(scale=d ** -0.5, window=window, **b.args())
    # one token of the chunk after the other: in a tile's middle, at its ends, in the last one
    for i in (0, 1, 70, first % 64, 127, 200, 300):
        b.cache.v_scale[at(first + i)][0] = (np.inf, np.nan)[i & 1]
        out = cuda.attention_chunk(b.q, b.cache, **args)
        sees = torch.arange(301, device="cuda") >= i
        if window:
            sees &= torch.arange(301, device="cuda") < i + window
        assert (out[:301][~sees] == clean[:301][~sees]).all() and (out[301:309] == clean[301:309]).all() and (out[:301, :group] == clean[:301, :group]).all()
        assert (out[:301, heads, 32:] == clean[:301, heads, 32:]).all() and (~torch.isfinite(out[:301][sees][:, heads, :32])).any(-1).all()
        b.cache.v_scale.copy_(was_v)
    b.cache.k_scale[at(first + 100)][d // 32 - 1] = np.nan
    out = cuda.attention_chunk(b.q, b.cache, **args)
    assert (out[:100] == clean[:100]).all() and not torch.isfinite(out[100:301 if not window else 300][:, heads]).any()
    b.cache.k_scale.copy_(was_k)
    # beside a scale that takes a value beyond f16, which has the call done anew: what is no number stays where it was seen
    b.cache.v_scale[at(first + 150)][0], b.cache.v_scale[at(first + 20)][1] = np.inf, 60000.0
    out = cuda.attention_chunk(b.q, b.cache, **args)
    assert torch.isfinite(out[:150]).all() and (~torch.isfinite(out[150:301, heads, :32])).any(-1).all() and torch.isfinite(out[150:301, heads, 32:]).all()
    b.cache.v_scale[at(first + 150)][0] = was_v[at(first + 150)][0]
    b.check(window=window)
    b.cache.v_scale.copy_(was_v)
    assert (b.check(window=window) == clean).all() and cuda.device_status() == 0


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_more_rows_than_positions_and_missing_pages_in_two_terms(cuda, kind):
    """As test_gpu_attn_chunk.py's test of rows that see nothing, with more rows than go to the kernel of trees."""
    b = Batch(cuda, 42, KINDS[kind], 128, 1, 4, 16, [5, 3, 200, 140], [2, 0, 130, 40], "f32")
    got = b.check()
    assert (got[:3] == 0).all() and (got[5:78] == 0).all() and (got[208:308] == 0).all() and (got[308:] != 0).any(-1).all()
    assert (b.check(sinks=b.torch.randn(4, device="cuda"))[:3] == 0).all()
    b.lens[1] = -7
    b.check()
    b.check(window=40)
    b = Batch(cuda, 43, KINDS[kind], 128, 1, 4, 16, [150, 20], [600, 20], "f32")
    b.table[0, :5], b.table[0, 9], b.table[0, 20], b.table[1, 0] = -1, 1 << 30, b.cache.n_pages, -5
    assert (b.check()[150:150 + 16] == 0).all()
    b.check(window=40)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("d", [192, 256])
def test_long_heads_with_sinks_and_soft_limits(cuda, kind, act, d):
    b = Batch(cuda, 44, KINDS[kind], d, 2, 3, 32, [90, 1, 33], [700, 64, 33], act, q_size=4.0)
    sinks = 3 * b.torch.randn(6, device="cuda", generator=b.torch.Generator("cuda").manual_seed(1))
    sinks[1], sinks[2] = -np.inf, 60.0
    b.check(sinks=sinks)
    b.check(softcap=20.0, sinks=sinks, window=70)
    b.check(window=1, sinks=sinks)
    check(b, 1e8)

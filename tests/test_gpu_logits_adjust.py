"""Biases, penalties and grammar masks of logits: against the definition, step by step in f32, equal to the bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain(x, hist=None, hist_len=None, rep=None, freq=None, pres=None, bias_ids=None, bias=None, bias_len=None, mask=None, mask_row=None):
    y = np.array(x, np.float32)
    rows, n = y.shape
    f32 = np.float32
    with np.errstate(all="ignore"):
        for r in range(rows):
            if bias is not None:
                m = bias.shape[1] if bias_len is None else min(max(int(bias_len[r]), 0), bias.shape[1])
                for i, b in {int(i): b for i, b in zip(bias_ids[r, :m], bias[r, :m]) if 0 <= i < n}.items():
                    y[r, i] = f32(y[r, i] + b)
            if hist is not None:
                m = hist.shape[1] if hist_len is None else min(max(int(hist_len[r]), 0), hist.shape[1])
                ids, times = np.unique(hist[r, :m], return_counts=True)
                for i, c in zip(ids, times):
                    if not 0 <= i < n:
                        continue
                    v, p = y[r, i], f32(1 if rep is None else rep[r])
                    if p > 0 and p != 1:
                        v = f32(v / p) if v > 0 else f32(v * p)
                    y[r, i] = f32(v - f32(f32(f32(0 if freq is None else freq[r]) * f32(c)) + f32(0 if pres is None else pres[r])))
            if mask is not None:
                m = r if mask_row is None else int(mask_row[r])
                if 0 <= m < len(mask):
                    i = np.arange(n)
                    y[r, (mask[m].view(np.uint32)[i // 32] >> (i % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return y


def run(cuda, x, **k):
    import torch
    dev = {n: None if a is None else torch.from_numpy(a).cuda() for n, a in k.items()}
    xt = torch.from_numpy(x).cuda()
    got = cuda.logits_adjust(xt, **dev)
    want = plain(x, **k)
    assert got.cpu().numpy().tobytes() == want.tobytes() or np.array_equal(got.cpu().numpy(), want, equal_nan=True)
    assert (xt.cpu().numpy().view(np.uint32) == x.view(np.uint32)).all()
    assert cuda.logits_adjust(xt, out=xt, **dev) is xt
    assert np.array_equal(xt.cpu().numpy(), want, equal_nan=True)
    return want


def lists(rng, rows, n, hist, biases, masks):
    ids = lambda m: (n * rng.random((rows, m)) ** 4).astype(np.int32)  # noqa: E731
    k = dict(hist=ids(hist), hist_len=rng.integers(-1, hist + 3, rows).astype(np.int32), rep=rng.uniform(0.8, 1.5, rows).astype(np.float32),
             freq=rng.uniform(-0.5, 1, rows).astype(np.float32), pres=rng.uniform(-1, 1, rows).astype(np.float32))
    k["hist"][:, ::7] = rng.choice([-1, n, -5, 2 ** 31 - 1, 0, n - 1], (rows, len(k["hist"][0, ::7])))
    if biases:
        k |= dict(bias_ids=ids(biases), bias=rng.standard_normal((rows, biases)).astype(np.float32), bias_len=rng.integers(-1, biases + 2, rows).astype(np.int32))
    if masks:
        k |= dict(mask=rng.integers(-2 ** 31, 2 ** 31, (masks, (n + 31) // 32 + 1)).astype(np.int32), mask_row=rng.integers(-2, masks + 1, rows).astype(np.int32))
    return k


@pytest.mark.parametrize("rows,n,hist,biases,masks", [(1, 1, 3, 1, 1), (1, 128256, 700, 20, 1), (3, 32000, 64, 0, 0), (5, 1023, 4000, 9, 2), (4, 4097, 1, 5, 4), (2, 50257, 5000, 300, 1), (33, 8192, 30, 40, 7), (2, 3000, 70000, 3, 1), (300, 9001, 65535, 1000, 5), (2, 5000, 10, 65600, 0)])
def test_against_the_definition(cuda, rows, n, hist, biases, masks):
    rng = np.random.default_rng(n)
    run(cuda, 4 * rng.standard_normal((rows, n)).astype(np.float32), **lists(rng, rows, n, hist, biases, masks))


def test_each_part_alone(cuda):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 5000)).astype(np.float32)
    k = lists(rng, 3, 5000, 100, 50, 3)
    run(cuda, x)
    run(cuda, x, hist=k["hist"], pres=k["pres"])
    run(cuda, x, hist=k["hist"], hist_len=k["hist_len"], freq=k["freq"])
    run(cuda, x, hist=k["hist"], rep=np.array([0.0, -2.0, np.nan], np.float32))
    run(cuda, x, bias_ids=k["bias_ids"], bias=k["bias"])
    run(cuda, x, mask=k["mask"])
    run(cuda, x, mask=k["mask"][:2])   # the third row has none
    assert np.isneginf(run(cuda, x, mask=np.zeros((3, 157), np.int32))).all()


def test_counts_of_long_histories(cuda):
    """One id 65,535 times, and beside its bias; 70,000 times."""
    x = np.array([[1.5, -2.0, 0.25, 3.0]], np.float32)
    for times in (65535, 70000):
        hist = np.full((1, times), 2, np.int32)
        run(cuda, x, hist=hist, freq=np.array([0.5], np.float32), bias_ids=np.array([[2, 3, 2]], np.int32), bias=np.array([[9, 8, 7]], np.float32))


def test_infinities_nan_and_zeros(cuda):
    x = np.array([[np.inf, -np.inf, np.nan, 0.0, -0.0, 1.0, -1.0, 3e38]], np.float32)
    hist = np.array([[0, 1, 2, 3, 4, 5, 6, 7, 7, 7]], np.int32)
    one = np.ones(1, np.float32)
    run(cuda, x, hist=hist, rep=2 * one, freq=one, pres=0 * one)
    run(cuda, x, hist=hist, rep=0.5 * one)
    want = run(cuda, x, mask=np.array([[0b00111000]], np.int32), bias_ids=np.array([[3, 3, 3]], np.int32), bias=np.array([[1, np.nan, 5]], np.float32))
    assert want[0, 3] == 5.0 and np.isneginf(want[0, [0, 1, 2, 6, 7]]).all()


def test_rows_that_are_not_contiguous(cuda):
    """Rows off 16-byte boundaries, lists and masks that are slices of wider ones, one row without a batch."""
    import torch
    rng = np.random.default_rng(2)
    for width, first in ((5003, 0), (5004, 1), (5004, 0), (6000, 4)):
        wide = rng.standard_normal((3, width)).astype(np.float32)
        x = np.ascontiguousarray(wide[:, first:first + 4999])
        k = lists(rng, 3, 4999, 60, 20, 2)
        t = torch.from_numpy(wide).cuda()
        dev = {n: torch.from_numpy(a).cuda() for n, a in k.items()}
        dev["hist"] = torch.nn.functional.pad(dev["hist"], (0, 5))[:, :60]
        dev["bias"], dev["bias_ids"] = (torch.nn.functional.pad(dev[n], (3, 0))[:, 3:] for n in ("bias", "bias_ids"))
        assert not dev["hist"].is_contiguous() and not dev["bias"].is_contiguous()
        out = torch.full((3, width), 9.0, device="cuda")
        cuda.logits_adjust(t[:, first:first + 4999], out=out[:, first:first + 4999], **dev)
        assert np.array_equal(out[:, first:first + 4999].cpu().numpy(), plain(x, **k))
        assert (out[:, :first] == 9).all() and (out[:, first + 4999:] == 9).all()
    one = cuda.logits_adjust(t[0], hist=dev["hist"][:1], rep=dev["rep"][:1])
    assert one.shape == (width,) and np.array_equal(one.cpu().numpy(), plain(wide[:1], hist=k["hist"][:1], rep=k["rep"][:1])[0])


def test_before_the_top_k(cuda):
    """A row under a grammar, then ranked: only allowed tokens come out, the penalised one behind."""
    import torch
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal(40000).astype(np.float32)).cuda()
    ok = torch.zeros(40000, dtype=torch.bool)
    ok[::100] = True
    mask = (ok.view(-1, 32).long() << torch.arange(32)).sum(1).to(torch.uint32).view(1, -1).cuda()
    best = int(torch.where(ok.cuda(), x, -torch.inf).argmax())
    y = cuda.logits_adjust(x, mask=mask)
    ids, vals, mass = cuda.logits_topk(y, 5)
    assert int(ids[0]) == best and all(int(i) % 100 == 0 for i in ids) and torch.isfinite(mass).all()
    y = cuda.logits_adjust(x, hist=torch.tensor([[best, best]], dtype=torch.int32, device="cuda"), pres=torch.full((1,), 100.0, device="cuda"), mask=mask)
    assert best not in cuda.logits_topk(y, 5)[0].tolist()


@pytest.mark.parametrize("rows,n", [(1, 1000), (70, 40000)])
def test_lists_that_are_not_there(cuda, rows, n):
    """Sizes, strides and other parts of a list whose pointer is NULL are not looked at."""
    import ctypes as C

    import torch
    x = torch.from_numpy(np.random.default_rng(n).standard_normal((rows, n)).astype(np.float32)).cuda()
    ones = torch.ones(rows, device="cuda")
    ids = torch.zeros((rows, 8), dtype=torch.int32, device="cuda")
    a = cuda.Adjust(n_rows=rows, n_vocab=n, stride=n, out_stride=n, hist_n=4096, hist_stride=4096, rep=ones.data_ptr(), freq=ones.data_ptr(), pres=ones.data_ptr(),
                    bias_ids=ids.data_ptr(), bias_n=8, bias_stride=8, mask_row=ids.data_ptr(), n_masks=3, mask_stride=0)
    out = torch.empty_like(x)
    assert cuda.lib.krk_cuda_logits_adjust(out.data_ptr(), x.data_ptr(), C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, x)


def test_masks_narrower_than_a_row(cuda):
    import torch
    x = torch.zeros((2, 1000), device="cuda")
    table = torch.full((2, 64), -1, dtype=torch.int32, device="cuda")
    for mask in (table[:, 40:], table[:, :31], table[1:, 33:64]):   # 24, 31 and 31 words where 32 are read; rows 64 apart
        with pytest.raises(ValueError):
            cuda.logits_adjust(x, mask=mask)
    assert torch.equal(cuda.logits_adjust(x, mask=table[:, 32:]), x)

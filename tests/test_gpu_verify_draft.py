"""Verification of drafted tokens, against the rule in 64 bits: what is accepted and drawn has to be equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def softmax(x, t):
    with np.errstate(all="ignore"):
        z = (x.astype(np.float64) - x.max()) / t
        e = np.exp(z)
        return e / e.sum(), z - np.log(e.sum())


def plain(x, start, draft, au, su, q=None, temp=None, draft_temp=None, fill=-9):
    tokens, count, lp = np.full(len(x), fill), np.zeros(len(start) - 1, int), np.full(len(x), float(fill))
    for s in range(len(start) - 1):
        rows = range(start[s], start[s + 1])
        t = 1.0 if temp is None else float(temp[s])
        tq = t if draft_temp is None else float(draft_temp[s])
        for j, r in enumerate(rows):
            p, log_p = softmax(x[r], t if t > 0 else 1.0)
            d, last = draft[r], r == rows[-1]
            there = 0 <= d < x.shape[1]
            if t <= 0:
                best = np.flatnonzero(x[r] == np.fmax.reduce(x[r]))
                best = int(best[0]) if len(best) and np.fmax.reduce(x[r]) > -np.inf else -1
                ok, token = d == best, best
            else:
                w = p.copy()
                ok = False
                if not last:
                    if q is None:
                        ok = there and au[r] * 1.0 < p[d]
                        if there:
                            w[d] = 0
                    else:
                        pq, _ = softmax(q[r], tq if tq > 0 else 1.0)
                        ok = there and np.float64(au[r]) * pq[d] < p[d]
                        w = np.maximum(p - pq, 0)
                    if not w.sum() > 0:
                        w = p
                c = np.cumsum(w)
                over = np.flatnonzero((c > np.float64(su[s]) * c[-1]) & (w > 0)) if c[-1] > 0 else []
                token = int(over[0]) if len(over) else int(np.flatnonzero(w > 0)[-1]) if c[-1] > 0 else -1
            if ok and not last:
                tokens[r], lp[r] = d, log_p[d]
                continue
            tokens[r], lp[r] = token, log_p[token] if token >= 0 else 0.0
            tokens[r + 1:rows[-1] + 1], lp[r + 1:rows[-1] + 1] = -1, 0.0
            count[s] = j
            break
    return tokens, count, lp


def run(cuda, x, start, draft, au, su, skew=0, **more):
    import torch
    x = np.asarray(x, np.float32)
    want = plain(x, start, draft, au, su, **more)

    def dev(a):
        t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
        if skew and a.ndim == 2:
            wide = torch.zeros((a.shape[0], a.shape[1] + 2 * skew), device="cuda")
            wide[:, skew:skew + a.shape[1]] = t
            return wide[:, skew:skew + a.shape[1]]
        return t
    outs = dict(tokens=torch.full((len(x),), -9, dtype=torch.int32, device="cuda"), logprob=torch.full((len(x),), -9.0, device="cuda"))
    more = {{"q": "draft_logits"}.get(k, k): dev(np.asarray(v, np.float32)) for k, v in more.items()}
    tokens, count, lp = cuda.verify_draft(dev(x), dev(np.asarray(start, np.int32)), dev(np.asarray(draft, np.int32)), dev(np.asarray(au, np.float32)),
                                          dev(np.asarray(su, np.float32)), **outs, **more)
    assert (tokens.cpu().numpy() == want[0]).all(), (tokens.cpu().numpy(), want[0])
    assert (count.cpu().numpy() == want[1]).all()
    # the greatest logit's sum of exponentials: f32 ones, 2^-21 relative and the argument's rounding, 2^-23 of the range times 1 / T at most where they count
    lp = lp.cpu().numpy().astype(np.float64)
    ok = np.isfinite(want[2])
    assert (np.isfinite(lp) == ok).all()
    assert (np.abs(lp - want[2])[ok] <= 2.0 ** -23 * np.abs(want[2][ok]) + 2.0 ** -18).all()
    return want


def batch(seed, counts, vocab, spread=3.5, near=0.7, drafter=True):
    rng = np.random.default_rng(seed)
    start = np.concatenate([[0], np.cumsum(np.array(counts) + 1)])
    rows = int(start[-1])
    x = (spread * rng.standard_normal((rows, vocab))).astype(np.float32)
    temp = rng.uniform(0.5, 1.2, len(counts)).astype(np.float32)
    q = x + (near * rng.standard_normal(x.shape)).astype(np.float32) if drafter else None
    draft = (q if drafter else x).argmax(1)
    other = rng.random(rows) < 0.3
    draft[other] = rng.integers(0, vocab, other.sum())
    return x, start, draft, rng.random(rows).astype(np.float32), rng.random(len(counts)).astype(np.float32), temp, q


@pytest.mark.parametrize("vocab", [1, 2, 5, 31, 32, 33, 1000, 4096, 4099, 8192, 8193, 50001, 128256])
@pytest.mark.parametrize("drafter", [True, False])
def test_vocabularies(cuda, vocab, drafter):
    accepted = 0
    for seed in range(3 if vocab > 10000 else 8):
        x, start, draft, au, su, temp, q = batch(seed, [0, 1, 3, 7, 2], vocab, drafter=drafter)
        more = dict(q=q) if drafter else {}
        accepted += run(cuda, x, start, draft, au, su, temp=temp, **more)[1].sum()
        run(cuda, x, start, draft, au, su, skew=1, **more)
    assert accepted > 0


def test_flat_rows(cuda):
    """Every token as likely as the next: the number falls among a hundred thousand equal weights."""
    for seed in range(6):
        x, start, draft, au, su, temp, q = batch(seed, [2, 2], 100003, spread=0.0, near=1e-3)
        run(cuda, x, start, draft, au * 0.5, su, q=q)
        run(cuda, x, start, draft, au, su)


def test_temperatures(cuda):
    """Greedy requests, with ties; temperatures of their own for the drafter; very low and high ones."""
    x, start, draft, au, su, temp, q = batch(1, [4, 4, 4, 4, 4, 4], 3000)
    temp[:] = [0.0, -1.0, 1e-3, 50.0, 0.7, 0.7]
    x[start[0], [5, 900]] = 40.0
    draft[start[0]] = 5
    x[start[1], [5, 900]] = 40.0
    draft[start[1]] = 900
    run(cuda, x, start, draft, au, su, temp=temp, q=q)
    run(cuda, x, start, draft, au, su, temp=temp)
    run(cuda, x, start, draft, au, su, temp=temp, q=q, draft_temp=temp[::-1].copy())


def test_temperatures_near_zero(cuda):
    """Positive temperatures down to the smallest normal one: all the weight on the greatest value, or shared by those that tie, wherever the row lies."""
    for i, t in enumerate((1e-6, 1e-20, 1e-30, 1.2e-38)):
        x, start, draft, au, su, temp, q = batch(20 + i, [4, 4, 1, 2], 5000)
        x += np.float32(17.3)
        q -= np.float32(5.1)
        x[start[1], [3, 4100]] = 90.0
        draft[::2] = x.argmax(1)[::2]
        run(cuda, x, start, draft, au * 0.5, su, temp=0 * temp + np.float32(t), q=q)
        run(cuda, x, start, draft, au * 0.5, su, temp=0 * temp + np.float32(t))
        run(cuda, x, start, draft, au, su, temp=temp, draft_temp=0 * temp + np.float32(t), q=q)


def test_numbers_at_their_ends(cuda):
    """0 accepts whatever the target has, 1 and the largest number below it draw the last token there is; equal models accept everything."""
    x, start, draft, au, su, temp, q = batch(2, [5, 5], 4000)
    run(cuda, x, start, draft, 0 * au, 0 * su, q=q)
    for v in (1.0, 1.0 - 2.0 ** -24):
        run(cuda, x, start, draft, 0 * au + v, 0 * su + v, q=q)
        run(cuda, x, start, draft, 0 * au + v, 0 * su + v)
    assert (run(cuda, x, start, draft, au, su, q=x)[1] == 5).all()
    x[:, 100:] = -np.inf   # tokens that a mask took out
    draft[:] = np.minimum(draft, 120)
    run(cuda, x, start, draft, 0 * au, su, q=q)
    run(cuda, x, start, draft, au, 0 * su + 1.0)


def test_rows_that_are_none(cuda):
    """NaN, infinities, nothing but -infinity, drafted ids outside the vocabulary, sequences without rows, rows of no sequence."""
    x, start, draft, au, su, temp, q = batch(3, [3] * 8, 9000)
    x[start[0] + 1, 77] = np.nan
    x[start[1], 8500] = np.inf
    x[start[2] + 2] = -np.inf
    q[start[3], 5] = np.nan
    q[start[4]] = -np.inf
    draft[start[5]], draft[start[6] + 1], draft[start[7]] = -1, 9000, 2 ** 31 - 1
    au *= 0.01
    run(cuda, x, start, draft, au, su, q=q)
    run(cuda, x, start, draft, au, su)
    run(cuda, x, start, draft, au, su, temp=0 * su)
    keep = [0, 0, start[1], start[1], start[3], start[3], start[4], start[4], start[4]]
    run(cuda, x, keep, draft, au, np.resize(su, 8), q=q)


def test_many_rows_and_capture(cuda):
    """More drafted tokens than warps; the same call captured, replayed on other numbers."""
    import torch
    x, start, draft, au, su, temp, q = batch(4, [40, 0, 20], 2000, near=0.1)
    want = run(cuda, x, start, draft, 0.3 * au, su, q=q)
    assert want[1].max() > 16
    dev = lambda a, t=None: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()  # noqa: E731
    numbers, drafter = dev(au), dev(q)
    args = (dev(x), dev(start, np.int32), dev(draft, np.int32), numbers, dev(su))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, count, _ = cuda.verify_draft(*args, draft_logits=drafter)
    numbers.mul_(0.3)
    graph.replay()
    assert (tokens.cpu().numpy() == want[0]).all() and (count.cpu().numpy() == want[1]).all()
    tokens, count, lp = cuda.verify_draft(torch.zeros((0, 10), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), *(torch.zeros(n, dtype=t, device="cuda") for n, t in
                                          ((0, torch.int32), (0, torch.float32), (3, torch.float32))))
    assert count.tolist() == [0, 0, 0] and tokens.shape == (0,)


def test_what_comes_out_has_the_targets_distribution(cuda):
    """20,000 requests of one drafted token over six ids: the first token that comes out, whoever chose it, is distributed as the target's."""
    import torch
    gen = torch.Generator("cuda").manual_seed(5)
    n, vocab = 20000, 6
    p, q = torch.randn(vocab, device="cuda", generator=gen), torch.randn(vocab, device="cuda", generator=gen)
    logits, drafter = p.repeat(2 * n, 1), q.repeat(2 * n, 1)
    draft = torch.multinomial(torch.softmax(q, 0).repeat(2 * n, 1), 1, generator=gen)[:, 0].int()
    start = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    u = torch.rand(2 * n, device="cuda", generator=gen)
    tokens, count, _ = cuda.verify_draft(logits, start, draft, u, torch.rand(n, device="cuda", generator=gen), draft_logits=drafter)
    got = torch.bincount(tokens[::2].long(), minlength=vocab).double() / n
    want = torch.softmax(p.double(), 0)
    # five standard deviations of a count
    assert ((got - want).abs() <= 5 * (want * (1 - want) / n).sqrt()).all()
    assert abs(float(count.double().mean()) - float(torch.minimum(want, torch.softmax(q.double(), 0)).sum())) < 5 * 0.5 / n ** 0.5

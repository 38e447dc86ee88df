"""Verification where the drafter took its greatest value (a draft_temp of 0 or less): q is 1 at it. The rule in 64 bits is that of test_gpu_verify_draft.py, whose form of a
drafter's row in a softmax is given one for these requests: a row whose softmax is that distribution."""
import numpy as np
import pytest

import test_gpu_verify_draft as base

pytestmark = pytest.mark.gpu


def one_hot(q, start, draft_temp):
    """The drafter's rows with those of greedy ones made -infinity but at the lowest of the greatest values (NaN passed over); and temperatures above 0 in their place."""
    q, t = q.copy(), np.array(draft_temp, np.float32)
    for s in np.flatnonzero(~(t > 0)):
        for r in range(start[s], start[s + 1]):
            top = np.fmax.reduce(q[r])
            at = int(np.flatnonzero(q[r] == top)[0]) if top > -np.inf else None
            q[r] = -np.inf
            if at is not None:
                q[r, at] = 0.0
        t[s] = 1.0
    return q, t


def run(cuda, x, start, draft, au, su, q, temp, draft_temp, skew=0):
    """The call with what it is given, against the plain rule over the rows that one_hot makes."""
    import torch
    q1, t1 = one_hot(q, start, draft_temp)
    want = base.plain(np.asarray(x, np.float32), start, draft, au, su, q=q1, temp=temp, draft_temp=t1)

    def dev(a, t):
        a = torch.from_numpy(np.ascontiguousarray(a, t)).cuda()
        if skew and a.dim() == 2:
            wide = torch.zeros((a.shape[0], a.shape[1] + 3), device="cuda")
            wide[:, 1:-2] = a
            return wide[:, 1:-2]
        return a
    f, i = np.float32, np.int32
    tokens, count, lp = cuda.verify_draft(dev(x, f), dev(start, i), dev(draft, i), dev(au, f), dev(su, f), draft_logits=dev(q, f), temp=None if temp is None else dev(temp, f),
                                          draft_temp=dev(draft_temp, f))
    assert (tokens.cpu().numpy() == want[0]).all(), (tokens.cpu().numpy(), want[0])
    assert (count.cpu().numpy() == want[1]).all()
    lp = lp.cpu().numpy().astype(np.float64)
    ok = np.isfinite(want[2])
    assert (np.isfinite(lp) == ok).all()
    assert (np.abs(lp - want[2])[ok] <= 2.0 ** -23 * np.abs(want[2][ok]) + 2.0 ** -18).all()   # as there
    return want


@pytest.mark.parametrize("vocab", [1, 2, 33, 3000, 8193, 128256])
def test_greedy_drafters(cuda, vocab):
    """Greedy drafters beside others and beside greedy requests; drafted tokens that are the greatest, and others, of which such a drafter says 0."""
    accepted = refused = 0
    for seed in range(6):
        x, start, draft, au, su, temp, q = base.batch(40 + seed, [4, 4, 1, 0, 4, 7], vocab, spread=2.0 if vocab > 100 else 3.5)
        x[start[0], draft[start[0]]] += 9.0   # (one of some weight)
        draft_temp = np.array([0.0, -1.0, 0.0, 0.0, 0.8, -0.0], np.float32)
        temp[seed % 6] = 0.0
        want = run(cuda, x, start, draft, 0.2 * au, su, q, temp, draft_temp, skew=seed & 1)
        run(cuda, x, start, draft, au, su, q, None, draft_temp)
        accepted += want[1].sum()
        refused += (want[1] < np.diff(start) - 1).sum()
    assert accepted > 0 and (refused > 0 or vocab == 1)


def test_ties_and_rows_that_are_none(cuda):
    """The lowest of greatest values that tie; NaN is passed over; nothing but -infinity, or NaN: nothing is accepted, the token is p's; infinities are the greatest; a token that has all
    of p's weight and is refused."""
    x, start, draft, au, su, temp, q = base.batch(60, [3] * 8, 9000, spread=1.0)
    draft_temp = np.zeros(8, np.float32)
    q[start[0], [50, 8999]] = 30.0
    draft[start[0]] = 50
    q[start[1], [50, 8500]] = 30.0
    draft[start[1]] = 8500
    q[start[2], 7], q[start[2] + 1, 8000] = np.nan, np.nan
    q[start[3]] = -np.inf
    q[start[4]] = np.nan
    q[start[5], 4444] = np.inf
    draft[start[5]] = 4444
    x[start[6]] = -np.inf
    x[start[6], 17] = 1.0
    q[start[6], 17] = 30.0
    draft[start[6]] = 17
    au[start[6]] = 1.0   # (1 < 1: refused, and nothing else is left)
    draft[start[7]] = -1
    for low in (1.0, 1e-4):
        u = low * au
        u[start[6]] = 1.0
        run(cuda, x, start, draft, u, su, q, temp, draft_temp)
        run(cuda, x, start, draft, u, 0 * su + np.float32(1 - 2.0 ** -24), q, temp, draft_temp)


def test_other_temperatures(cuda):
    """What test_gpu_verify_draft.py tries of temperatures, with drafters' of their own that are above 0."""
    x, start, draft, au, su, temp, q = base.batch(1, [4, 4, 4, 4, 4, 4], 3000)
    temp[:] = [0.0, -1.0, 1e-3, 50.0, 0.7, 0.7]
    x[start[0], [5, 900]] = 40.0
    draft[start[0]] = 5
    x[start[1], [5, 900]] = 40.0
    draft[start[1]] = 900
    base.run(cuda, x, start, draft, au, su, temp=temp, q=q)
    base.run(cuda, x, start, draft, au, su, temp=temp)
    base.run(cuda, x, start, draft, au, su, temp=temp, q=q, draft_temp=np.array([0.7, 0.7, 50.0, 1e-3, 1.0, 0.6], np.float32))


def test_what_comes_out_of_a_greedy_drafter_has_the_targets_distribution(cuda):
    """20,000 requests whose drafter took its greatest of six ids."""
    import torch
    gen = torch.Generator("cuda").manual_seed(6)
    n, vocab = 20000, 6
    p, q = torch.randn(vocab, device="cuda", generator=gen), torch.randn(vocab, device="cuda", generator=gen)
    start = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    draft = q.argmax().int().repeat(2 * n)
    tokens, count, _ = cuda.verify_draft(p.repeat(2 * n, 1), start, draft, torch.rand(2 * n, device="cuda", generator=gen), torch.rand(n, device="cuda", generator=gen),
                                         draft_logits=q.repeat(2 * n, 1), draft_temp=torch.zeros(n, device="cuda"))
    got = torch.bincount(tokens[::2].long(), minlength=vocab).double() / n
    want = torch.softmax(p.double(), 0)
    # five standard deviations of a count
    assert ((got - want).abs() <= 5 * (want * (1 - want) / n).sqrt()).all()
    assert abs(float(count.double().mean()) - float(want[int(q.argmax())])) < 5 * 0.5 / n ** 0.5

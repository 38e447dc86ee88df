"""The plan of a step from its requests' lengths, against a plain loop over the sequences."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain(before, new, table, free, n_free, page, room):
    stack = list(free[:max(0, min(n_free, len(free)))])
    taken = missing = 0
    table, pos, slots, start, length, last = table.copy(), [], [], [0], [], []
    wanted = 0
    for s, (b, c) in enumerate(zip(np.maximum(before, 0).tolist(), np.maximum(new, 0).tolist())):
        wanted += c
        c = min(c, room - len(pos))
        for i in range(-(-b // page), -(-(b + c) // page)):
            if i >= table.shape[1]:
                missing += 1
                continue
            missing += not stack
            taken += bool(stack)
            table[s, i] = stack.pop() if stack else -1
        for p in range(b, b + c):
            pos.append(p)
            t = table[s, p // page] if p // page < table.shape[1] else -1
            slots.append(int(t) * page + p % page if t >= 0 else -1)
        start.append(len(pos))
        length.append(b + c)
        last.append(len(pos) - 1 if c else -1)
    n = len(pos)
    return (start, length, pos + [0] * (room - n), slots + [-1] * (room - n), last, [len(stack), missing, n, wanted - n], table)


def run(cuda, before, new, table, free, n_free, page, room, **more):
    import torch
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    args = (i32(before), i32(new), i32(table), i32(free), i32([n_free]), page, room)
    got = cuda.step_plan(*args, **more)
    want = plain(np.asarray(before), np.asarray(new), np.asarray(table, np.int32), np.asarray(free), n_free, page, room)
    for name, g, w in zip(got._fields, got, want):
        assert g.dtype == (torch.int64 if name == "slots" else torch.int32)
        assert (g.cpu().numpy() == np.asarray(w)).all(), name
    again = cuda.step_plan(*args, out=got)
    for name, g, w in zip(got._fields, again, want):
        assert (g.cpu().numpy() == np.asarray(w)).all(), f"{name}, a second time"
    assert all(a is b for a, b in zip(again, got))
    return got


@pytest.mark.parametrize("n_seq,most,context,page,spare", [(1, 1, 0, 16, 0), (1, 3000, 5000, 16, 0), (8, 4, 2000, 16, 1), (3, 1, 40, 1, 2), (300, 50, 700, 48, 0),
                                                           (1500, 3, 100, 16, 5), (2500, 1, 64, 32, 0), (40, 500, 1000, 64, -30), (1100, 2, 30, 16, -200)])
@pytest.mark.parametrize("share", [1.0, 0.6, 1.7])
def test_batches(cuda, n_seq, most, context, page, spare, share):
    """Buffers that are full, cut the batch short, or have room behind it; stacks with too few pages."""
    rng = np.random.default_rng(n_seq + most)
    before, new = rng.integers(0, context + 1, n_seq), rng.integers(0, most + 1, n_seq)
    new[0] = most
    have, need = -(-before // page), -(-(before + new) // page)
    width = int(need.max())
    order = rng.permutation(int(need.sum()) + 40)
    table = np.full((n_seq, max(width, 1)), -1, np.int32)
    table[np.arange(table.shape[1]) < have[:, None]] = order[:have.sum()]
    free = order[have.sum():]
    run(cuda, before, new, table, free, max(0, int((need - have).sum()) + spare), page, int(new.sum() * share))


def test_edges(cuda):
    """Negative lengths, a stack whose number is out of its range, a table that is too narrow, an old page that is none, no tokens, no sequences."""
    t = np.arange(6).reshape(2, 3)
    run(cuda, [-5, 20], [3, -1], t, [7, 8], 2, 16, 5)
    run(cuda, [0, 0], [100, 20], t, [7, 8], 9, 16, 120)
    run(cuda, [0, 0], [100, 20], t, [7, 8], -4, 16, 120)
    run(cuda, [40, 3], [30, 50], np.where(t == 2, -1, t), [9, 10, 11], 3, 16, 80)
    run(cuda, [0, 5], [0, 0], t, [7], 1, 16, 4)
    run(cuda, [0, 5], [4, 4], t, [7, 8], 2, 16, 0)
    run(cuda, [2 ** 31 - 3], [2], np.zeros((1, 1)), [1], 1, 2 ** 20, 4)
    run(cuda, [], [], np.zeros((0, 3)), [1], 1, 16, 3)
    run(cuda, [3], [2], np.zeros((1, 0)), [1], 1, 16, 3)
    run(cuda, [3, 16], [2, 2], t, [], 0, 16, 4)


def test_capture(cuda):
    """A captured plan replays on other lengths."""
    import torch
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    before, new, table, free, n_free = i32(3, 14), i32(1, 5), torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), i32(5, 6, 7, 8), i32(4)
    table[:, 0] = i32(1, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = cuda.step_plan(before, new, table, free, n_free, 16, 12)
    new.copy_(i32(9, 2))
    graph.replay()
    assert plan.kv_len.tolist() == [12, 16] and plan.counts.tolist() == [4, 0, 11, 0] and plan.slots.tolist() == list(range(19, 28)) + [46, 47, -1]
    # the next step goes on from where this one came to
    before.copy_(plan.kv_len), n_free.copy_(plan.counts[:1]), new.copy_(i32(5, 1))
    graph.replay()
    assert plan.positions.tolist() == [12, 13, 14, 15, 16, 16, 0, 0, 0, 0, 0, 0] and plan.slots.tolist() == [28, 29, 30, 31, 128, 112] + [-1] * 6
    assert table.tolist() == [[1, 8, -1, -1], [2, 7, -1, -1]] and plan.counts.tolist() == [2, 0, 6, 0]


def test_two_plans_in_turn(cuda):
    """A plan's lengths and counts are the next one's input where they lie; one plan in the place of its own is refused."""
    import torch
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table, free = torch.full((3, 40), -1, dtype=torch.int32, device="cuda"), torch.arange(100, dtype=torch.int32, device="cuda")
    new = [i32(30, 1, 7), i32(5, 16, 0), i32(1, 1, 400)]
    plans = [cuda.step_plan(i32(0, 0, 0), new[0], table, free, i32(100), 16, 50)]
    plans.append(cuda.step_plan(plans[0].kv_len, new[1], table, free, plans[0].counts[:1], 16, 50))
    cuda.step_plan(plans[1].kv_len, new[2], table, free, plans[1].counts[:1], 16, 500, out=None)
    want = cuda.step_plan(plans[1].kv_len, i32(1, 1, 43), table.clone(), free, plans[1].counts[:1], 16, 50)
    got = cuda.step_plan(plans[1].kv_len, i32(1, 1, 43), table, free, plans[1].counts[:1], 16, 50, out=plans[0]._replace(page_table=table))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert got.kv_len.tolist() == [36, 18, 50] and got.counts[0].item() == 100 - 3 - 2 - 4
    for bad in (dict(kv_before=got.kv_len), dict(n_free=got.counts[:1]), dict(n_new=got.last)):
        args = {**dict(kv_before=plans[1].kv_len, n_new=new[0], n_free=plans[1].counts[:1]), **bad}
        with pytest.raises((ValueError, cuda.KrkCudaError)):
            cuda.step_plan(args["kv_before"], args["n_new"], table, free, args["n_free"], 16, 50, out=got)

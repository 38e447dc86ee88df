"""What the entry points of a step of prompts and drafted tokens refuse, on the host: nothing is launched."""
import ctypes as C

import pytest

from kraken_b200 import capi
from test_step_refusals import EALIGN, EARG, EDTYPE, ENULL, ESHAPE, L, P, attention, cache, nothing_launched  # noqa: F401


def step(**k):
    f = dict(kv_before=P, n_new=P, page_table=P, free_pages=P, n_free=P, q_start=P, kv_len=P, last=P, positions=P, slots=P, counts=P, max_tok=10, free_cap=4, n_seq=2, table_width=3,
             page_size=16)
    return capi.Step(*[{**f, **k}[n] for n, _ in capi.Step._fields_])


def norm(**k):
    f = dict(residual=P, gate=P, post_weight=P, weight=P, rows=2, n=100, x_stride=100, residual_stride=100, gate_stride=0, h_stride=100, y_stride=100, post_norm=1, y_dtype=0,
             alpha=1.0, eps=1e-6, offset=0.0)
    return capi.Norm(*[{**f, **k}[n] for n, _ in capi.Norm._fields_])


def verify(**k):
    f = dict(row_start=P, draft=P, accept_u=P, sample_u=P, temp=0, draft_temp=0, draft_logits=P, n_rows=6, n_vocab=100, stride=100, draft_stride=100, n_seq=2)
    return capi.Verify(*[{**f, **k}[n] for n, _ in capi.Verify._fields_])


@pytest.mark.parametrize("rc,k", [
    (ESHAPE, dict(n_seq=-1)), (ESHAPE, dict(n_heads=33)), (ESHAPE, dict(n_heads=0)), (ESHAPE, dict(max_q=-1)), (ESHAPE, dict(max_q=1 << 25)), (ESHAPE, dict(table_width=0)),
    (ESHAPE, dict(max_kv_len=1601)), (ESHAPE, dict(q_stride=4092)), (ESHAPE, dict(out_stride=4092)), (EALIGN, dict(q_stride=4098)), (EALIGN, dict(out_stride=4097)),
    (EARG, dict(window=-1)), (EARG, dict(softcap=-1.0)), (EARG, dict(softcap=float("inf"))), (EARG, dict(softcap=float("nan"))), (EARG, dict(tree=P)), (ENULL, dict(q_start=0)),
    (ENULL, dict(kv_len=0)), (ENULL, dict(page_table=0)), (EALIGN, dict(q_start=P + 2)), (EALIGN, dict(sinks=P + 1))])
def test_chunks(rc, k):
    a = attention(**{**dict(max_q=500), **k})
    assert L.krk_cuda_attention_chunk(P, 0, P, 0, C.byref(cache()), C.byref(a), P, 1 << 40, None) == rc


def test_chunk_types_and_pointers():
    c, a = C.byref(cache()), C.byref(attention(max_q=500))
    for out, q in ((0, 1), (2, 0), (0, 2), (-1, 0)):
        assert L.krk_cuda_attention_chunk(P, out, P, q, c, a, P, 1 << 40, None) == EARG
    assert L.krk_cuda_attention_chunk(None, 0, P, 0, c, a, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_attention_chunk(P, 0, None, 0, c, a, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_attention_chunk(P, 0, P, 0, None, a, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_attention_chunk(P, 0, P, 0, c, None, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_attention_chunk(P + 8, 1, P, 1, c, a, P, 1 << 40, None) == EALIGN
    assert L.krk_cuda_attention_chunk(P, 1, P, 1, c, C.byref(attention(max_q=500, q_stride=4100)), P, 1 << 40, None) == EALIGN
    assert L.krk_cuda_attention_chunk(P, 1, P, 0, c, C.byref(attention(max_q=500, out_stride=4100)), P, 1 << 40, None) == EALIGN
    assert L.krk_cuda_attention_chunk(P, 0, P, 0, C.byref(cache(type=5)), a, P, 1 << 40, None) == EDTYPE
    assert L.krk_cuda_attention_chunk(P, 0, P, 0, C.byref(cache(head_dim=160)), a, P, 1 << 40, None) == ESHAPE
    assert L.krk_cuda_attention_chunk_workspace_bytes(c, C.byref(attention(tree=P)), 0) == 0
    for k in (dict(n_seq=0), dict(max_q=0)):   # nothing to do
        assert L.krk_cuda_attention_chunk(None, 0, None, 0, c, C.byref(attention(**k)), None, 0, None) == 0


@pytest.mark.parametrize("rc,k", [
    (ESHAPE, dict(n_seq=-1)), (ESHAPE, dict(table_width=-1)), (ESHAPE, dict(page_size=0)), (ESHAPE, dict(max_tok=-1)), (ESHAPE, dict(max_tok=1 << 31)), (ESHAPE, dict(free_cap=-1)),
    (EALIGN, dict(slots=P + 4)), (EALIGN, dict(counts=P + 2)), *[(ENULL, {n: 0}) for n, t in capi.Step._fields_ if t is C.c_void_p]])
def test_plans(rc, k):
    assert L.krk_cuda_step_plan(C.byref(step(**k)), None) == rc


def test_plan_without_a_struct():
    assert L.krk_cuda_step_plan(None, None) == ENULL


@pytest.mark.parametrize("rc,k", [
    (EARG, dict(y_dtype=2)), (ESHAPE, dict(rows=-1)), (ESHAPE, dict(n=-1)), (ESHAPE, dict(n=65537)), (ESHAPE, dict(x_stride=99)), (ESHAPE, dict(y_stride=99)), (ESHAPE, dict(h_stride=99)),
    (ESHAPE, dict(residual_stride=99)), (ESHAPE, dict(gate_stride=50)), (ESHAPE, dict(gate_stride=-1)), (EARG, dict(eps=-1.0)), (EARG, dict(eps=float("nan"))),
    (EALIGN, dict(weight=P + 2)), (EALIGN, dict(gate=P + 1))])
def test_norms(rc, k):
    assert L.krk_cuda_block_norm(P, P + 0x1000, P + 0x2000, C.byref(norm(**k)), None) == rc


def test_norm_pointers():
    X = P + 0x10000
    assert L.krk_cuda_block_norm(P, None, X, None, None) == ENULL
    assert L.krk_cuda_block_norm(None, None, X, C.byref(norm()), None) == ENULL
    assert L.krk_cuda_block_norm(P, None, None, C.byref(norm()), None) == ENULL
    assert L.krk_cuda_block_norm(P + 1, None, X, C.byref(norm(y_dtype=1)), None) == EALIGN
    assert L.krk_cuda_block_norm(P, X, X, C.byref(norm(h_stride=104)), None) == EARG       # h in x's place under another stride
    assert L.krk_cuda_block_norm(X, P, X + 8, C.byref(norm(h_stride=104)), None) == EARG   # in the residual's
    for k in (dict(rows=0), dict(n=0)):
        assert L.krk_cuda_block_norm(None, None, None, C.byref(norm(**k)), None) == 0


@pytest.mark.parametrize("rc,k", [
    (ESHAPE, dict(n_seq=-1)), (ESHAPE, dict(n_rows=-1)), (ESHAPE, dict(n_rows=(1 << 24) + 1)), (ESHAPE, dict(n_vocab=-1)), (ESHAPE, dict(n_vocab=(1 << 30) + 1, stride=1 << 31)),
    (ESHAPE, dict(stride=99)), (ESHAPE, dict(draft_stride=99)), (ENULL, dict(row_start=0)), (ENULL, dict(draft=0)), (ENULL, dict(accept_u=0)), (ENULL, dict(sample_u=0)),
    (EALIGN, dict(temp=P + 2)), (EALIGN, dict(draft_logits=P + 1))])
def test_verifications(rc, k):
    assert L.krk_cuda_verify_draft(P, P, P, P, C.byref(verify(**k)), P, 1 << 40, None) == rc


def test_verification_pointers():
    v = C.byref(verify())
    assert L.krk_cuda_verify_draft(P, P, P, P, None, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_verify_draft(None, P, P, P, v, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_verify_draft(P, None, P, P, v, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_verify_draft(P, P, P, None, v, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_verify_draft(P, P, P + 2, P, v, P, 1 << 40, None) == EALIGN
    assert L.krk_cuda_verify_draft_workspace_bytes(v) > 0 and L.krk_cuda_verify_draft_workspace_bytes(C.byref(verify(n_rows=0))) == 0
    assert L.krk_cuda_verify_draft(None, None, None, None, C.byref(verify(n_seq=0)), None, 0, None) == 0


def test_what_is_written_meets_nothing_else():
    """Lists of a plan and of a verification in each other's place; y of a norm in the place of x as f16, under another stride, and in h's."""
    at = {n: P + 0x10000 * i for i, n in enumerate(("kv_before", "n_new", "page_table", "free_pages", "n_free", "q_start", "kv_len", "last", "positions", "slots", "counts"))}

    def plan(**k):
        return L.krk_cuda_step_plan(C.byref(capi.Step(**{**at, **dict(max_tok=8, free_cap=9, n_seq=4, table_width=3, page_size=16), **k})), None)
    for k in (dict(kv_len=at["kv_before"]), dict(kv_before=at["kv_len"] + 12), dict(counts=at["n_free"]), dict(n_free=at["counts"] + 8), dict(last=at["n_new"]),
              dict(page_table=at["free_pages"] + 32), dict(kv_len=at["q_start"] + 16), dict(slots=at["positions"] + 24)):
        assert plan(**k) == EARG
    t, n, lp, x, W = (P + 0x10000 * i for i in range(5))
    at = {n: P + 0x100000 + 0x10000 * i for i, n in enumerate(("row_start", "draft", "accept_u", "sample_u", "temp", "draft_temp"))}

    def judge(tokens=t, accepted=n, logprob=lp, **k):
        return L.krk_cuda_verify_draft(tokens, accepted, logprob, x, C.byref(capi.Verify(**{**at, **dict(n_rows=6, n_vocab=100, stride=100, n_seq=2), **k})), W, 1 << 20, None)
    for k in (dict(tokens=at["draft"]), dict(logprob=at["accept_u"]), dict(tokens=at["draft"] + 20), dict(accepted=at["row_start"]), dict(logprob=t), dict(accepted=at["temp"])):
        assert judge(**k) == EARG
    X, Y = P + 0x10000, P + 0x20000
    assert L.krk_cuda_block_norm(X, None, X, C.byref(norm(y_dtype=1)), None) == EARG
    assert L.krk_cuda_block_norm(X, None, X, C.byref(norm(y_stride=104)), None) == EARG
    assert L.krk_cuda_block_norm(Y, Y, X, C.byref(norm()), None) == EARG


def test_the_binding_refuses():
    """On tensors that are not on a GPU, and what is no tensor."""
    import torch
    f, i = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    c = capi.KvCache.empty(capi.KV_F16, 2, 1, 16, 64, device="cpu")
    for call in (lambda: capi.attention_chunk(torch.zeros(1, 1, 64), c, i, i[:1], i.view(1, 2), 1), lambda: capi.step_plan(i, i, i.view(2, 1), i, i[:1], 16, 4),
                 lambda: capi.block_norm(f), lambda: capi.verify_draft(f, i, i, f[:, 0], f[0, :1])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        capi.block_norm([1.0])

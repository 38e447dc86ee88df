"""What the entry points between the projections and the logits refuse, on the host: nothing is launched."""
import ctypes as C

import pytest

from kraken_b200 import capi

L = capi.lib
P = 0x10000   # an address that is never looked at
EDTYPE, ESHAPE, ENULL, EALIGN, EWORKSPACE, EARG = -1, -2, -3, -4, -6, -8


def cache(**k):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, type=capi.KV_Q8, head_dim=128, n_kv_heads=8, page_size=16, n_pages=10)
    return capi.KvCacheStruct(*[{**f, **k}[n] for n, _ in capi.KvCacheStruct._fields_])


def attention(**k):
    f = dict(q_start=P, kv_len=P, page_table=P, tree=0, sinks=0, q_stride=4096, out_stride=4096, max_kv_len=0, n_seq=2, n_heads=32, max_q=4, table_width=100,
             window=0, scale=0.1, softcap=0.0)
    return capi.Attention(*[{**f, **k}[n] for n, _ in capi.Attention._fields_])


def rope(**k):
    f = dict(pos=P, inv_freq=P, q_weight=0, k_weight=0, n_tok=3, q_stride=4096, k_stride=1024, q_out_stride=4096, k_out_stride=1024, n_heads=32, n_kv_heads=8,
             head_dim=128, rot_dim=128, norm=1, interleaved=0, eps=1e-6)
    return capi.Rope(*[{**f, **k}[n] for n, _ in capi.Rope._fields_])


def adjust(**k):
    f = dict(n_rows=2, n_vocab=100, stride=100, out_stride=100, hist=P, hist_len=0, hist_n=10, hist_stride=10, rep=0, freq=0, pres=0, bias_ids=P, bias=P, bias_len=0,
             bias_n=4, bias_stride=4, mask=P, mask_row=0, n_masks=2, mask_stride=4)
    return capi.Adjust(*[{**f, **k}[n] for n, _ in capi.Adjust._fields_])


@pytest.fixture(autouse=True)
def nothing_launched():
    before = L.krk_cuda_launch_count()
    yield
    assert L.krk_cuda_launch_count() == before


@pytest.mark.parametrize("rc,k", [
    (EDTYPE, dict(type=3)), (EDTYPE, dict(type=-1)), (ESHAPE, dict(head_dim=48)), (ESHAPE, dict(head_dim=288)), (ESHAPE, dict(head_dim=0)), (ESHAPE, dict(n_kv_heads=0)),
    (ESHAPE, dict(page_size=8)), (ESHAPE, dict(page_size=40)), (ESHAPE, dict(n_pages=-1)), (ENULL, dict(k=0)), (ENULL, dict(v_scale=0)), (EALIGN, dict(k_scale=P + 8)),
    (EALIGN, dict(v=P + 2))])
def test_caches(rc, k):
    c = cache(**k)
    assert L.krk_cuda_kv_append(C.byref(c), P, P, 1024, 1024, P, 1, None) == rc
    assert L.krk_cuda_kv_read(C.byref(c), P, P, P, 1, None) == rc
    assert L.krk_cuda_attention_tree(P, P, C.byref(c), C.byref(attention()), P, 1 << 40, None) == rc
    assert L.krk_cuda_attention_tree_workspace_bytes(C.byref(c), C.byref(attention())) == 0


def test_append_and_read():
    c = C.byref(cache())
    assert L.krk_cuda_kv_append(None, P, P, 1024, 1024, P, 1, None) == ENULL
    assert L.krk_cuda_kv_append(c, None, P, 1024, 1024, P, 1, None) == ENULL
    assert L.krk_cuda_kv_append(c, P, P, 1024, 1024, None, 1, None) == ENULL
    assert L.krk_cuda_kv_append(c, P, P, 1020, 1024, P, 2, None) == ESHAPE
    assert L.krk_cuda_kv_append(c, P, P, 1026, 1024, P, 2, None) == EALIGN
    assert L.krk_cuda_kv_append(c, P, P + 4, 1024, 1024, P, 1, None) == EALIGN
    assert L.krk_cuda_kv_append(c, P, P, 1024, 1024, P + 4, 1, None) == EALIGN
    assert L.krk_cuda_kv_append(c, P, P, 1024, 1024, P, -1, None) == ESHAPE
    assert L.krk_cuda_kv_append(c, None, None, 0, 0, None, 0, None) == 0
    assert L.krk_cuda_kv_read(c, P, None, P, 1, None) == ENULL
    assert L.krk_cuda_kv_read(c, P + 4, P, P, 1, None) == EALIGN
    assert L.krk_cuda_kv_read(c, P, P, P, -1, None) == ESHAPE
    assert L.krk_cuda_kv_read(c, None, None, None, 0, None) == 0


@pytest.mark.parametrize("rc,k", [
    (ESHAPE, dict(n_heads=30)), (ESHAPE, dict(n_heads=0)), (ESHAPE, dict(max_q=65)), (ESHAPE, dict(max_q=-1)), (ESHAPE, dict(n_seq=-1)), (ESHAPE, dict(table_width=0)),
    (ESHAPE, dict(max_kv_len=1601)), (ESHAPE, dict(max_kv_len=-1)), (ESHAPE, dict(table_width=1 << 30)), (ESHAPE, dict(q_stride=4092)), (ESHAPE, dict(out_stride=0)),
    (EARG, dict(window=63)), (EARG, dict(window=-1)), (EARG, dict(softcap=-1.0)), (EARG, dict(softcap=float("nan"))), (ENULL, dict(q_start=0)), (ENULL, dict(kv_len=0)),
    (ENULL, dict(page_table=0)), (EALIGN, dict(tree=P + 4)), (EALIGN, dict(out_stride=4098)), (EALIGN, dict(sinks=P + 2)), (0, dict(n_seq=0, q_start=0)), (0, dict(max_q=0))])
def test_attention(rc, k):
    assert L.krk_cuda_attention_tree(P, P, C.byref(cache()), C.byref(attention(**k)), P, 1 << 40, None) == rc


def test_attention_pointers():
    c, a = C.byref(cache()), C.byref(attention())
    assert L.krk_cuda_attention_tree(None, P, c, a, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_attention_tree(P, None, c, a, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_attention_tree(P, P, c, None, P, 1 << 40, None) == ENULL
    assert L.krk_cuda_attention_tree(P + 4, P, c, a, P, 1 << 40, None) == EALIGN
    assert L.krk_cuda_attention_tree(P, P + 8, c, a, P, 1 << 40, None) == EALIGN
    for d in (32, 160, 224):
        assert L.krk_cuda_attention_tree(P, P, C.byref(cache(head_dim=d)), a, P, 1 << 40, None) == ESHAPE
    # short contexts take no workspace
    assert L.krk_cuda_attention_tree_workspace_bytes(c, C.byref(attention(table_width=4))) == 0
    assert L.krk_cuda_attention_tree_workspace_bytes(c, a) > 0


@pytest.mark.parametrize("rc,k", [
    (ESHAPE, dict(head_dim=12)), (ESHAPE, dict(head_dim=264)), (ESHAPE, dict(head_dim=0)), (ESHAPE, dict(rot_dim=136)), (ESHAPE, dict(rot_dim=4)), (ESHAPE, dict(rot_dim=-8)),
    (ESHAPE, dict(n_tok=-1)), (ESHAPE, dict(n_heads=-1)), (ESHAPE, dict(q_stride=4092)), (ESHAPE, dict(k_out_stride=8)), (EALIGN, dict(q_stride=4097)), (EARG, dict(eps=-1.0)),
    (EARG, dict(eps=float("nan"))), (ENULL, dict(pos=0)), (ENULL, dict(inv_freq=0)), (EALIGN, dict(q_weight=P + 4)), (EALIGN, dict(pos=P + 2)), (0, dict(n_tok=0)),
    (0, dict(n_heads=0, n_kv_heads=0))])
def test_rope(rc, k):
    assert L.krk_cuda_qk_norm_rope(P, P, P, P, C.byref(rope(**k)), None) == rc


def test_rope_pointers():
    assert L.krk_cuda_qk_norm_rope(P, P, P, P, None, None) == ENULL
    for i in range(4):
        for bad, rc in ((None, ENULL), (P + 4, EALIGN)):
            assert L.krk_cuda_qk_norm_rope(*[bad if i == j else P for j in range(4)], C.byref(rope()), None) == rc


@pytest.mark.parametrize("rc,k", [
    (ESHAPE, dict(n_rows=-1)), (ESHAPE, dict(n_vocab=1 << 31)), (ESHAPE, dict(stride=99)), (ESHAPE, dict(out_stride=0)), (ESHAPE, dict(hist_n=-1)), (ESHAPE, dict(hist_stride=9)),
    (ESHAPE, dict(bias_stride=3)), (ESHAPE, dict(mask_stride=3)), (ENULL, dict(bias_ids=0)), (EALIGN, dict(hist=P + 2)), (EALIGN, dict(mask_row=P + 1)), (0, dict(n_rows=0)),
    (0, dict(n_vocab=0))])
def test_adjust(rc, k):
    assert L.krk_cuda_logits_adjust(P, P, C.byref(adjust(**k)), None) == rc


def test_adjust_pointers():
    assert L.krk_cuda_logits_adjust(None, P, C.byref(adjust()), None) == ENULL
    assert L.krk_cuda_logits_adjust(P, None, C.byref(adjust()), None) == ENULL
    assert L.krk_cuda_logits_adjust(P, P, None, None) == ENULL
    assert L.krk_cuda_logits_adjust(P + 2, P, C.byref(adjust()), None) == EALIGN


def test_python_checks_what_it_is_given():
    import torch
    c = capi.KvCache.empty(capi.KV_Q8, 2, 2, 16, 64, device="cpu")
    k = torch.zeros((3, 2, 64))
    with pytest.raises(ValueError, match="GPU"):
        capi.kv_append(c, k, k, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="on cpu"):
        capi.kv_append(c, k.to("meta"), k, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError):
        capi.qk_norm_rope(k, None, None, None)
    with pytest.raises(ValueError):
        capi.logits_adjust(torch.zeros(3))
    with pytest.raises(TypeError):
        capi.logits_adjust([1.0])
    with pytest.raises(ValueError):
        capi.KvCache(capi.KV_Q8, c.k, c.v)
    with pytest.raises(ValueError):
        capi.KvCache(capi.KV_Q8, c.k, c.v, c.k_scale, c.v_scale.transpose(0, 1))
    with pytest.raises(KeyError):
        capi.KvCache(7, c.k, c.v)


def test_a_softcap_without_end():
    a = attention(softcap=float("inf"))   # (infinity times tanh(0) is no score)
    assert L.krk_cuda_attention_tree(P, P, C.byref(cache()), C.byref(a), P, 1 << 40, None) == EARG
    assert L.krk_cuda_attention_tree_workspace_bytes(C.byref(cache()), C.byref(a)) == 0


def test_rows_in_place_keep_their_strides():
    """A row written over another one's place before that one is read."""
    Q, K = 1 << 40, 1 << 41
    for r in (rope(q_out_stride=4100), rope(k_out_stride=1028)):
        assert L.krk_cuda_qk_norm_rope(Q, K, Q, K, C.byref(r), None) == EARG
    for a in (adjust(out_stride=104), adjust(stride=104)):
        assert L.krk_cuda_logits_adjust(Q, Q, C.byref(a), None) == EARG

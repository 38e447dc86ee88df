"""What verify_draft writes, its workspace among it, in the place of what it reads: refused on the host, nothing is launched."""
import ctypes as C

import pytest

from kraken_b200 import capi
from test_step_refusals import EARG, L, P, nothing_launched  # noqa: F401

ROWS, VOCAB, SEQS = 6, 100, 2
AT = {n: P + 0x100000 + 0x10000 * i for i, n in enumerate(("row_start", "draft", "accept_u", "sample_u", "temp", "draft_temp", "draft_logits"))}
T, N, LP, X, W = (P + 0x10000 * i for i in range(5))


def judge(tokens=T, accepted=N, logprob=LP, logits=X, workspace=W, **k):
    v = capi.Verify(**{**AT, **dict(n_rows=ROWS, n_vocab=VOCAB, stride=VOCAB, draft_stride=VOCAB, n_seq=SEQS), **k})
    return L.krk_cuda_verify_draft(tokens, accepted, logprob, logits, C.byref(v), workspace, 1 << 20, None)


NEED = L.krk_cuda_verify_draft_workspace_bytes(C.byref(capi.Verify(**AT, n_rows=ROWS, n_vocab=VOCAB, stride=VOCAB, draft_stride=VOCAB, n_seq=SEQS)))
END = 4 * ROWS * VOCAB


@pytest.mark.parametrize("k", [
    # outputs in the target's rows, at their ends, and reaching into them from before
    dict(tokens=X), dict(tokens=X + END - 4), dict(tokens=X - 20), dict(accepted=X + 400), dict(logprob=X + 1204), dict(logprob=X - 4),
    # in the drafter's
    dict(tokens=AT["draft_logits"]), dict(accepted=AT["draft_logits"] + END - 4), dict(logprob=AT["draft_logits"] - 20),
    # rows apart: across the beginning of one
    dict(tokens=X + 4 * 120 - 20, stride=120), dict(logprob=AT["draft_logits"] + 5 * 4 * 130 + 396, draft_stride=130), dict(tokens=X + 8 * 120 + 396, stride=120),
    # the workspace in what is read, in what is written, and across rows
    dict(workspace=X), dict(workspace=X + END - 16), dict(workspace=X - NEED + 16), dict(workspace=AT["draft_logits"] + 16), dict(workspace=T), dict(workspace=N - NEED + 16), dict(workspace=LP + 16),
    *[dict(workspace=AT[n]) for n in AT]])
def test_refused(k):
    assert judge(**k) == EARG


@pytest.mark.parametrize("k", [
    dict(), dict(tokens=X + END), dict(tokens=X - 4 * ROWS), dict(workspace=X + END), dict(logprob=None), dict(accepted=AT["draft_logits"] + END),
    dict(tokens=X + 400, stride=120), dict(logprob=X + 5 * 480 + 400, stride=120), dict(draft_logits=None, tokens=AT["draft_logits"]), dict(logprob=None, workspace=LP)])
def test_beside_them_and_between_rows(k):
    """Not refused for where they lie: without a GPU the next thing that is missed is the device."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("these addresses are not a GPU's")
    assert judge(**k) not in (0, EARG)

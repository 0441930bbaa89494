"""The largest calls of beam_select, and those that are refused because they are larger."""
import pytest
import torch

from cachegen_b200 import _lib, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,beams,k", [(_lib.CG_MAX_BEAM_ROWS, 1, 1), (_lib.CG_MAX_BEAM_ROWS // 256, 256, 2)])
def test_as_many_rows_as_a_call_takes(requests, beams, k):
    """All rows are the same: the best tokens are the lowest beams'."""
    logits = torch.tensor([[0.0, 2.0, 1.0]], device="cuda").expand(requests * beams, 3)
    scores, tokens, parents = paged.beam_select(logits, torch.zeros((requests, beams), device="cuda"), k)
    assert torch.equal(tokens, torch.ones_like(tokens))
    want = torch.arange(requests, device="cuda", dtype=torch.int32)[:, None] * beams + torch.arange(k, device="cuda", dtype=torch.int32)
    assert torch.equal(parents, want)
    best = torch.log_softmax(logits[0].double(), -1)[1].item()
    assert (scores.double() - best).abs().max().item() <= 5e-6 + 2.0 ** -24 * abs(best)


@pytest.mark.parametrize("requests,beams,vocab,dtype,what", [
    (_lib.CG_MAX_BEAM_ROWS + 1, 1, 2, torch.float16, "rows of logits"), (4097, 256, 2, torch.bfloat16, "rows of logits"),
    (1100, 256, 1 << 24, torch.float32, "more than a call takes")])
def test_more_rows_are_refused(requests, beams, vocab, dtype, what):
    logits = torch.zeros((1, vocab), dtype=dtype, device="cuda").expand(requests * beams, vocab)
    with pytest.raises(RuntimeError, match=what):
        paged.beam_select(logits, torch.zeros((requests, beams), device="cuda"), 1)

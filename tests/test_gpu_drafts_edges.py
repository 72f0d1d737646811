"""Calls at the edges of the operators for drafted tokens: no history yet, rows
that a step's plan leaves out, waits that run out."""
import numpy as np
import pytest
import torch

import drafts_ref as D
from test_gpu_drafts import DTYPES, S, _dev, _logit_case, _on_gpu      # noqa: F401  (S: the fixture)

pytestmark = pytest.mark.gpu


# ── logits without a history ─────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,kw", [
    (None, {}), (None, dict(biases=9, masked=True)), ([3, 0, 1, 5], dict(extra=2)),
    ([3, 0, 1, 5], dict(extra=2, tree=True, biases=9, masked=True))])
def test_a_first_step_has_no_history(S, dtype, counts, kw):
    """`history[:, :0]` with its lengths (which may say more: there are no more tokens than columns) is no history."""
    x, starts, rules = _logit_case(counts, 1000, dtype, 3, **kw)
    y, of = D.adjust(x.float().numpy(), starts, rules)
    g = _on_gpu(starts, rules)
    requests = len(rules["repetition"])
    none = dict(history=torch.zeros(requests, 5, dtype=torch.int32, device="cuda")[:, :0],
                history_lens=torch.arange(requests, dtype=torch.int32, device="cuda"))
    want = torch.from_numpy(y).to(dtype)
    for more in ({}, dict(prompt_lens=torch.ones(requests, dtype=torch.int32, device="cuda"))):
        assert torch.equal(S.adjust_logits(x.cuda(), **g, **none, **more).cpu(), want)
        np.testing.assert_array_equal(S.pick_tokens(x.cuda(), **g, **none, **more).cpu().numpy(), D.pick(y, of))

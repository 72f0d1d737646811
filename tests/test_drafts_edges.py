"""Calls at the edges of the operators for drafted tokens, as far as they can
be looked at without a GPU."""
import pytest
import torch

from sili__new_b200 import serving as S
from test_drafts import I32, I64, _logits, _settle


def _rules(history=0, width=0, lens=0, prompts=0):
    """Rules of one request with no more than a history (the pointers are looked at, not the arrays)."""
    return S._cuda.LogitRules(0, history, width, width, lens, prompts, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("pick", [False, True])
def test_a_history_without_a_column_is_none(pick):
    """An array without elements has no address, its lengths have one: no history, and no more scratch space than that."""
    size = lambda rules: S._cuda.logits_scratch(0, 1, 64, 1, rules, pick)  # noqa: E731
    assert size(_rules(lens=16)) == size(_rules(lens=16, prompts=16)) == size(_rules())
    for rules in (_rules(history=16, width=3), _rules(width=3, lens=16)):
        with pytest.raises(ValueError, match="together"):
            size(rules)


@pytest.mark.parametrize("call", [S.adjust_logits, S.pick_tokens])
def test_a_history_without_a_column_passes_the_checks(call):
    with pytest.raises(ValueError, match="CUDA"):
        _logits(call, history=torch.zeros(3, 9, dtype=I32)[:, :0], prompt_lens=torch.zeros(3, dtype=I32))


@pytest.mark.parametrize("masks", [torch.zeros(5, dtype=I64), torch.zeros(5, 5, dtype=I64), torch.zeros(4, 1, dtype=I64),
                                   torch.zeros(5, 1, dtype=I32), torch.zeros(5, 4, dtype=I64)[:, ::2]])
def test_settling_takes_the_masks_of_its_rows(masks):
    with pytest.raises(ValueError, match="masks"):
        _settle(masks=masks)


def test_settling_takes_masks():
    with pytest.raises(ValueError, match="CUDA"):
        _settle(masks=torch.zeros(5, 2, dtype=I64))


def test_caches_must_not_share_an_array():
    """Each array is moved once: two caches with one array of codes, or of scales, would move it twice."""
    codes = [torch.zeros(3, 2, 2, 16, 32, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.zeros(3, 2, 2, 16, 2, dtype=torch.uint8) for _ in range(2)]
    for caches in ([(codes[0], scales[0]), (codes[1], scales[0])], [(codes[0], scales[0]), (codes[0], scales[1])]):
        with pytest.raises(ValueError, match="twice"):
            _settle(caches=caches)
    with pytest.raises(ValueError, match="CUDA"):
        _settle(caches=list(zip(codes, scales)))

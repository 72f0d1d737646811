"""What the calls for drafted tokens refuse before they look for a device, and
the test restatements' own consistency (no GPU)."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import drafts_ref as D
from sili__new_b200 import serving as S

I32, I64 = torch.int32, torch.int64


def _tree(**kw):
    a = dict(parents=torch.zeros(5, dtype=I32), starts=torch.zeros(3, dtype=I32), lens=torch.zeros(2, dtype=I32), most_new=5)
    return S.draft_tree(**{**a, **kw})


def _attend(**kw):
    a = dict(q=torch.zeros(5, 4, 64), codes=torch.zeros(3, 2, 2, 16, 32, dtype=torch.uint8),
             scales=torch.zeros(3, 2, 2, 16, 2, dtype=torch.uint8), table=torch.zeros(2, 2, dtype=I32),
             lens=torch.zeros(2, dtype=I32), starts=torch.zeros(3, dtype=I32), masks=torch.zeros(5, 1, dtype=I64))
    return S.tree_attention(**{**a, **kw})


def _logits(call=S.adjust_logits, **kw):
    a = dict(logits=torch.zeros(3, 40), history=torch.zeros(3, 9, dtype=I32), history_lens=torch.zeros(3, dtype=I32),
             repetition=torch.ones(3), allowed=torch.zeros(3, 2, dtype=I32), bias_tokens=torch.zeros(3, 4, dtype=I32),
             bias_values=torch.zeros(3, 4))
    return call(**{**a, **kw})


def _settle(**kw):
    a = dict(drafted=torch.zeros(5, dtype=I32), parents=torch.zeros(5, dtype=I32), picked=torch.zeros(5, dtype=I64),
             starts=torch.zeros(3, dtype=I32), lens=torch.zeros(2, dtype=I32), table=torch.zeros(2, 2, dtype=I32),
             caches=[(torch.zeros(3, 2, 2, 16, 32, dtype=torch.uint8), torch.zeros(3, 2, 2, 16, 2, dtype=torch.uint8))],
             ring=torch.zeros(3, dtype=I32), pool=torch.zeros(2, dtype=I64))
    return S.settle_drafts(**{**a, **kw})


@pytest.mark.parametrize("call", [_tree, _attend, _logits, lambda **k: _logits(S.pick_tokens, **k), _settle])
def test_host_arrays_are_refused(call):
    with pytest.raises(ValueError, match="CUDA"):
        call()


@pytest.mark.parametrize("call,kw,match", [
    (_tree, dict(parents=torch.zeros(5, dtype=I64)), "parents"), (_tree, dict(starts=torch.zeros(2, dtype=I32)), "starts"),
    (_tree, dict(lens=torch.zeros(2)), "lens"), (_tree, dict(most_new=257), "most_new"), (_tree, dict(most_new=-1), "most_new"),
    (_tree, dict(window=-1), "window"), (_tree, dict(parents=torch.zeros(10, dtype=I32)[::2]), "contiguous"),
    (_attend, dict(masks=torch.zeros(5, dtype=I64)), "masks"), (_attend, dict(masks=torch.zeros(5, 5, dtype=I64)), "masks"),
    (_attend, dict(masks=torch.zeros(4, 1, dtype=I64)), "masks"), (_attend, dict(masks=torch.zeros(5, 1, dtype=I32)), "masks"),
    (_attend, dict(masks=torch.zeros(1, 5, dtype=I64).T), None), (_attend, dict(starts=torch.zeros(2, dtype=I32)), "starts"),
    (_attend, dict(q=torch.zeros(5, 3, 64)), "kv heads"), (_attend, dict(q=torch.zeros(5, 4, 128)), "head dimension"),
    (_attend, dict(q=torch.zeros(5, 4, 64, dtype=torch.float64)), "float32"), (_attend, dict(window=-3), "window"),
    (_attend, dict(most_new=-3), "most_new"), (_attend, dict(table=torch.zeros(3, 2, dtype=I32)), "table"),
    (_logits, dict(logits=torch.zeros(40)), "rows, vocab"), (_logits, dict(logits=torch.zeros(40, 3).T), "contiguous"),
    (_logits, dict(logits=torch.zeros(3, 40, dtype=torch.float64)), "float32"), (_logits, dict(history_lens=None), "together"),
    (_logits, dict(logits=torch.zeros(99).as_strided((3, 40), (20, 1))), "overlap"),
    (_logits, dict(history=None, history_lens=None, prompt_lens=torch.zeros(3, dtype=I32)), "together"),
    (_logits, dict(history=torch.zeros(2, 9, dtype=I32)), "history"), (_logits, dict(starts=torch.zeros(3, dtype=I32)), "history"),
    (_logits, dict(drafted=torch.zeros(3, dtype=I32)), "together"), (_logits, dict(repetition=torch.ones(2)), "repetition"),
    (_logits, dict(drafted=torch.zeros(3, dtype=I32), masks=torch.zeros(3, 1, dtype=I64)), "starts"),
    (_logits, dict(temperature=torch.ones(3, dtype=torch.float16)), "temperature"), (_logits, dict(bias_values=None), "together"),
    (_logits, dict(bias_tokens=torch.zeros(3, 5, dtype=I32)), "bias_values"), (_logits, dict(allowed=torch.zeros(3, 1, dtype=I32)), "allowed"),
    (_logits, dict(allowed=torch.zeros(3, 2, dtype=I64)), "allowed"), (_logits, dict(out=torch.zeros(3, 41)), "out"),
    (_logits, dict(out=torch.zeros(3, 40, dtype=torch.float16)), "out"),
    (_settle, dict(drafted=torch.zeros(5, dtype=I64)), "drafted"), (_settle, dict(picked=torch.zeros(5)), "picked"),
    (_settle, dict(picked=torch.zeros(4, dtype=I32)), "picked"), (_settle, dict(caches=[]), "cache"),
    (_settle, dict(ring=torch.zeros(0, dtype=I32)), "ring"), (_settle, dict(pool=torch.zeros(3, dtype=I64)), "pool"),
    (_settle, dict(parents=torch.zeros(4, dtype=I32)), "parents"), (_settle, dict(table=torch.zeros(1, 2, dtype=I32)), "table")])
def test_refusals(call, kw, match):
    with pytest.raises(ValueError, match=match or "CUDA"):
        call(**kw)


def test_caches_must_be_alike_and_different():
    one = torch.zeros(3, 2, 2, 16, 32, dtype=torch.uint8), torch.zeros(3, 2, 2, 16, 2, dtype=torch.uint8)
    other = torch.zeros(3, 2, 1, 16, 32, dtype=torch.uint8), torch.zeros(3, 2, 1, 16, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="shapes"):
        _settle(caches=[one, other])
    with pytest.raises(ValueError, match="twice"):
        _settle(caches=[one, one])
    with pytest.raises(ValueError, match="scales"):
        _settle(caches=[(one[0], other[1])])


def test_an_output_that_meets_the_logits_is_refused():
    flat = torch.zeros(500)
    x = flat[:120].view(3, 40)
    for out in (flat[1:121].view(3, 40), flat[:126].view(3, 42)[:, :40], flat[80:200].view(3, 40)):
        with pytest.raises(ValueError, match="out"):
            _logits(logits=x, out=out)
    for out in (x, flat[120:240].view(3, 40)):
        with pytest.raises(ValueError, match="CUDA"):
            _logits(logits=x, out=out)


def test_an_output_that_meets_the_queries_is_refused():
    flat = torch.zeros(6 * 4 * 64)
    q = flat[:5 * 256].view(5, 4, 64)
    for out in (q, flat[256:].view(5, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            _attend(q=q, out=out)
    with pytest.raises(ValueError, match="CUDA"):
        _attend(q=q, out=torch.zeros(5, 4, 64))


@pytest.mark.parametrize("width,biases", [(2 ** 29 + 1, 0), (2 ** 31 - 1, 0), (0, 2 ** 29 + 1), (0, 2 ** 31 - 1)])
def test_lists_too_long_to_count_are_refused(width, biases):
    # (the sizes are looked at, not the arrays)
    rules = S._cuda.LogitRules(0, 8 if width else 0, width, width, 8 if width else 0, 0, 0, 0, 0, 0, 0, 0, 0,
                               8 if biases else 0, 8 if biases else 0, biases, 0, 0)
    with pytest.raises(ValueError, match="too long"):
        S._cuda.logits_scratch(0, 1, 64, 1, rules, False)


def test_a_cache_is_a_pair():
    with pytest.raises(ValueError, match="codes, scales"):
        _settle(caches=[(torch.zeros(3, 2, 2, 16, 32, dtype=torch.uint8),)])


@pytest.mark.parametrize("name,call", [("q", _attend), ("logits", _logits), ("repetition", _logits), ("bias_values", _logits),
                                       ("logits", lambda **k: _logits(S.pick_tokens, **k))])
def test_a_gradient_that_would_be_lost_is_refused(name, call):
    x = {"q": torch.zeros(5, 4, 64), "logits": torch.zeros(3, 40), "repetition": torch.ones(3), "bias_values": torch.zeros(3, 4)}[name]
    with pytest.raises(ValueError, match="no gradient"):
        call(**{name: x.clone().requires_grad_()})
    with forward_ad.dual_level(), pytest.raises(ValueError, match="no gradient"):
        call(**{name: forward_ad.make_dual(x, torch.ones_like(x))})
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        call(**{name: x.clone().requires_grad_()})


def test_the_restatements_agree_with_each_other():
    """A tree's masks and its accepted way: each accepted row's mask holds exactly the way up to it."""
    rng = np.random.default_rng(1)
    for n in (1, 2, 9, 70, 200):
        parents = np.array(D.random_tree(n, rng))
        masks, positions = D.draft_tree(parents, [0, n], [n + 5], n, -(-n // 64), 0)
        bits = D.bits_of(masks)
        drafted, picked = np.arange(n), np.full(n, -1)
        for i in range(n):
            children = np.flatnonzero(parents == i)
            if len(children):
                picked[i] = children[-1]
        path, kept, token, lens = D.accept(drafted, parents, picked, [0, n], [n + 5], n)
        way = path[:kept[0]]
        for k, i in enumerate(way):
            assert sorted(np.flatnonzero(bits[i])) == sorted(way[:k + 1]) and positions[i] == 5 + k
        assert lens[0] == 5 + kept[0] and token[0] == picked[way[-1]]

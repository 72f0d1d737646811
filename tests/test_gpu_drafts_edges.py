"""Calls at the edges of the operators for drafted tokens: no history yet, rows
that a step's plan leaves out, waits that run out."""
import numpy as np
import pytest
import torch

import drafts_ref as D
from test_gpu_drafts import DTYPES, S, _dev, _logit_case, _on_gpu, _own_kernel, _tree_case      # noqa: F401  (S: the fixture)

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


# ── rows that the plan leaves out ────────────────────────────────────────────
def _chain_step(S, n, most_new, dtype=torch.bfloat16, page=16, hk=2, h=4, dim=64, committed=5):
    """One request's chain of n drafts whose picks agree all the way, planned for most_new of them."""
    parents, drafted = _dev(np.arange(n) - 1), _dev(np.arange(n) + 7)
    picked = _dev(np.arange(n) + 8)
    pages = -(-(committed + n) // page) + 2
    ring, pool = S.page_pool(pages)
    table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    t = S.page_tables(_dev([0]), _dev([committed]), table, ring, pool, page, committed)
    t = S.page_tables(t.lens, _dev([n]), table, ring, t.pool, page, n)
    tree = S.draft_tree(parents, t.starts, t.lens, most_new)
    return parents, drafted, picked, table, ring, t, tree, pages, (S.KVCache4(pages, page, hk, dim),)


@pytest.mark.parametrize("n,most_new,there", [(300, 256, 256), (70, 10, 64), (130, 65, 128), (64, 64, 64), (200, 200, 200)])
def test_a_row_past_the_plan_is_not_accepted(S, n, most_new, there):
    """Rows past the masks' bits have no key: the accepted way ends before them, and their pages go back."""
    parents, drafted, picked, table, ring, t, tree, pages, caches = _chain_step(S, n, most_new)
    end = S.settle_drafts(drafted, parents, picked, t.starts, t.lens, table, caches, ring, t.pool, tree.masks)
    assert end.kept.tolist() == [there] and end.lens.tolist() == [5 + there] and end.token.tolist() == [there + 7]
    assert end.path.tolist() == list(range(there)) + [-1] * (n - there)
    assert int(end.pool[0] - end.pool[1]) + pages == -(-(5 + there) // 16)


def test_a_row_without_a_bit_is_not_accepted(S):
    """Parents that are none, as the plan has it; a sibling that is one takes the place of one that is none."""
    #           0   1  2  3  4  5
    parents = [-1, 0, 0, 1, 2, 4]
    drafted, picked = [3, 5, 5, 6, 8, 9], [5, 6, 8, 1, 9, 4]
    masks = np.array([[1], [0], [5], [0], [21], [53]])          # rows 1 and 3 are none
    table, (ring, pool) = _dev([[0, 1]]), S.page_pool(4)
    args = [_dev(x) for x in (drafted, parents, picked, [0, 6], [26])]
    end = lambda m: S.settle_drafts(*args, table, [S.KVCache4(4, 16, 1, 64)], ring, pool, m)  # noqa: E731
    a = end(_dev(masks, torch.int64))
    assert a.path.tolist() == [0, 2, 4, 5, -1, -1] and a.kept.tolist() == [4] and a.token.tolist() == [4]
    masks[0] = 0                                                # no root, nothing
    a = end(_dev(masks, torch.int64))
    assert a.kept.tolist() == [0] and a.token.tolist() == [-1] and a.lens.tolist() == [20]


@pytest.mark.parametrize("seed", range(3))
def test_settling_with_a_plan_of_all_rows_changes_nothing(S, seed):
    """Trees whose rows are all there: with the masks and without them, the same."""
    from test_gpu_drafts import _settle_case
    starts, tokens, parents, drafted, picked, lens, table, ring, pool, n_pages = _settle_case(
        [64, 1, 0, 130, 256], [10, 0, 3, 300, 47], 16, seed, extra=3, first=2, chain=seed == 1)
    args = [_dev(x) for x in (drafted, parents, picked, starts, lens, table)]
    masks = S.draft_tree(args[1], args[3], args[4], 256).masks
    caches = [torch.randint(0, 255, shape, dtype=torch.uint8, device="cuda") for shape in ((n_pages, 2, 2, 16, 32), (n_pages, 2, 2, 16, 2))]
    got = []
    for m in (None, masks):
        mine, held = [x.clone() for x in caches], _dev(ring)
        a = S.settle_drafts(*args, [tuple(mine)], held, _dev(pool, torch.int64), m)
        got.append([*a, *mine, held])
    assert all(torch.equal(x, y) for x, y in zip(*got))


def test_a_chain_past_the_plan_goes_on_where_it_ended(S):
    """Keys through the append, picks through the attention: the cache after a step whose plan left rows out is the cache
    of a step that had only the others."""
    outs = []
    for n, most_new in ((80, 20), (64, 64)):
        g = torch.Generator("cuda").manual_seed(1)
        parents, drafted, picked, table, ring, t, tree, pages, (c,) = _chain_step(S, n, most_new)
        x = torch.randn(80, 8, 64, generator=g, device="cuda")[:n].bfloat16()
        cos, sin = S.rotary_table(512, 64)
        S.cache_append(x[:, :2], x[:, 2:4], c.codes, c.scales, t.slots, cos=cos, sin=sin, positions=tree.positions)
        end = S.settle_drafts(drafted, parents, picked, t.starts, t.lens, table, [c], ring, t.pool, tree.masks)
        q = x[:1, 4:8].contiguous()
        outs.append((end.lens, end.token, S.cache_attention(q, c.codes, c.scales, table, end.lens)))
    assert outs[0][0].tolist() == [69] and all(torch.equal(a, b) for a, b in zip(*outs))


# ── waits that run out ───────────────────────────────────────────────────────
def _runs_out(S, case, most_new, **limits):
    """(a call's out and lse, those of a call under these limits); each of its rows is NaN or whole, the status tells which
    there were, and the next call is whole again."""
    from sili__new_b200 import _cuda
    q, codes, scales, table, lens, starts, masks = case

    def call():
        return S.tree_attention(q, codes, scales, table, lens, _dev(starts), masks, most_new=most_new, return_lse=True)

    S.check_attention()
    want = call()
    S.check_attention()
    try:
        _cuda.kv4_attention_wait_limit(**limits)
        got = call()
        torch.cuda.synchronize()
    finally:
        _cuda.kv4_attention_wait_limit()
    nan = torch.isnan(got[1])
    assert torch.equal(torch.isnan(got[0]), nan[..., None].expand_as(got[0]))
    assert all(torch.equal(a[~nan], b[~nan]) for a, b in zip(got, want))
    if nan.any():
        with pytest.raises(RuntimeError, match="gave up"):
            S.check_attention()
    S.check_attention()
    again = call()
    S.check_attention()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    return want, got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,h,hk,dim", [([40, 12], 32, 8, 64), ([30, 20], 8, 4, 128), ([9, 11], 32, 8, 128), ([33], 1, 1, 64)])
def test_the_last_wait_of_a_piece_runs_out(S, dtype, counts, h, hk, dim):
    """The softmax warps' wait for the output gives up by itself, in some lanes and not in others: whole warps go on.  One
    row tile and two, with rows to spare in each."""
    case = _tree_case([700, 300][:len(counts)], counts, h, hk, dim, 16, dtype, dim)
    assert _own_kernel(dtype, dim, h, hk, max(counts))
    for _ in range(4):
        _runs_out(S, case, max(counts), output_polls=0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h,hk,dim,page,most,longest", [(8, 2, 64, 16, 60, 200), (4, 2, 128, 48, 64, 150), (20, 4, 64, 32, 51, 90)])
def test_segments_behind_a_wait_that_ran_out_are_nan(S, dtype, h, hk, dim, page, most, longest):
    """CTAs whose runs go on over many segments: behind a wait that gave up none of them passes for whole."""
    rng = np.random.default_rng(most)
    counts = [int(c) for c in rng.integers(1, most + 1, 90)]
    counts[3] = most
    assert _own_kernel(dtype, dim, h, hk, most)
    case = _tree_case([int(c) for c in rng.integers(0, longest, 90)], counts, h, hk, dim, page, dtype, most)
    assert 90 * hk > 148          # more segments than CTAs
    want, got = _runs_out(S, case, most, polls=0)
    assert torch.isnan(got[0]).all() and torch.isnan(got[1]).all()
    for _ in range(3):
        _runs_out(S, case, most, output_polls=0)

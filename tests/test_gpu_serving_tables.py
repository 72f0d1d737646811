"""A step that runs out of pages, taken back and asked for again."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_step_that_lacked_pages_is_asked_for_again():
    """With the lengths and the pool of before the step, no page is lost or held twice."""
    from sili__new_b200 import serving as S
    page, pages, width = 16, 12, 8
    ring, pool = S.page_pool(pages)
    table = torch.full((4, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(4, dtype=torch.int32, device="cuda")
    fresh = torch.tensor([60, 30, 50, 0], dtype=torch.int32, device="cuda")      # 4 + 2 + 4 of 12 pages
    t = S.page_tables(lens, fresh, table, ring, pool, page, 160)
    assert t.status.tolist() == [0, 0, 0]
    lens, pool = t.lens, t.pool
    fresh = torch.tensor([0, 40, 0, 40], dtype=torch.int32, device="cuda")       # 3 + 3 more, where 2 are left
    t = S.page_tables(lens, fresh, table, ring, pool, page, 160)
    assert t.status.tolist() == [4, 0, 0] and int((t.slots[:80] >= 0).sum()) == 2 + 2 * page
    # the first request ends; the step is asked for again
    pool = S.release_pages(torch.tensor([True, False, False, False], device="cuda"), lens, table, ring, pool, page)
    t = S.page_tables(lens, fresh, table, ring, pool, page, 160)
    assert t.status.tolist() == [0, 0, 0] and t.lens.tolist() == [0, 70, 50, 40]
    held = table[table >= 0].tolist()
    assert len(held) == len(set(held)) == 5 + 4 + 3 == int(t.pool[0] - t.pool[1]) + pages
    # every token has a place of its own, in its request's pages
    slots = t.slots[:80].tolist()
    assert len(set(slots)) == 80 and min(slots) >= 0
    where = [(1, 30 + i) for i in range(40)] + [(3, i) for i in range(40)]
    assert slots == [int(table[r, x // page]) * page + x % page for r, x in where]
    # all of them end: every page is free, once
    pool = S.release_pages(torch.ones(4, dtype=torch.bool, device="cuda"), t.lens, table, ring, t.pool, page)
    assert int(pool[1] - pool[0]) == pages and sorted(ring.tolist()) == list(range(pages)) and bool((table == -1).all())

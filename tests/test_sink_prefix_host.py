"""Host bookkeeping of windows with sinks and of shared prefixes (CPU only)."""
import numpy as np
import pytest

from lnskv import NO_PAGE, BlockTables, LnskvError, PagePool, kv_p_start, sink_window_pages, window_pages


@pytest.mark.parametrize("window,sink", [(16, 4), (17, 16), (40, 17), (1, 1), (100, 0), (33, 200)])
def test_a_pool_of_sink_window_pages_never_runs_dry(window, sink):
    n = sink_window_pages(window, sink)
    pool, t = PagePool(n), BlockTables(1, 40)
    for pos in range(500):
        t.step_pages_sink(pool, 0, pos, window, sink)
        row = t.array()[0]
        for tok in range(pos + 1):
            attended = tok < sink or tok >= kv_p_start(pos, window)
            assert not attended or row[tok // 16] != NO_PAGE, (pos, tok)
        held = {p for p in range(40) if row[p] != NO_PAGE}
        assert held == {tok // 16 for tok in range(pos + 1) if tok < sink or tok >= kv_p_start(pos, window)} | \
            {p for p in range(-(-sink // 16)) if p <= pos // 16}


def test_without_sinks_it_is_the_plain_step():
    a, b = (PagePool(20), BlockTables(1, 20)), (PagePool(20), BlockTables(1, 20))
    for pos in range(300):
        a[1].step_pages(a[0], 0, pos, 50)
        b[1].step_pages_sink(b[0], 0, pos, 50, 0)
        assert np.array_equal(a[1].array(), b[1].array())
    assert sink_window_pages(50, 0) == window_pages(50) and sink_window_pages(0, 9) == 0


def test_sink_eviction_arguments():
    pool, t = PagePool(4), BlockTables(1, 4)
    for seq, sink in ((1, 0), (0, -1)):
        with pytest.raises(LnskvError):
            t.evict_kv_pages_sink(pool, seq, 5, 16, sink)
    t.ensure_kv_page(pool, 0, 20)
    t.evict_kv_pages_sink(pool, 0, 63, 0, 0)  # no window: nothing goes
    assert pool.num_free == 3


def _filled(pool, t, seq, n_tok):
    for p in range(0, n_tok, 16):
        t.ensure_kv_page(pool, seq, p)


def test_groups_of_forked_rows():
    pool, t = PagePool(100), BlockTables(9, 12)
    _filled(pool, t, 0, 75)   # 4 whole pages and a tail
    for c in (1, 2):
        t.fork_sequence(pool, 0, c, 75)
    _filled(pool, t, 3, 33)
    _filled(pool, t, 4, 160)  # 10 whole pages
    t.fork_sequence(pool, 4, 5, 100)  # 6 of them and a tail
    t.fork_sequence(pool, 4, 6, 48)   # 3 of them
    _filled(pool, t, 6, 60)
    assert t.shared_prefix_groups() == [(0, 3, 64), (4, 3, 48)]
    assert t.shared_prefix_groups(min_pages=4) == [(0, 3, 64), (4, 2, 96)]
    assert t.shared_prefix_groups(min_pages=5) == [(4, 2, 96)]
    assert t.shared_prefix_groups(n_seq=2) == [(0, 2, 64)]
    assert t.shared_prefix_groups(n_seq=0) == [] and t.shared_prefix_groups(n_seq=1) == []
    with pytest.raises(LnskvError):
        t.shared_prefix_groups(n_seq=10)
    with pytest.raises(LnskvError):
        t.shared_prefix_groups(min_pages=0)


def test_the_last_page_of_a_row_is_not_shared():
    """A row that ends on a page boundary may still be written there by its fork's steps."""
    pool, t = PagePool(20), BlockTables(2, 8)
    _filled(pool, t, 0, 64)
    t.fork_sequence(pool, 0, 1, 64)
    assert t.shared_prefix_groups() == [(0, 2, 48)]
    for s in (0, 1):
        t.ensure_kv_page(pool, s, 64)
    assert t.shared_prefix_groups() == [(0, 2, 64)]


def test_no_more_groups_than_a_call_takes():
    pool, t = PagePool(2000), BlockTables(300, 4)
    for s in range(0, 300, 2):
        _filled(pool, t, s, 40)
        t.fork_sequence(pool, s, s + 1, 40)
    g = t.shared_prefix_groups()
    assert len(g) == 128 and g[-1] == (254, 2, 32)


def test_evicted_pages_are_not_shared():
    pool, t = PagePool(20), BlockTables(2, 8)
    _filled(pool, t, 0, 80)
    t.fork_sequence(pool, 0, 1, 70)
    for s in (0, 1):
        t.evict_kv_pages(pool, s, 69, 40)
    assert t.array()[0, 0] == NO_PAGE
    assert t.shared_prefix_groups() == []

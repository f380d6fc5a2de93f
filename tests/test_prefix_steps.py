"""Which rows of a prepared batch share a prefix, and the shared step's refusals
that need no device. No GPU calls are made here."""

import ctypes

import numpy as np
import pytest

import ferric_amd
from ferric_amd.pool import PagePool
from ferric_amd.runner import PagedLimits, TpBatchRunner, _groups_to_c

LIB = ferric_amd.load()
LIMITS = PagedLimits(context_tokens=640, physical_page_count=400, page_table_stride=40)


def grown(pool, sid, tokens):
    st = pool.sequences[sid]
    pool._ensure(st, tokens)
    st.length = tokens


def test_forks_of_two_prompts_and_a_sequence_of_its_own():
    pool = PagePool(LIMITS, seed=3)
    a, b = pool.admit(100), pool.admit(37)  # 6 whole pages and 4 tokens; 2 and 5
    forks = [pool.fork(a)[0] for _ in range(3)]
    more = [pool.fork(b)[0] for _ in range(2)]
    alone = pool.admit(200)
    grown(pool, forks[1], 130)  # further on than the others: still 6 shared pages
    batch = pool.prepare([(s, 1) for s in [a, *forks, b, *more, alone]])
    assert PagePool.prefix_groups(batch) == [(0, 4, 6), (4, 3, 2)]
    assert PagePool.prefix_groups(batch, min_pages=3) == [(0, 4, 6)]
    assert PagePool.prefix_groups(batch, min_pages=7) == []
    assert PagePool.prefix_groups(pool.prepare([(a, 1), (b, 1), (forks[0], 1)])) == []  # runs only


def test_rows_of_one_sequence_share_what_none_of_them_writes():
    pool = PagePool(LIMITS, seed=4)
    a = pool.admit(62)
    batch = pool.prepare([(a, t) for t in range(5)])  # positions 62..66: pages 3 and 4 are written
    assert PagePool.prefix_groups(batch) == [(0, 5, 3)]
    b = pool.admit(0)
    assert PagePool.prefix_groups(pool.prepare([(b, 1), (b, 2)])) == []


def test_a_fork_at_a_page_boundary_and_forks_of_forks():
    pool = PagePool(LIMITS, seed=5)
    a = pool.admit(64)
    b, moves = pool.fork(a)
    assert moves == []
    grown(pool, b, 160)  # ten pages of its own list, four of them shared
    c, d = pool.fork(b)[0], pool.fork(b)[0]
    batch = pool.prepare([(s, 1) for s in (b, c, d, a)])
    # Three rows save 2 * 10 page reads; with the fourth they would share 4 pages and save 12.
    assert PagePool.prefix_groups(batch) == [(0, 3, 10)]
    batch = pool.prepare([(s, 1) for s in (a, b, c, d)])
    assert PagePool.prefix_groups(batch) == [(0, 4, 4)]


@pytest.mark.parametrize("seed", range(20))
def test_groups_are_what_the_step_asks_for(seed):
    r = np.random.default_rng(seed)
    pool = PagePool(LIMITS, seed=seed)
    live = [pool.admit(int(r.integers(0, 120)))]
    for _ in range(9):
        s = live[r.integers(len(live))]
        live.append(pool.fork(s)[0] if r.random() < 0.7 else pool.admit(int(r.integers(0, 60))))
        grown(pool, live[-1], pool.sequences[live[-1]].length + int(r.integers(0, 40)))
    rows = [(s, 1) for s in live for _ in range(1 + int(r.random() < 0.2))]
    batch = pool.prepare(rows)
    end = 0
    for first, count, pages in PagePool.prefix_groups(batch):
        assert first >= end and count >= 2 and pages >= 1
        end = first + count
        lists = [batch.rows[i] for i in range(first, end)]
        assert all(x.position // 16 >= pages for x in lists)
        assert all(list(x.physical_pages[:pages]) == list(lists[0].physical_pages[:pages]) for x in lists)
    assert end <= len(rows)


def test_group_lists_of_other_forms_are_refused():
    assert _groups_to_c([]).shape == (0, 3)
    assert _groups_to_c([(0, 2, 5)]).tolist() == [[0, 2, 5]]
    for bad in ([(0, 2)], [(0, 2, -1)], [(0, 2, 2**32)], [(0.0, 2.0, 1.0)], [0, 2, 5]):
        with pytest.raises(ValueError):
            _groups_to_c(bad)


def test_no_context():
    g = np.array([[0, 1, 1]], np.uint32)
    assert LIB.fh_execute_batch_shared(None, 1, None, 1, g.ctypes.data, 1, None, 0, None) == 1
    assert LIB.fh_execute_batch_shared(None, 1, None, 1, None, 0, None, 0, None) == 1
    n = ctypes.c_uint64()
    assert LIB.fh_expected_dispatch_count_shared(None, 1, None, 1, g.ctypes.data, 1, None, 0, ctypes.byref(n)) == 1


@pytest.mark.parametrize("rows,prefix,context,gains", [
    # Measured steps of Qwen3-0.6B and Qwen3-8B shapes, shared against not: slower in both, or faster in both.
    (2, 16, 1280, 0), (8, 64, 1280, 0), (16, 256, 1280, 0), (32, 256, 1280, 0), (32, 1024, 1280, 1), (8, 256, 4352, 0),
    (16, 1024, 4352, 1), (2, 64, 33024, 0), (4, 64, 33024, 0), (16, 16, 33024, 1), (32, 16, 33024, 1), (4, 4096, 33024, 1),
    (2, 32000, 33024, 1), (32, 32000, 33024, 1)])
def test_groups_that_gain(rows, prefix, context, gains):
    class Runner(TpBatchRunner):
        def __init__(self):
            self._lib, self.model = LIB, ferric_amd.QWEN3_8B
            self.limits = PagedLimits(context, context // 16 + 300, context // 16)

    runner = Runner()
    pool = PagePool(runner.limits, seed=1)
    live = [pool.admit(prefix + 5)]
    live += [pool.fork(live[0])[0] for _ in range(rows - 1)]
    batch = pool.prepare([(s, 1) for s in live])
    groups = PagePool.prefix_groups(batch)
    assert groups == [(0, rows, prefix // 16)]
    assert runner.gaining_groups(batch, groups) == (groups if gains else [])
    assert runner.gaining_groups(batch, []) == []


def test_gains_of_several_groups_add_up_and_refused_groups_have_none():
    def gain(groups, rows, heads=8, context=16384):
        g = np.array(groups, np.uint32).reshape(-1, 3)
        return LIB.fh_prefix_groups_gain(g.ctypes.data, len(g), rows, heads, context)

    # Of 140000: 34 * 8 rows * 8 heads * 32 parts of the context = 69632; 3 rows * 256 pages * 16 * 8 heads = 98304.
    assert gain([(0, 4, 256)], 8) == 1 and gain([(4, 4, 256)], 8) == 1 and gain([(0, 4, 256), (4, 4, 256)], 8) == 1
    assert gain([(0, 4, 128)], 8) == 0 and gain([(4, 4, 128)], 8) == 0 and gain([(0, 4, 128), (4, 4, 128)], 8) == 1
    assert gain([(0, 4, 128)], 8, heads=16) == 1  # heads count as keys do
    assert gain([], 32) == 0 and gain([(0, 32, 900)], 32) == 1
    for bad in ([(0, 33, 900)], [(0, 0, 900)], [(0, 32, 1025)], [(8, 8, 900), (0, 8, 900)]):
        assert gain(bad, 32) == 0
    assert gain([(0, 32, 900)], 0) == 0 and gain([(0, 32, 900)], 32, heads=0) == 0 and gain([(0, 32, 0)], 32, context=0) == 0
    assert LIB.fh_prefix_groups_gain(None, 1, 32, 8, 16384) == 0


@pytest.mark.parametrize("min_pages", [0, -3])
def test_no_group_without_pages(min_pages):
    """A step refuses a prefix of no pages, so none is listed."""
    pool = PagePool(LIMITS, seed=6)
    a, b = pool.admit(40), pool.admit(20)
    c, _ = pool.fork(b)
    batch = pool.prepare([(s, 1) for s in (a, b, c)])
    assert PagePool.prefix_groups(batch, min_pages=min_pages) == [(1, 2, 1)]
    d, e = pool.admit(0), pool.admit(5)
    assert PagePool.prefix_groups(pool.prepare([(d, 1), (e, 1)]), min_pages=min_pages) == []

"""Pages of the KV cache on any host: sequences that share pages in the pool
(fork, release, truncate, compaction), run against a model of the cache's
contents, and the lists of page moves that the library refuses. No GPU calls
are made here."""

import ctypes
import random

import numpy as np
import pytest

import ferric_amd
from ferric_amd import _lib
from ferric_amd.pool import PagePool
from ferric_amd.runner import PagedLimits, TpBatchRunner

LIB = ferric_amd.load()


class Cache:
    """One value a slot, moved as the kernels move pages."""

    def __init__(self, pages):
        self.slots = np.full((pages, 16), -1, np.int64)

    def move(self, moves):
        sources, targets = [m[0] for m in moves], [m[1] for m in moves]
        assert len(set(targets)) == len(targets) and not set(targets) & set(sources)
        for src, dst, n in moves:
            self.slots[dst, :n] = self.slots[src, :n]

    def write(self, batch):
        for r in batch.rows:
            self.slots[r.physical_pages[r.position // 16], r.position % 16] = r.token

    def read(self, pool, sid):
        st = pool.sequences[sid]
        return [int(self.slots[st.pages[i // 16], i % 16]) for i in range(st.length)]


def consistent(pool):
    """Every page is free once or owned as often as the pool counts."""
    owners = {}
    for st in pool.sequences.values():
        assert len(set(st.pages.tolist())) == len(st.pages)
        for p in st.pages.tolist():
            owners[p] = owners.get(p, 0) + 1
    assert sorted(list(owners) + pool.free) == list(range(pool.limits.physical_page_count))
    assert {p: n for p, n in owners.items() if n > 1} == pool._shared


def step(pool, cache, rows, texts):
    batch = pool.prepare(rows)
    cache.write(batch)
    pool.commit(batch)
    for s, t in rows:
        texts[s].append(t)


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 33])
def test_a_fork_has_the_tokens_and_only_the_last_page_of_its_own(length):
    pool, cache, texts = PagePool(PagedLimits(256, 40, 16), seed=4), Cache(40), {}
    a = pool.admit()
    texts[a] = []
    for t in range(length):
        step(pool, cache, [(a, t)], texts)
    b, moves = pool.fork(a)
    texts[b] = list(texts[a])
    assert moves == ([] if length % 16 == 0 else [(int(pool.sequences[a].pages[-1]), int(pool.sequences[b].pages[-1]), length % 16)])
    assert pool.sequences[a].pages[:length // 16].tolist() == pool.sequences[b].pages[:length // 16].tolist()
    cache.move(moves)
    consistent(pool)
    for t in range(40):  # both go on, in one batch
        step(pool, cache, [(a, 100 + t), (b, 200 + t)], texts)
    consistent(pool)
    assert cache.read(pool, a) == texts[a] and cache.read(pool, b) == texts[b]
    pool.release(a)
    consistent(pool)
    assert cache.read(pool, b) == texts[b]
    pool.release(b)
    consistent(pool)
    assert len(pool.free) == 40 and pool._shared == {}


def test_a_fork_without_a_free_page_changes_nothing():
    pool = PagePool(PagedLimits(256, 2, 16))
    a = pool.admit(20)
    with pytest.raises(MemoryError):
        pool.fork(a)
    consistent(pool)
    assert list(pool.sequences) == [a]
    pool.truncate(a, 16)  # its second page stays reserved
    b, moves = pool.fork(a)  # whole pages only: none is needed
    assert moves == [] and pool.sequences[b].pages.tolist() == pool.sequences[a].pages[:1].tolist()
    consistent(pool)


def test_a_commit_end_inside_shared_pages_is_refused():
    pool = PagePool(PagedLimits(256, 20, 16))
    a = pool.admit(40)
    b, _ = pool.fork(a)
    for sid in (a, b):
        with pytest.raises(ValueError):
            pool.truncate(sid, 31)  # would write into the second shared page
        pool.truncate(sid, 32)  # the next write goes to a page of its own
        pool.truncate(sid, 40 if sid == a else 33)
    pool.release(b)
    pool.truncate(a, 31)  # nobody shares it any more
    consistent(pool)


def test_random_forks_releases_and_compactions_keep_every_sequence():
    r = random.Random(7)
    for seed in range(6):
        pool, cache, texts = PagePool(PagedLimits(512, 60, 32), seed=seed), Cache(60), {}
        token = 0
        for _ in range(250):
            live = list(pool.sequences)
            what = r.random()
            try:
                if not live or what < 0.1:
                    texts[pool.admit()] = []
                elif what < 0.25:
                    a = r.choice(live)
                    b, moves = pool.fork(a)
                    cache.move(moves)
                    texts[b] = list(texts[a])
                elif what < 0.35:
                    s = r.choice(live)
                    pool.release(s)
                    del texts[s]
                elif what < 0.42:
                    cache.move(pool.compact())
                    used = {p for st in pool.sequences.values() for p in st.pages.tolist()}
                    assert used == set(range(len(used)))
                else:
                    rows = []
                    for s in r.sample(live, r.randint(1, len(live))):
                        for _ in range(r.randint(1, 3)):
                            token += 1
                            rows.append((s, token))
                    step(pool, cache, rows, texts)
            except MemoryError:
                for s in live[::2]:
                    pool.release(s)
                    del texts[s]
            consistent(pool)
            for s in pool.sequences:
                # A step that ran out of pages reserved some and committed nothing.
                assert cache.read(pool, s) == texts[s]


def test_compaction_of_a_compact_pool_moves_nothing():
    pool = PagePool(PagedLimits(256, 30, 16), shuffle=False)
    pool.free.reverse()  # takes 0, 1, 2, ...
    a = pool.admit(50)
    batch = pool.prepare([(a, 1)])
    assert pool.compact() == []
    pool.commit(batch)  # nothing moved: the batch still holds


def test_a_batch_of_before_a_compaction_is_not_committed():
    pool = PagePool(PagedLimits(256, 30, 16), shuffle=True, seed=1)
    a = pool.admit(50)
    batch = pool.prepare([(a, 1)])
    old = batch.rows[0].physical_pages.copy()
    assert pool.compact()
    assert np.array_equal(batch.rows[0].physical_pages, old)  # a snapshot
    with pytest.raises(ValueError):
        pool.commit(batch)
    after = pool.prepare([(a, 1)])
    assert after.rows[0].physical_pages.tolist() == pool.sequences[a].pages.tolist()
    pool.commit(after)


def test_decode_batches_after_a_compaction_list_the_new_pages():
    pool = PagePool(PagedLimits(256, 64, 16), seed=3)
    seqs = [pool.admit(20) for _ in range(8)]
    rows = [(s, 5) for s in seqs]
    pool.commit(pool.prepare(rows))  # the pool keeps this batch's page lists
    assert pool.compact()
    batch = pool.prepare(rows)
    for r in batch.rows:
        assert list(r.physical_pages) == pool.sequences[r.sequence].pages.tolist()


def refusal(moves, pages=64, caches=1, stride=0, kvh=8, pointer=4096):
    a = np.array(moves, np.uint32).reshape(-1, 3)
    return LIB.fh_op_kv_copy_pages(pointer, caches, stride, a.ctypes.data if len(a) else None, len(a), kvh, pages, None)


def test_moves_the_library_refuses():
    """Refused by the host before any launch: the cache pointers here are no memory."""
    many = [(40 + i, i, 16) for i in range(20)]  # more than the short lists' check
    for bad in ([(64, 1, 16)], [(1, 64, 16)], [(1, 2, 17)], [(1, 1, 16)], [(1, 2, 16), (3, 2, 1)], [(1, 2, 16), (2, 3, 1)],
                [(1, 2, 0), (2, 3, 0)], many + [(60, 3, 1)], many + [(3, 63, 1)], many + [(63, 40, 1)]):
        assert refusal(bad) == 1, bad
        assert b"KV move" in LIB.fh_last_error(None)
    page = 16 * 8 * 128
    for kwargs in (dict(pointer=None), dict(pointer=4104), dict(caches=0), dict(caches=65536, stride=64 * page),
                   dict(caches=2, stride=64 * page - 8), dict(caches=2, stride=64 * page + 4), dict(kvh=0), dict(pages=0)):
        assert refusal([(1, 2, 3)], **kwargs) == 1, kwargs
    assert LIB.fh_op_kv_copy_pages(4096, 1, 0, None, 1, 8, 64, None) == 1
    assert refusal([]) == 0  # nothing to copy
    assert LIB.fh_kv_copy_pages(None, None, 0) == 1


def test_the_runner_refuses_moves_that_are_none():
    class Runner(TpBatchRunner):
        def __init__(self):
            self._ctx = None

    for bad in ([(1, 2)], [1, 2, 3], [(-1, 2, 3)], [(1, 2, 2**32)], [(1.0, 2.0, 3.0)]):
        with pytest.raises(ValueError):
            Runner.copy_kv_pages(Runner(), bad)
    assert ctypes.sizeof(_lib.KvMove) == 12

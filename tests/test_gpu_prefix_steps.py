"""Decode steps whose rows share prefixes, against the same steps without groups.

The two attentions differ by the order of FP32 sums, so by at most one bf16
step, 2^-7 of the value, in elements of their outputs that lie at a rounding's
edge. Through a layer a relative change of the residual stream's norm grows by
at most 1 (the stream) + 3 (the MLP: gate, up and silu's slope of 1.1 each once);
with one in each of two layers the logits' norm changes by at most 2^-7 * 4 * 4
= 2^-3 (2^-7 is reached only if every element lay at an edge). Rows that saw
another prefix, or lost it, are off by about 1. Replays of a step have to
give the eager step's bits."""

import ctypes

import numpy as np
import pytest

import ferric_amd
from ferric_amd import PagedLimits, PagePool, TpBatchRunner, _lib

pytestmark = pytest.mark.gpu

LIMITS = PagedLimits(context_tokens=768, physical_page_count=300, page_table_stride=48)
VOCABULARY = 4096


def model(base, layers=2):
    cfg = dict(base)
    cfg.update(layers=layers, vocabulary=VOCABULARY)
    return cfg


def start(base, prompts, forks, graphs=True, seed=5, capacity=32):
    """A runner whose sequences are `forks` forks of each prompt, behind one another."""
    runner = TpBatchRunner(model(base), LIMITS, row_capacity=capacity, use_graphs=graphs, prefill_rows=512)
    runner.synthesize_weights(seed=seed, sigma=0.02)
    pool = PagePool(LIMITS, seed=9)
    r = np.random.default_rng(seed)
    rows = []
    for tokens in prompts:
        a = pool.admit()
        batch = pool.prepare([(a, int(t)) for t in r.integers(0, VOCABULARY, tokens)])
        runner.execute_batch(batch, [])
        pool.commit(batch)
        rows.append(a)
        for _ in range(forks):
            b, moves = pool.fork(a)
            runner.copy_kv_pages(moves)
            rows.append(b)
    return runner, pool, rows


def step(runner, pool, rows, tokens, groups, commit=True):
    batch = pool.prepare(list(zip(rows, tokens)))
    groups = PagePool.prefix_groups(batch) if groups is True else groups
    outs = list(range(len(rows)))
    (expected,) = runner.expected_dispatch_counts_for_selection(batch, outs, groups)
    (before,) = runner.dispatch_counts()
    out = runner.execute_batch(batch, outs, groups)
    assert runner.dispatch_counts()[0] - before == expected
    if commit:
        pool.commit(batch)
    return out.choices, runner.read_logits(), groups


def off(a, b):
    return np.linalg.norm(a.astype(np.float64) - b, axis=1) / np.linalg.norm(b.astype(np.float64), axis=1)


@pytest.mark.parametrize("base", [ferric_amd.QWEN3_8B, ferric_amd.QWEN3_0_6B], ids=["8b", "0.6b"])
@pytest.mark.parametrize("prompts,forks", [([300], 0), ([300], 2), ([333, 96], 6), ([400], 31), ([70, 17, 200], 3)])
def test_shared_steps_equal_plain_ones(base, prompts, forks):
    runner, pool, rows = start(base, prompts, forks)
    try:
        r = np.random.default_rng(1)
        for _ in range(3):
            tokens = r.integers(0, VOCABULARY, len(rows)).tolist()
            _, want, _ = step(runner, pool, rows, tokens, (), commit=False)
            groups = True if len(rows) > 1 else [(0, 1, 18)]  # a group of one row is one, too
            _, got, used = step(runner, pool, rows, tokens, groups)
            assert len(used) == len(prompts)
            assert off(got, want).max() <= 2.0 ** -3
            assert np.isfinite(got).all()
    finally:
        runner.close()


def test_replays_and_changes_of_groups_give_the_eager_bits():
    pairs = [start(ferric_amd.QWEN3_0_6B, [300, 123], 3, graphs=g) for g in (True, False)]
    try:
        r = np.random.default_rng(2)
        kinds = [True, True, True, True, (), True, [(0, 4, 18)], [(0, 4, 18)], [(0, 2, 9), (4, 4, 7)], True, (), True, True]
        for i, groups in enumerate(kinds):
            n = 8 if i != 5 else 4
            tokens = r.integers(0, VOCABULARY, n).tolist()
            (ca, la, ga), (cb, lb, gb) = (step(x, p, rows[:n], tokens, groups) for x, p, rows in pairs)
            assert ga == gb and ca == cb and np.array_equal(la, lb), (i, groups)
    finally:
        for x, _, _ in pairs:
            x.close()


def test_rows_of_one_sequence_in_a_shared_step():
    """A verify of drafted tokens: later rows read the slots that earlier ones write in the same step."""
    runner, pool, rows = start(ferric_amd.QWEN3_8B, [250], 2)
    try:
        tokens = np.random.default_rng(3).integers(0, VOCABULARY, 9).tolist()
        verify = [rows[0]] * 5 + [rows[1]] * 3 + [rows[2]]
        _, want, _ = step(runner, pool, verify, tokens, (), commit=False)
        _, got, used = step(runner, pool, verify, tokens, True)
        assert used == [(0, 9, 15)]
        assert off(got, want).max() <= 2.0 ** -3
    finally:
        runner.close()


def test_refusals_leave_the_context_usable():
    runner, pool, rows = start(ferric_amd.QWEN3_0_6B, [100], 2, capacity=8)
    try:
        alone = pool.admit()
        rows.append(alone)
        batch = pool.prepare([(s, 5) for s in rows])
        outs = list(range(4))
        for bad in ([(0, 3, 7)], [(0, 4, 1)], [(0, 3, 0)], [(0, 5, 1)], [(1, 2, 3), (0, 1, 3)], [(0, 0, 1)], [(0, 3, 2**20)],
                    [(0, 3, 2**32 - 1)]):
            with pytest.raises(ferric_amd.FerricError) as refused:
                runner.execute_batch(batch, outs, bad)
            assert refused.value.status == 1 and "prefix groups" in str(refused.value)
            with pytest.raises(ferric_amd.FerricError):
                runner.expected_dispatch_counts_for_selection(batch, outs, bad)
        runner.execute_batch(batch, outs, [(0, 3, 6)])
        pool.commit(batch)
        long = pool.prepare([(alone, t) for t in range(20)])
        with pytest.raises(ferric_amd.FerricError) as refused:  # a prefill chunk
            runner.execute_batch(long, [], [(0, 1, 1)])
        assert refused.value.status == 1
        runner.execute_batch(long, [])
        pool.commit(long)
        ms = ctypes.c_float()
        assert _lib.load().fh_time_attention(runner._ctx, 2, ctypes.byref(ms)) != 0  # the last batch was a chunk
        step(runner, pool, rows, [1, 2, 3, 4], True)
        assert _lib.load().fh_time_attention(runner._ctx, 3, ctypes.byref(ms)) == 0 and ms.value > 0
    finally:
        runner.close()


def test_profiled_and_repeated_steps_with_growing_scratch():
    runner, pool, rows = start(ferric_amd.QWEN3_8B, [260], 20)
    try:
        for n in (2, 5, 21, 3, 21, 21):
            tokens = np.random.default_rng(n).integers(0, VOCABULARY, n).tolist()
            _, want, _ = step(runner, pool, rows[:n], tokens, (), commit=False)
            _, got, _ = step(runner, pool, rows[:n], tokens, True, commit=False)
            assert off(got, want).max() <= 2.0 ** -3
        assert _lib.load().fh_set_profiling(runner._ctx, 1) == 0
        _, again, _ = step(runner, pool, rows[:21], tokens, True, commit=False)
        assert np.array_equal(again, got)
    finally:
        runner.close()


# ---- what a step writes and reads ---------------------------------------------------
# The bound on the logits is too wide to show one key of hundreds. Here the value of one slot is made to outweigh
# the others' sum in every layer, and a plain step that reads zeros in its place shows what losing it would do.

def edit_slots(runner, slots, values, which=(0, 1)):
    """values(layer, which) [kv_heads * 128] bits into the slots [(page, slot)] of every layer."""
    pages = {}
    for page, slot in slots:
        pages.setdefault(int(page), []).append(slot)
    for layer in range(runner.model["layers"]):
        for w in which:
            for page, at in pages.items():
                data = runner.read_kv_page(layer, w, page).reshape(16, -1)
                data[at] = values(layer, w)
                runner.write_kv_page(layer, w, page, data)


def written(pool, rows):
    """(page, slot) of each row's new token."""
    batch = pool.prepare([(s, 0) for s in rows])
    return [(r.physical_pages[r.position // 16], r.position % 16) for r in batch.rows]


def read_slots(runner, slots):
    return np.array([[[runner.read_kv_page(layer, w, int(p)).reshape(16, -1)[s] for p, s in slots] for w in range(2)]
                     for layer in range(runner.model["layers"])])


NAN = 0x7FC0


@pytest.mark.parametrize("base", [ferric_amd.QWEN3_8B, ferric_amd.QWEN3_0_6B], ids=["8b", "0.6b"])
@pytest.mark.parametrize("prompts,forks,per", [([300], 2, 1), ([333, 96], 6, 1), ([250], 2, 3), ([304], 31, 1)])
def test_a_shared_step_writes_its_slots_before_it_reads_them(base, prompts, forks, per):
    """The slots hold NaN before the step: a row that read one would end the step with an error."""
    runner, pool, rows = start(base, prompts, forks)
    try:
        rows = [s for s in rows for _ in range(per)]
        slots = written(pool, rows)
        tokens = np.random.default_rng(4).integers(0, VOCABULARY, len(rows)).tolist()
        edit_slots(runner, slots, lambda layer, w: NAN)
        _, want, _ = step(runner, pool, rows, tokens, (), commit=False)
        plain = read_slots(runner, slots)
        for _ in range(3):  # eager, captured, replayed
            edit_slots(runner, slots, lambda layer, w: NAN)
            _, got, used = step(runner, pool, rows, tokens, True, commit=False)
            assert len(used) == len(prompts)
            new = read_slots(runner, slots)
            assert np.array_equal(new[0], plain[0])  # the first layer's keys and values do not depend on attention
            assert np.all((new & 0x7F80) != 0x7F80)
            assert off(got, want).max() <= 2.0 ** -3
    finally:
        runner.close()


def outweigh(runner, pool, rows, tokens, slots, value, groups=True):
    """A shared step with a value at the slots against a plain one, and against one that reads zeros there."""
    signs = np.where(np.random.default_rng(6).random(runner.model["kv_heads"] * 128) < 0.5, 0x8000, 0).astype(np.uint16)
    kept = read_slots(runner, slots)
    edit_slots(runner, slots, lambda layer, w: value | signs, which=(1,))
    _, want, _ = step(runner, pool, rows, tokens, (), commit=False)
    _, got, used = step(runner, pool, rows, tokens, groups, commit=False)
    edit_slots(runner, slots, lambda layer, w: 0, which=(1,))
    _, lost, _ = step(runner, pool, rows, tokens, (), commit=False)
    for i, slot in enumerate(slots):
        edit_slots(runner, [slot], lambda layer, w: kept[layer, w, i], which=(1,))
    assert off(got, want).max() <= 2.0 ** -3
    assert off(lost, want).min() > 2.0 ** -2
    return used


@pytest.mark.parametrize("base", [ferric_amd.QWEN3_8B, ferric_amd.QWEN3_0_6B], ids=["8b", "0.6b"])
@pytest.mark.parametrize("forks", [2, 11, 31])
def test_a_shared_step_reads_every_rows_keys(base, forks):
    runner, pool, rows = start(base, [301], forks)
    try:
        lists = [pool.sequences[s].pages for s in rows]
        tokens = np.random.default_rng(5).integers(0, VOCABULARY, len(rows)).tolist()
        for t in (0, 15, 127, 128, 255, 287, 288, 300):  # ends of pages and chunks, of the prefix and of the own keys
            slots = sorted({(int(pages[t // 16]), t % 16) for pages in lists})
            assert len(slots) == (1 if t < 288 else len(rows))
            used = outweigh(runner, pool, rows, tokens, slots, 0x4580)  # 2^12
            assert used == [(0, len(rows), 18)]
    finally:
        runner.close()


@pytest.mark.parametrize("pages", [1030, 1541])
def test_steps_behind_long_prefixes(pages):
    """32 rows of four heads behind a prefix long enough for blocks of 128 vectors, the longer one streamed."""
    limits = PagedLimits(context_tokens=25600, physical_page_count=1700, page_table_stride=1600)
    runner = TpBatchRunner(model(ferric_amd.QWEN3_8B), limits, row_capacity=32)
    try:
        runner.synthesize_weights(seed=5, sigma=0.02)
        pool = PagePool(limits, seed=9)
        a = pool.admit(16 * pages + 5)
        r = np.random.default_rng(1)
        first = [int(p) for p in pool.sequences[a].pages[:7]]  # content, repeated over the rest of the list
        for layer in range(2):
            for w in range(2):
                for p in first:
                    runner.write_kv_page(layer, w, p, (r.standard_normal(16 * 1024).astype(np.float32).view(np.uint32) >> 16)
                                         .astype(np.uint16))
        runner.copy_kv_pages([(first[i % 7], int(p), 16) for i, p in enumerate(pool.sequences[a].pages) if i >= 7])
        rows = [a]
        for _ in range(31):
            b, moves = pool.fork(a)
            runner.copy_kv_pages(moves)
            rows.append(b)
        tokens = r.integers(0, VOCABULARY, 32).tolist()
        lists = [pool.sequences[s].pages for s in rows]
        for t in (0, 63, 64, 511, 512, 831, 832, 16 * pages - 1, 16 * pages, 16 * pages + 4):
            slots = sorted({(int(p[t // 16]), t % 16) for p in lists})
            used = outweigh(runner, pool, rows, tokens, slots, 0x4780)  # 2^16
            assert used == [(0, 32, pages)]
        slots = written(pool, rows)
        edit_slots(runner, slots, lambda layer, w: NAN)
        _, want, _ = step(runner, pool, rows, tokens, (), commit=False)
        plain = read_slots(runner, slots)
        edit_slots(runner, slots, lambda layer, w: NAN)
        _, got, _ = step(runner, pool, rows, tokens, True, commit=False)
        assert np.array_equal(read_slots(runner, slots)[0], plain[0])
        assert off(got, want).max() <= 2.0 ** -3
    finally:
        runner.close()

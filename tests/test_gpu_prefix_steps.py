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

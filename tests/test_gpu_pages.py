"""KV page copies on the GPU: the kernel root against the same copies on the
host (every byte of the buffers, what lies between and behind them included),
and forks and compactions of a context's sequences, whose steps have to give
the bits of sequences that never shared a page."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tests import devutil as du  # noqa: E402
import ferric_amd  # noqa: E402
from ferric_amd import PagedLimits, PagePool, TpBatchRunner, _lib  # noqa: E402

LIB = ferric_amd.load()


def moves_of(r, pages, count, slots=None, fan=False):
    order = r.permutation(pages)
    m = np.empty((count, 3), np.uint32)
    m[:, 1] = order[:count]
    m[:, 0] = order[count] if fan else order[count:][r.integers(0, pages - count, count)]
    m[:, 2] = r.integers(0, 17, count) if slots is None else slots
    return m


def copy_host(caches, moves):
    """caches: [count, pages, 16, width], moved in place."""
    for src, dst, n in moves.tolist():
        caches[:, dst, :n] = caches[:, src, :n]


def call(caches, count, stride, moves, kvh, pages, stream=None):
    _lib.check(LIB.fh_op_kv_copy_pages(caches.data_ptr(), count, stride, moves.ctypes.data, len(moves), kvh, pages,
                                       du.stream() if stream is None else stream))


@pytest.mark.parametrize("kvh,caches,pages,count,gap", [(8, 1, 20, 1, 0), (8, 72, 40, 13, 8), (1, 5, 700, 300, 64),
                                                        (2, 3, 600, 512, 0), (3, 2, 513, 256, 24), (8, 2, 600, 257, 8)])
@pytest.mark.parametrize("slots", [None, 16, 5, 0])
def test_copies_equal_those_of_the_host(kvh, caches, pages, count, gap, slots):
    r = np.random.default_rng(pages + count)
    moves = moves_of(r, pages, count if pages > count else pages - 1, slots, fan=slots == 5)
    page = 16 * kvh * 128
    stride = pages * page + gap
    flat = r.integers(0, 65536, caches * stride + 256, dtype=np.uint64).astype(np.uint16)
    dev = du.to_dev(flat)
    call(dev, caches, stride, moves, kvh, pages)
    whole = flat[:caches * stride].reshape(caches, stride)[:, :pages * page].reshape(caches, pages, 16, kvh * 128).copy()
    copy_host(whole, moves)
    flat[:caches * stride].reshape(caches, stride)[:, :pages * page] = whole.reshape(caches, -1)
    assert np.array_equal(du.to_host(dev, np.uint16), flat)


def test_pages_beyond_32_bits_of_offset():
    kvh, pages = 8, 270_000  # 4.4e9 elements
    page = 16 * kvh * 128
    cache = torch.zeros(pages * page, dtype=torch.int16, device="cuda")
    view = cache.view(pages, 16, kvh * 128)
    last = torch.arange(page, device="cuda").to(torch.int16).view(16, -1)
    view[pages - 1] = last
    view[3] = -last
    moves = np.array([[pages - 1, 5, 16], [3, pages - 2, 7]], np.uint32)
    call(cache, 1, 0, moves, kvh, pages)
    torch.cuda.synchronize()
    assert torch.equal(view[5], last) and torch.equal(view[pages - 2, :7], -last[:7])
    assert int(view[pages - 2, 7:].abs().max()) == 0 and int(view[6:pages - 2].abs().amax()) == 0


def test_copies_on_another_stream_and_in_a_replayed_graph():
    r = np.random.default_rng(3)
    pages, kvh, caches = 400, 8, 4
    page = 16 * kvh * 128
    moves = moves_of(r, pages, 300)
    host = r.integers(0, 65536, caches * pages * page, dtype=np.uint64).astype(np.uint16)
    want = host.reshape(caches, pages, 16, -1).copy()
    copy_host(want, moves)
    side = torch.cuda.Stream()
    dev = du.to_dev(host)
    side.wait_stream(torch.cuda.current_stream())
    call(dev, caches, pages * page, moves, kvh, pages, side.cuda_stream)
    side.synchronize()
    assert np.array_equal(du.to_host(dev, np.uint16), want.reshape(-1))
    fresh, dev = du.to_dev(host), du.to_dev(host)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        listed = moves.copy()
        call(dev, caches, pages * page, listed, kvh, pages)
        listed[:] = 0  # the list is the caller's again after the call
    for _ in range(3):
        dev.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(du.to_host(dev, np.uint16), want.reshape(-1))


def small_model(layers=2):
    cfg = dict(ferric_amd.QWEN3_0_6B)
    cfg.update(layers=layers, vocabulary=4096)
    return cfg


def run(runner, pool, rows):
    batch = pool.prepare(rows)
    out = runner.execute_batch(batch, list(range(len(rows))))
    pool.commit(batch)
    return out.choices, runner.read_logits()


def test_forked_and_compacted_sequences_step_like_ones_that_share_nothing():
    limits = PagedLimits(context_tokens=512, physical_page_count=96, page_table_stride=32)
    runner = TpBatchRunner(small_model(), limits, row_capacity=8, prefill_rows=64)
    try:
        runner.synthesize_weights(seed=5, sigma=0.02)
        pool = PagePool(limits, seed=9)
        prompt = np.random.default_rng(0).integers(0, 4096, 37).tolist()
        a, c = pool.admit(), pool.admit()
        for s in (a, c):  # c runs the same prompt on pages of its own
            run(runner, pool, [(s, t) for t in prompt])
        b, moves = pool.fork(a)
        runner.copy_kv_pages(moves)
        d, more = pool.fork(b)
        runner.copy_kv_pages(more)
        e = pool.admit()
        run(runner, pool, [(e, t) for t in prompt])
        for t in range(3):
            # One row each: pages shared by sequences of one batch are read only.
            for token, shared, own in ((11 + t, b, c), (900 + t, d, e)):
                got, want = run(runner, pool, [(shared, token)]), run(runner, pool, [(own, token)])
                assert got[0] == want[0] and np.array_equal(got[1], want[1])
        _, before = run(runner, pool, [(b, 7), (d, 8), (a, 9)])
        _, apart = run(runner, pool, [(c, 7), (e, 8)])
        assert np.array_equal(before[:2], apart)
        pool.release(e)
        moves = pool.compact()
        assert moves
        runner.copy_kv_pages(moves)
        got, want = run(runner, pool, [(b, 21)]), run(runner, pool, [(c, 21)])
        assert got[0] == want[0] and np.array_equal(got[1], want[1])
        with pytest.raises(ferric_amd.FerricError) as refused:
            runner.copy_kv_pages([(1, 2, 16), (2, 3, 16)])
        assert refused.value.status == 1
        run(runner, pool, [(a, 3)])  # a refusal does not poison
    finally:
        runner.close()


def test_moves_reach_every_layer_of_k_and_v_and_no_other_page():
    limits = PagedLimits(context_tokens=128, physical_page_count=8, page_table_stride=8)
    runner = TpBatchRunner(small_model(3), limits, row_capacity=2)
    try:
        r = np.random.default_rng(2)
        content = r.integers(0, 65536, (3, 2, 8, 16, 1024), dtype=np.uint64).astype(np.uint16)
        for l in range(3):
            for w in range(2):
                for p in range(8):
                    runner.write_kv_page(l, w, p, content[l, w, p].reshape(-1))
        runner.copy_kv_pages([(7, 0, 3), (7, 1, 16), (2, 5, 0)])
        content[:, :, 0, :3] = content[:, :, 7, :3]
        content[:, :, 1] = content[:, :, 7]
        for l in range(3):
            for w in range(2):
                assert np.array_equal(runner.read_kv_cache(l, w), content[l, w].reshape(-1))
    finally:
        runner.close()


@pytest.mark.parametrize("count", [255, 700])
def test_calls_of_more_than_the_caches_hold(count):
    """From 256 MB on the copies stream past the caches: one launch and several, whole pages and parts of them."""
    r = np.random.default_rng(count)
    kvh, caches, pages = 8, 72, 1500
    moves = moves_of(r, pages, count, 16 if count < 256 else None)
    assert int(moves[:, 2].sum()) * kvh * 256 * caches >= 1 << 28
    g = torch.Generator(device="cuda").manual_seed(count)
    dev = torch.empty(caches, pages, 16, kvh * 128, dtype=torch.int16, device="cuda").random_(-32768, 32768, generator=g)
    want = dev.clone()
    src, dst, n = (torch.from_numpy(moves[:, i].astype(np.int64)).cuda() for i in range(3))
    kept = (torch.arange(16, device="cuda")[None, :] < n[:, None])[:, :, None]
    for c in range(caches):  # no destination is a source or occurs twice
        want[c, dst] = torch.where(kept, want[c, src], want[c, dst])
    call(dev, caches, pages * 16 * kvh * 128, moves, kvh, pages)
    torch.cuda.synchronize()
    assert torch.equal(dev, want)

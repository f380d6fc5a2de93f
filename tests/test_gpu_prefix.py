"""Shared-prefix attention on the GPU against the formula in 64 bits.

Tolerance, from the roundings: a score is an FP32 sum of 128 products, off by at
most 128 * 2^-24 * sum |q k| / sqrt(128), and enters an exponential (2^-22
relative, its argument one more rounding of the score); a probability enters
the value product in two bf16 terms (2^-17 relative); the sums of the values
and of the denominators are FP32 (one rounding of 2^-24 per key at most). With
w the exact weights, the output is off by at most (2 d + 2^-16 + keys 2^-24) *
sum w |v| plus half a bf16 step, 2^-8 of the value. Every slot that is no key of
a row, and every page that no row lists, holds NaN."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tests import devutil as du  # noqa: E402
import ferric_amd  # noqa: E402
from ferric_amd import _lib  # noqa: E402

LIB = ferric_amd.load()
NAN = float("nan")


class Batch:
    """groups: [(rows' own lengths, prefix pages)]; a group of prefix 0 is given as rows in no group. `per`: rows of
    one sequence at consecutive positions, the last one at the own length."""

    def __init__(self, seed, groups, qh, kvh, sharp=2.0, extra_stride=1, per=1, list_empty=False):
        r = np.random.default_rng(seed)
        self.qh, self.kvh = qh, kvh
        lengths, self.groups, rows = [], [], []
        for owns, prefix in groups:
            if prefix or list_empty:
                self.groups.append((len(lengths), len(owns) * per, prefix))
            for own in owns:
                for i in range(per):
                    lengths.append(prefix * 16 + own - per + 1 + i)
        self.lengths = np.array(lengths)
        assert self.lengths.min() >= 1
        self.rows = len(lengths)
        self.stride = int(-(-self.lengths.max() // 16)) + extra_stride
        self.context = self.stride * 16
        need = sum(p for _, p in groups) + sum(-(-own // 16) for owns, _ in groups for own in owns)
        self.pages = need + 5
        free = list(r.permutation(self.pages))
        table = np.full((self.rows, self.stride), 0xFFFFFFFF, np.uint32)
        k = torch.full((self.pages, 16, kvh, 128), NAN, dtype=torch.bfloat16)
        v = k.clone()
        at = 0
        for owns, prefix in groups:
            shared = [free.pop() for _ in range(prefix)]
            for own in owns:
                mine = shared + [free.pop() for _ in range(-(-own // 16))]
                for _ in range(per):
                    table[at, :len(mine)] = mine
                    at += 1
                for i, page in enumerate(mine):
                    n = min(16, prefix * 16 + own - 16 * i)
                    if i < prefix and not torch.isnan(k[page, 0, 0, 0]):
                        continue  # the prefix is written once
                    k[page, :n] = torch.from_numpy(r.standard_normal((n, kvh, 128)).astype(np.float32)).bfloat16()
                    v[page, :n] = torch.from_numpy(r.standard_normal((n, kvh, 128)).astype(np.float32)).bfloat16()
        self.table = table
        self.q = torch.from_numpy((r.standard_normal((self.rows, qh, 128)) * sharp).astype(np.float32)).bfloat16()
        self.k, self.v = k, v

    def device(self):
        self.d = dict(q=self.q.cuda(), k=self.k.cuda(), v=self.v.cuda(), table=du.to_dev(self.table),
                      pos=du.to_dev((self.lengths - 1).astype(np.uint32)))
        return self

    def exact(self, rows=None):
        """(output, tolerance) in 64 bits, per row."""
        g = self.qh // self.kvh
        want = torch.zeros(self.rows, self.qh, 128, dtype=torch.float64)
        tol = torch.zeros_like(want)
        for r in range(self.rows) if rows is None else rows:
            n = int(self.lengths[r])
            idx = torch.from_numpy(self.table[r, :-(-n // 16)].astype(np.int64))
            k = self.k[idx].reshape(-1, self.kvh, 128)[:n].double().permute(1, 0, 2)  # [kvh][n][128]
            v = self.v[idx].reshape(-1, self.kvh, 128)[:n].double().permute(1, 0, 2)
            q = self.q[r].double().view(self.kvh, g, 128)
            s = q @ k.transpose(1, 2) / math.sqrt(128)
            most = (q.abs() @ k.abs().transpose(1, 2)).amax((1, 2)).view(-1, 1, 1) / math.sqrt(128)
            w = torch.softmax(s, -1)
            want[r] = (w @ v).view(self.qh, 128)
            d = 128 * 2.0 ** -24 * most + 2.0 ** -22 + 2.0 ** -23 * s.abs().amax()
            a = (w @ v.abs()) * (2 * d + 2.0 ** -16 + n * 2.0 ** -24)
            tol[r] = a.reshape(self.qh, 128)
        return want, tol + 2.0 ** -8 * (want.abs() + tol)

    def scratch(self, groups=None):
        g = self.group_array(groups)
        n = LIB.fh_prefix_attention_scratch_bytes(g.ctypes.data, len(g), self.rows, self.qh, self.kvh, self.context)
        assert n > 0
        return torch.full((n // 4 + 64,), NAN, device="cuda"), n

    def group_array(self, groups=None):
        return np.array(self.groups if groups is None else groups, np.uint32).reshape(-1, 3)

    def run(self, tiled=0, groups=None, scratch=None, out=None, stream=None, context=None):
        """(output bits, error word); the scratch's and the output's ends are checked."""
        g = self.group_array(groups)
        buf, n = scratch or self.scratch(groups)
        rows = int(LIB.fh_activation_rows(self.rows)) if tiled else self.rows
        out = du.to_dev(np.full((rows + 1) * self.qh * 128, 0x1357, np.uint16)) if out is None else out
        err = du.empty(1, np.uint32)
        _lib.check(LIB.fh_op_prefix_attention(
            self.d["q"].data_ptr(), self.d["k"].data_ptr(), self.d["v"].data_ptr(), du.ptr(self.d["pos"]),
            du.ptr(self.d["table"]), g.ctypes.data, len(g), du.ptr(out), tiled, du.ptr(buf), n, self.rows, self.qh,
            self.kvh, self.stride, self.pages, context or self.context, du.ptr(err), stream or du.stream()))
        torch.cuda.synchronize()
        assert bool(torch.isnan(buf[n // 4:]).all())
        got = du.to_host(out, np.uint16)
        assert np.all(got[rows * self.qh * 128:] == 0x1357)
        return got[:rows * self.qh * 128], int(du.to_host(err, np.uint32)[0])


def values(bits, batch):
    return torch.from_numpy((bits.astype(np.uint32) << 16).view(np.float32)).double().view(-1, batch.qh, 128)


def holds(batch, bits, rows=None):
    want, tol = batch.exact(rows)
    rows = range(batch.rows) if rows is None else rows
    got = values(bits, batch)
    for r in rows:
        off = (got[r] - want[r]).abs()
        assert bool((off <= tol[r]).all()), (r, float((off / tol[r]).max()))


PATTERNS = {
    "one row": [([1], 1)],
    "one row alone": [([1], 0)],
    "two": [([5, 40], 2)],
    "no own keys": [([0, 1, 16, 17], 3)],
    "exact chunks": [([512, 513, 1, 511], 8)],
    "two groups and two rows of their own": [([3, 700, 20], 9), ([33], 0), ([64, 1], 21), ([1], 0)],
    "a full batch": [(list(range(1, 320, 10)), 33)],
    "33 rows": [([7] * 32 + [600], 5)],
    "100 rows and others": [([(i * 37) % 90 for i in range(100)], 17), ([9], 0), ([1] * 20, 1)],
    "long": [([1, 30, 9], 513), ([1100], 0)],
}


@pytest.mark.parametrize("heads", [(32, 8), (16, 8), (8, 8), (64, 8), (4, 1), (6, 3)])
@pytest.mark.parametrize("name", list(PATTERNS))
def test_equals_the_formula(name, heads):
    b = Batch(len(name), PATTERNS[name], *heads).device()
    bits, err = b.run()
    assert err == 0
    holds(b, bits)


@pytest.mark.parametrize("per,own", [(2, 2), (5, 5), (5, 21), (8, 40)])
def test_several_rows_of_a_sequence(per, own):
    b = Batch(per, [([own, own + 16, own + 1], 6), ([own], 0)], 32, 8, per=per).device()
    bits, err = b.run()
    assert err == 0
    holds(b, bits)


@pytest.mark.parametrize("heads", [(32, 8), (16, 8), (8, 8), (64, 8), (4, 4)])
@pytest.mark.parametrize("per,own", [(3, 3), (4, 18), (5, 600), (9, 33), (17, 1500), (17, 17)])
def test_runs_of_rows_of_one_sequence(per, own, heads):
    """Runs that end inside and at the rows taken together, that cross pages, and whose keys are cut into parts."""
    b = Batch(per + own, [([own, own + 15], 3), ([own + 2], 0), ([per], 1)], *heads, per=per).device()
    bits, err = b.run()
    assert err == 0
    holds(b, bits)


def test_consecutive_positions_of_different_sequences():
    b = Batch(30, [([40, 41, 42, 43, 44], 2), ([16, 17, 18], 0), ([1, 2, 3, 4], 1), ([0, 1, 2], 3)], 32, 8)
    # Row 2's list like row 1's from its third own page on, and row 4's like row 3's but for the prefix's successor.
    b.table[2, 4:] = b.table[1, 4:]
    swap = [p for p in range(b.pages) if p not in b.table][0]
    b.k[swap], b.v[swap] = b.k[int(b.table[3, 2])] * 2, b.v[int(b.table[3, 2])] + 1
    b.table[4] = b.table[3]
    b.table[4, 2] = swap
    for r in (1, 3):  # the slots of the later rows' last positions
        page = int(b.table[r, 4])
        b.k[page, 8:13] = b.k[page, :5]
        b.v[page, 8:13] = b.v[page, :5]
    bits, err = b.device().run()
    assert err == 0
    holds(b, bits)


@pytest.mark.parametrize("heads", [(32, 8), (8, 8)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_a_later_rows_nonfinite_slot_does_not_reach_the_earlier_rows(bad, which, heads):
    b = Batch(31, [([37], 2)], *heads, per=6)  # positions 63..68
    page = int(b.table[0, 66 // 16])
    (b.k if which == "k" else b.v)[page, 66 % 16, :, 11] = bad
    bits, err = b.device().run()
    assert err == NONFINITE
    holds(b, bits, [0, 1, 2])
    got = values(bits, b)
    # An infinite key against a negative query component has the score -inf, the weight 0 and a finite row.
    hit = b.q[3:, :, 11] > 0 if which == "k" and bad == float("inf") else torch.ones(3, heads[0], dtype=torch.bool)
    assert not torch.isfinite(got[3:, :, 11])[hit].any()


def test_a_later_row_whose_own_key_scores_minus_infinity_is_reported():
    b = Batch(33, [([37], 2)], 8, 8, per=6)
    b.q[3:, :, 11] = -1
    b.k[int(b.table[0, 66 // 16]), 66 % 16, :, 11] = float("inf")
    bits, err = b.device().run()
    assert err == NONFINITE
    holds(b, bits, [0, 1, 2])


def test_a_run_with_a_position_or_page_out_of_range_in_its_midst():
    b = Batch(32, [([50], 2)], 32, 8, per=8).device()
    b.d["pos"][3] = b.context
    bits, err = b.run()
    assert err == POSITION
    holds(b, bits, [0, 1, 2, 4, 5, 6, 7])
    b = Batch(32, [([50], 2)], 32, 8, per=8)  # lengths 75..82: the last two rows begin page 5
    b.table[7, 5] = b.pages
    bits, err = b.device().run()
    assert err == PAGE
    holds(b, bits, range(7))


@pytest.mark.parametrize("heads", [(32, 8), (16, 8), (8, 8), (64, 8)])
@pytest.mark.parametrize("longest", [1, 127, 128, 129, 300, 520])
def test_many_rows_with_short_and_longer_own_keys(longest, heads):
    """Own keys around the steps of both forms of workgroup, and a context that bounds them and one that does not."""
    owns = [longest - (i * 7) % longest for i in range(66)]
    b = Batch(longest, [(owns, 5), ([longest, 1], 7)], *heads, extra_stride=40).device()
    for context in (int(b.lengths.max()), b.context):
        bits, err = b.run(context=context)
        assert err == 0
        holds(b, bits)


def test_sixty_four_groups_of_one_row_and_empty_ones():
    b = Batch(1, [([1 + i % 40], 1 + i % 3) for i in range(64)], 16, 8).device()
    bits, err = b.run()
    assert err == 0
    holds(b, bits)
    b = Batch(2, [([4, 50], 0), ([3], 2), ([700], 0)], 32, 8, list_empty=True).device()
    assert len(b.groups) == 3
    bits, err = b.run()
    assert err == 0
    holds(b, bits)


def test_no_groups_is_ordinary_attention():
    b = Batch(3, [([900, 1, 17, 512], 0)], 32, 8).device()
    bits, err = b.run()
    assert err == 0
    holds(b, bits)


def test_long_units_and_long_chunks():
    """Sizes at which one workgroup walks more pages than it holds table entries for at once: 40 rows over the same
    8300 keys without a group (own keys of 33 steps), and 1024 rows of a group (prefix chunks of 17 tiles)."""
    b = Batch(20, [([8300], 0)], 32, 8)
    b.table, b.lengths, b.rows = np.repeat(b.table, 40, 0), np.repeat(b.lengths, 40), 40
    b.lengths[1::2] -= 1 + np.arange(20)
    b.q = torch.randn(40, 32, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    bits, err = b.device().run()
    assert err == 0
    holds(b, bits, [0, 1, 20, 39])
    b = Batch(21, [([1 + i % 5 for i in range(1024)], 132)], 32, 8).device()
    bits, err = b.run()
    assert err == 0
    holds(b, bits, [0, 1, 33, 500, 1023])


def test_groups_change_the_order_of_sums_only():
    """The same rows with their shared prefix given whole, in part, and not at all."""
    b = Batch(4, [([40, 3, 77, 1, 250], 30)], 32, 8).device()
    for groups in ([(0, 5, 30)], [(0, 5, 7)], [(0, 2, 30), (2, 3, 30)], [(1, 3, 29)], []):
        bits, err = b.run(groups=groups)
        assert err == 0
        holds(b, bits)


@pytest.mark.parametrize("rows", [5, 40])
def test_tiled_output_is_the_same_in_the_projections_order(rows):
    b = Batch(5, [([9 + i for i in range(rows - 1)], 12), ([3], 0)], 32, 8).device()
    plain, _ = b.run()
    tiled, err = b.run(tiled=1)
    assert err == 0
    m = int(LIB.fh_activation_rows(rows))
    t = tiled.reshape(4096 // 32, m // 16, 4, 16, 8).transpose(1, 3, 0, 2, 4).reshape(m, 4096)
    assert np.array_equal(t[:rows], plain.reshape(rows, 4096)) and np.all(t[rows:] == 0x1357)


def test_repeated_calls_give_the_same_bits_and_any_larger_context_serves():
    b = Batch(6, [([100, 600, 1], 70)], 32, 8, extra_stride=200).device()
    first, _ = b.run(context=int(b.lengths.max()))
    again, _ = b.run(context=int(b.lengths.max()))
    assert np.array_equal(first, again)
    wide, err = b.run()  # a capacity of 200 pages more
    assert err == 0
    holds(b, wide)


def test_sharp_and_flat_softmaxes():
    for sharp in (0.0, 0.1, 20.0):
        b = Batch(7, [([40, 600], 40)], 32, 8, sharp=sharp).device()
        bits, err = b.run()
        assert err == 0
        holds(b, bits)


def test_pages_beyond_32_bits_of_offset():
    b = Batch(8, [([3, 40], 4)], 32, 8)
    pages = 270_000  # 4.4e9 elements a cache
    far = b.table.copy()
    used = sorted({int(p) for row in b.table for p in row if p != 0xFFFFFFFF})
    to = {p: pages - 1 - i for i, p in enumerate(used)}
    for p, t in to.items():
        far[b.table == p] = t
    b.device()
    k = torch.empty(pages, 16, 8, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    for p, t in to.items():
        k[t], v[t] = b.d["k"][p], b.d["v"][p]
    b.d.update(k=k, v=v, table=du.to_dev(far))
    b.pages = pages
    bits, err = b.run()
    assert err == 0
    holds(b, bits)


# ---- what the error word reports ----------------------------------------------

POSITION, PAGE, NONFINITE = 4, 8, 1


def test_a_row_whose_prefix_is_not_all_visible_is_reported_and_left():
    b = Batch(9, [([20, 0, 5], 4), ([8], 0)], 32, 8)
    b.lengths[1] = 4 * 16 - 1  # one token short
    bits, err = b.device().run()
    assert err == POSITION
    holds(b, bits, [0, 2, 3])
    assert np.all(bits.reshape(4, -1)[1] == 0x1357)


def test_positions_beyond_the_context_are_reported_and_left():
    b = Batch(10, [([20, 3], 4), ([8], 0)], 32, 8).device()
    pos = (b.lengths - 1).astype(np.uint32)
    pos[2] = 0xFFFFFFFF
    pos[0] = b.context
    b.d["pos"] = du.to_dev(pos)
    bits, err = b.run()
    assert err == POSITION
    holds(b, bits, [1])
    assert np.all(bits.reshape(3, -1)[[0, 2]] == 0x1357)


@pytest.mark.parametrize("row,entry", [(0, 1), (0, 4), (2, 0)])
def test_pages_outside_the_pool_are_reported(row, entry):
    b = Batch(11, [([20, 3], 4), ([8], 0)], 32, 8)
    page = b.table[row, entry]
    b.table[(b.table == page)] = b.pages + 7
    bits, err = b.device().run()
    assert err & PAGE


def test_tables_that_do_not_share_the_prefix_are_reported():
    b = Batch(12, [([20, 3, 9], 40)], 32, 8)
    b.table[2, 39] = b.table[2, 38]
    bits, err = b.device().run()
    assert err == PAGE


@pytest.mark.parametrize("where", ["prefix key", "own value", "query"])
@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf")])
def test_nonfinite_inputs_are_reported_and_stay_in_their_rows(where, bad):
    b = Batch(13, [([20, 3], 4), ([8], 0)], 32, 8)
    if where == "prefix key":
        b.k[int(b.table[0, 2]), 3, 5, 7] = bad
    elif where == "own value":
        b.v[int(b.table[0, 4]), 3, 5, 7] = bad
    else:
        b.q[0, 9, 100] = bad
    bits, err = b.device().run()
    assert err == NONFINITE
    holds(b, bits, [2] if where == "prefix key" else [1, 2])


# ---- streams, graphs, calls at once ---------------------------------------------

def test_two_streams_at_once_with_a_scratch_each():
    a = Batch(14, [([200, 30, 5, 9], 100)], 32, 8).device()
    b = Batch(15, [([50] * 20, 30), ([1], 0)], 16, 8).device()
    want = [x.run()[0] for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = []
    for x, s in zip((a, b), streams):
        g = x.group_array()
        buf, n = x.scratch()
        out, err = du.empty(x.rows * x.qh * 128, np.uint16), du.empty(1, np.uint32)
        work.append((x, s, g, buf, n, out, err))
    torch.cuda.synchronize()
    for _ in range(5):
        for x, s, g, buf, n, out, err in work:
            _lib.check(LIB.fh_op_prefix_attention(
                x.d["q"].data_ptr(), x.d["k"].data_ptr(), x.d["v"].data_ptr(), du.ptr(x.d["pos"]), du.ptr(x.d["table"]),
                g.ctypes.data, len(g), du.ptr(out), 0, du.ptr(buf), n, x.rows, x.qh, x.kvh, x.stride, x.pages, x.context,
                du.ptr(err), s.cuda_stream))
    torch.cuda.synchronize()
    for w, (x, s, g, buf, n, out, err) in zip(want, work):
        assert np.array_equal(du.to_host(out, np.uint16), w) and int(du.to_host(err, np.uint32)[0]) == 0


def test_a_captured_call_follows_its_positions_and_tables():
    """Replayed with other positions (a decode step later) and another page order; eager calls between the replays."""
    b = Batch(16, [([40, 17, 33], 20), ([9], 0)], 32, 8).device()
    g = b.group_array()
    buf, n = b.scratch()
    out, err = du.empty(b.rows * b.qh * 128, np.uint16), du.empty(1, np.uint32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _lib.check(LIB.fh_op_prefix_attention(
            b.d["q"].data_ptr(), b.d["k"].data_ptr(), b.d["v"].data_ptr(), du.ptr(b.d["pos"]), du.ptr(b.d["table"]),
            g.ctypes.data, len(g), du.ptr(out), 0, du.ptr(buf), n, b.rows, b.qh, b.kvh, b.stride, b.pages, b.context,
            du.ptr(err), du.stream()))
    g[:] = 7  # the groups are the caller's again after the call
    for step in range(4):
        if step:
            b.lengths = np.maximum(b.lengths - 3, [321, 321, 321, 1])
            b.d["pos"].copy_(du.to_dev((b.lengths - 1).astype(np.uint32)))
            b.d["q"].copy_(b.d["q"].flip(0))
            b.q = b.d["q"].cpu()
        graph.replay()
        torch.cuda.synchronize()
        got = du.to_host(out, np.uint16)
        holds(b, got)
        eager, e = b.run()
        assert np.array_equal(got, eager) and e == 0 and int(du.to_host(err, np.uint32)[0]) == 0


# ---- the operators together --------------------------------------------------------

def test_fork_then_shared_attention_then_a_4_bit_projection():
    """A prompt is forked (its last page copied), every fork attends to the shared pages, and the attention's
    tile-ordered output is the 4-bit output projection's operand."""
    r = np.random.default_rng(17)
    b = Batch(17, [([5, 5, 5], 9)], 32, 8).device()
    # Rows 1 and 2 are forks of row 0: their own page is a copy of the five slots, then one token of their own.
    src = int(b.table[0, 9])
    moves = np.array([[src, int(b.table[i, 9]), 4] for i in (1, 2)], np.uint32)
    for cache in ("k", "v"):
        _lib.check(LIB.fh_op_kv_copy_pages(b.d[cache].data_ptr(), 1, 0, moves.ctypes.data, 2, 8, b.pages, du.stream()))
        torch.cuda.synchronize()
        setattr(b, cache, b.d[cache].cpu())
        assert torch.equal(getattr(b, cache)[int(b.table[1, 9]), :4], getattr(b, cache)[src, :4])
    tiled, err = b.run(tiled=1)
    assert err == 0
    plain = tiled.reshape(128, 2, 4, 16, 8).transpose(1, 3, 0, 2, 4).reshape(32, 4096)[:3]
    holds(b, np.ascontiguousarray(plain).reshape(-1))
    n, k, group = 64, 4096, 128
    w = r.standard_normal((n, k)).astype(np.float32) * 0.02
    src = du.to_dev((torch.from_numpy(w).bfloat16().view(torch.int16).numpy()).view(np.uint16).reshape(-1))
    packed = torch.zeros(n * k // 2, dtype=torch.uint8, device="cuda")
    scales, st = du.empty(n * k // group, np.uint16), du.empty(n * k // group, np.uint16)
    wt = torch.zeros(n * k // 8, dtype=torch.int32, device="cuda")
    _lib.check(LIB.fh_op_quantize_w4(du.ptr(src), du.ptr(packed), du.ptr(scales), n, k, group, None, du.stream()))
    _lib.check(LIB.fh_op_tile_weight_w4(du.ptr(packed), du.ptr(scales), None, du.ptr(wt), du.ptr(st), None, n, k, group, 0,
                                        du.stream()))
    y = torch.zeros(3, n, device="cuda")
    x = du.to_dev(tiled)
    _lib.check(LIB.fh_op_gemm_w4(du.ptr(x), du.ptr(wt), du.ptr(st), None, 3, n, k, group, 3, 1, None, du.ptr(y), n, None,
                                 du.stream()))
    p = packed.cpu().numpy().reshape(n, k // 2)
    q = np.stack([p & 15, p >> 4], -1).reshape(n, k // group, group).astype(np.float64) - 8
    s = (du.to_host(scales, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(n, -1, 1)
    a = (np.ascontiguousarray(plain).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    want = a @ (q * s).reshape(n, k).T
    # The products' FP32 error, 1e-5 of the result's norm if independent, and the weight's rounding to 4 bits.
    assert np.linalg.norm(y.cpu().numpy() - want) <= 2e-5 * np.linalg.norm(want)
    assert np.all(np.abs((q * s).reshape(n, k) - w) <= np.repeat(s[..., 0], group, 1) * 0.52 + 2.0 ** -8 * np.abs(w))


# ---- long prefixes: chunks of many tiles, blocks of 128 vectors, streamed loads -----

class Long(Batch):
    """The formula on the device, and values that mark the keys: with queries of zero every key has the same weight,
    and key t is 1 in one (KV head, dim) of 1024 and 0 elsewhere, so a key more or less changes an output by one part
    in about n / 1024."""

    def exact(self, rows=None):
        g = self.qh // self.kvh
        want = torch.zeros(self.rows, self.qh, 128, dtype=torch.float64)
        tol = torch.zeros_like(want)
        for r in range(self.rows) if rows is None else rows:
            n = int(self.lengths[r])
            idx = torch.from_numpy(self.table[r, :-(-n // 16)].astype(np.int64)).cuda()
            k = self.d["k"][idx].view(-1, self.kvh, 128)[:n].double().permute(1, 2, 0).contiguous()  # [kvh][128][n]
            v = self.d["v"][idx].view(-1, self.kvh, 128)[:n].double().permute(1, 0, 2).contiguous()
            q = self.d["q"][r].double().view(self.kvh, g, 128)
            s = torch.matmul(q, k) / math.sqrt(128)
            most = torch.matmul(q.abs(), k.abs()).amax((1, 2)).view(-1, 1, 1) / math.sqrt(128)
            w = torch.softmax(s, -1)
            want[r] = torch.matmul(w, v).view(self.qh, 128).cpu()
            d = 128 * 2.0 ** -24 * most + 2.0 ** -22 + 2.0 ** -23 * s.abs().amax()
            tol[r] = (torch.matmul(w, v.abs()) * (2 * d + 2.0 ** -16 + n * 2.0 ** -24)).view(self.qh, 128).cpu()
        return want, tol + 2.0 ** -8 * (want.abs() + tol)

    def mark(self):
        assert self.kvh == 8
        self.d["q"].zero_()
        ones = torch.eye(1024, dtype=torch.bfloat16, device="cuda").view(1024, 8, 128)
        for r in range(self.rows):
            t = torch.arange(int(self.lengths[r]), device="cuda")
            page = torch.from_numpy(self.table[r].astype(np.int64)).cuda()[t // 16]
            self.d["v"][page, t % 16] = ones[t % 1024]

    def marked(self):
        """(output, tolerance) of the marked values: keys of a bin over all keys; the scores are 0 exactly."""
        n = torch.from_numpy(self.lengths.astype(np.float64)).view(-1, 1, 1)
        bins = torch.arange(1024, dtype=torch.float64).view(1, 8, 128)
        want = (torch.floor((n - 1 - bins) / 1024) + 1) / n
        want = want.repeat_interleave(self.qh // self.kvh, 1)
        tol = want * (2.0 ** -21 + 2.0 ** -16 + n * 2.0 ** -24)
        return want, tol + 2.0 ** -8 * (want + tol)


@pytest.mark.parametrize("heads", [(8, 8), (16, 8), (32, 8), (64, 8)])
@pytest.mark.parametrize("vectors", [16, 40, 64, 72, 128, 136])
@pytest.mark.parametrize("pages", [1030, 1541])
def test_long_prefixes(heads, vectors, pages):
    """One and several blocks of 16, 64 and 128 vectors, part of them filled; the longer prefix is streamed where one
    block holds the rows."""
    rows = vectors // (heads[0] // heads[1])
    groups = [([i * 5 % 23 for i in range(rows)], pages)] + ([([5, 1], 2), ([9], 0)] if vectors == 40 else [])
    b = Long(vectors + pages, groups, *heads).device()
    bits, err = b.run()
    assert err == 0
    holds(b, bits, sorted({0, rows // 2, rows - 1, b.rows - 1}))
    again, _ = b.run()
    assert np.array_equal(bits, again)
    b.mark()
    bits, err = b.run()
    assert err == 0
    want, tol = b.marked()
    off = (values(bits, b) - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    # One key less would be seen: the largest bin's output falls by more than twice its tolerance.
    n = int(b.lengths[0])
    assert (1 / n) > 2 * float(tol[0].max())

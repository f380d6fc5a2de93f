"""Shared-prefix attention on any host: what the entry points refuse before
any launch, and the scratch they ask for. No GPU calls are made here (the
pointers are no memory)."""

import ctypes

import numpy as np
import pytest

import ferric_amd
from ferric_amd import _lib

LIB = ferric_amd.load()
P = 4096  # an aligned address that is never read


def groups_of(*g):
    return np.array(g, np.uint32).reshape(-1, 3)


def call(groups=groups_of((0, 4, 2)), q=P, k=P, v=P, pos=P, table=P, out=P, scratch=P, nbytes=1 << 40, rows=4, qh=32,
         kvh=8, stride=8, pages=64, context=128, null=False, count=None):
    count = len(groups) if count is None else count
    return LIB.fh_op_prefix_attention(q, k, v, pos, table, None if null else groups.ctypes.data, count, out, 0, scratch,
                                      nbytes, rows, qh, kvh, stride, pages, context, None, None)


BAD_GROUPS = [groups_of((0, 0, 1)), groups_of((0, 5, 1)), groups_of((4, 1, 1)), groups_of((2, 2, 1), (0, 2, 1)),
              groups_of((0, 3, 1), (2, 2, 1)), groups_of((0, 4, 9)), groups_of((2**32 - 1, 2, 1)),
              groups_of((0, 1, 2**28))]


@pytest.mark.parametrize("groups", BAD_GROUPS)
def test_groups_that_are_refused(groups):
    assert call(groups) == 1
    assert b"prefix groups" in LIB.fh_last_error(None)
    assert LIB.fh_prefix_attention_scratch_bytes(groups.ctypes.data, len(groups), 4, 32, 8, 128) == 0


def test_more_groups_than_a_launch_holds_are_refused():
    many = np.array([(i, 1, 1) for i in range(65)], np.uint32)
    assert call(many, rows=65) == 1
    assert call(null=True, count=1) == 1


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(table=None), dict(out=None),
                                 dict(scratch=None), dict(rows=0, groups=groups_of()), dict(rows=65536), dict(context=2**24 + 16, stride=2**21), dict(qh=31),
                                 dict(qh=24), dict(qh=128), dict(kvh=0), dict(stride=7), dict(stride=0), dict(pages=0),
                                 dict(context=0, groups=groups_of()), dict(q=P + 8), dict(k=P + 8), dict(v=P + 8),
                                 dict(out=P + 4), dict(scratch=P + 4), dict(nbytes=100)])
def test_shapes_and_pointers_that_are_refused(bad):
    assert call(**bad) == 1


def test_scratch_is_asked_for_and_checked():
    g = groups_of((0, 4, 8))
    n = LIB.fh_prefix_attention_scratch_bytes(g.ctypes.data, 1, 4, 32, 8, 128)
    assert n > 0 and call(g, nbytes=n - 1) == 1
    assert LIB.fh_prefix_attention_scratch_bytes(None, 0, 4, 32, 8, 128) > 0
    for rows, qh, kvh, context in [(0, 32, 8, 128), (65535, 65, 65, 128), (65536, 8, 8, 128), (4, 31, 8, 128), (4, 32, 0, 128), (4, 32, 8, 0)]:
        assert LIB.fh_prefix_attention_scratch_bytes(None, 0, rows, qh, kvh, context) == 0
    assert ctypes.sizeof(_lib.PrefixGroup) == 12


@pytest.mark.parametrize("rows,qh,kvh", [(65535, 128, 16), (65535, 512, 64), (1024, 32768, 4096), (1, 4096, 4096)])
def test_scratch_of_the_largest_batches(rows, qh, kvh):
    g = groups_of((0, rows, 1 << 20))
    n = LIB.fh_prefix_attention_scratch_bytes(g.ctypes.data, 1, rows, qh, kvh, 1 << 24)
    assert n >= rows * qh * 132 * 4  # a record a query head at least

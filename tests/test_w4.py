"""4-bit projections on any host: what the entry points refuse before any
launch. No GPU calls are made here (the pointers are no memory)."""

import importlib.util
import itertools
import random
from pathlib import Path

import pytest

import ferric_amd

LIB = ferric_amd.load()
P = 4096  # an aligned address that is never read


def gemm(x=P, w=P, s=P, z=None, m=1, n=32, k=256, group=64, epi=0, splits=1, residual=None, out=P, ldo=32):
    return LIB.fh_op_gemm_w4(x, w, s, z, m, n, k, group, epi, splits, residual, out, ldo, None, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(w=None), dict(s=None), dict(out=None), dict(m=0), dict(m=33), dict(k=(1 << 24) + 128), dict(n=2**31, k=128, ldo=2**31), dict(n=0),
                                 dict(n=24), dict(k=0), dict(k=192), dict(group=16), dict(group=256), dict(group=0),
                                 dict(epi=5), dict(splits=0), dict(splits=2), dict(epi=4, splits=3), dict(epi=1), dict(ldo=31),
                                 dict(epi=2, n=16), dict(x=P + 8), dict(w=P + 8), dict(s=P + 4), dict(z=P + 2),
                                 dict(epi=4, splits=65536, k=128 * 65536)])
def test_gemm_refusals(bad):
    assert gemm(**bad) == 1


@pytest.mark.parametrize("bad", [dict(n=0), dict(k=64), dict(k=0), dict(group=48), dict(src=None), dict(packed=None),
                                 dict(scales=None), dict(src=P + 2), dict(packed=P + 1), dict(n=2**28, k=128)])
def test_quantize_refusals(bad):
    a = dict(src=P, packed=P, scales=P, n=16, k=128, group=32) | bad
    assert LIB.fh_op_quantize_w4(a["src"], a["packed"], a["scales"], a["n"], a["k"], a["group"], None, None) == 1


@pytest.mark.parametrize("bad", [dict(n=8), dict(k=64), dict(group=96), dict(packed=None), dict(scales=None), dict(w=None),
                                 dict(st=None), dict(z=P, zt=None), dict(part=3), dict(packed=P + 2), dict(w=P + 8),
                                 dict(n=2**28, k=128)])
def test_tile_refusals(bad):
    a = dict(packed=P, scales=P, z=None, w=P, st=P, zt=None, n=16, k=128, group=32, part=0) | bad
    assert LIB.fh_op_tile_weight_w4(a["packed"], a["scales"], a["z"], a["w"], a["st"], a["zt"], a["n"], a["k"], a["group"],
                                    a["part"], None) == 1


def test_default_splits_fill_the_gpu_and_fit_the_width():
    for n, k in itertools.product([16, 32, 48, 1024, 4096, 6144, 24576, 151936], [128, 256, 1024, 4096, 12288]):
        s = LIB.fh_gemm_w4_default_splits(n, k)
        assert 1 <= s <= max(1, k // 128)
    assert LIB.fh_gemm_w4_default_splits(4096, 4096) == 2
    assert LIB.fh_gemm_w4_default_splits(24576, 4096) == 1
    assert LIB.fh_gemm_w4_default_splits(0, 4096) == 1


def test_measured_swiglu_cases_have_whole_blocks_of_output_columns():
    """Their outputs are the next projection's operand, whose buffers are cut to blocks of 32 columns."""
    spec = importlib.util.spec_from_file_location("operators", Path(__file__).resolve().parents[1] / "perf" / "operators.py")
    operators = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(operators)
    cases = operators.listed() + [operators.draw(random.Random(s)) for s in range(4000)]
    wide = [c for c in cases if c.get("epilogue") == "swiglu"]
    assert len(wide) > 100
    assert all(c["n"] % 64 == 0 for c in wide)

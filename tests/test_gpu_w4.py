"""4-bit projections on the GPU against the formula in 64 bits.

Two kinds of inputs. Small whole activations and scales that are powers of two
make every product and sum exact in FP32 (a group's sum of (16 + q) x stays
below 31 * 128 * 8 < 2^15, an output below 2^24 steps of its last place), so
the outputs have to be equal to the bit, whatever the order of the sums. Random
ones are held to the roundings: FP32 sums of a group pass through partial sums
of at most |sum (16 + q) x| over a run of its columns, at most one rounding of
2^-24 of that per column and as many for the part taken off, then one per
group; bf16 outputs add half a step, 2^-8 of the value."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tests import devutil as du  # noqa: E402
import ferric_amd  # noqa: E402
from ferric_amd import _lib  # noqa: E402
from oracle import oracle as orc  # noqa: E402

LIB = ferric_amd.load()
BF16, RESIDUAL, SWIGLU, F32, PARTIAL = range(5)


def widen(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def narrow(x):
    """float64 to bf16 bits, one rounding (through FP32 only where that is exact)."""
    x = np.asarray(x, np.float64)
    f = x.astype(np.float32)
    # Nearest FP32 with the sticky bit of what was lost: rounding it again is the one rounding to bf16.
    b = f.view(np.uint32).copy()
    off = np.abs(f.astype(np.float64)) > np.abs(x)
    b[off] -= 1
    b[(f.astype(np.float64) != x)] |= 1
    return orc.f32_to_bf16(b.view(np.float32).reshape(-1)).reshape(x.shape)


class Weight:
    """Quantized values, scales and zero points on the host, and tiled on the device."""

    def __init__(self, r, n, k, group, zeros, scales=None, half=False):
        self.n, self.k, self.group = n, k, group
        self.q = r.integers(0, 16, (n, k), dtype=np.uint8)
        self.s = orc.f32_to_bf16((2.0 ** r.integers(-3, 4, n * (k // group))).astype(np.float32)) if scales is None else scales
        self.s = self.s.reshape(n, k // group)
        self.z = r.integers(0, 16, (n, k // group), dtype=np.uint8) if zeros else None
        packed = self.q[:, 0::2] | (self.q[:, 1::2] << 4)
        rows = 2 * n if half else n
        d = dict(p=torch.from_numpy(packed.copy()).cuda(), s=du.to_dev(self.s))
        d["z"] = torch.from_numpy(self.z).cuda() if zeros else None
        self.dev = d
        self.wt = torch.zeros(rows * k // 8, dtype=torch.int32, device="cuda")
        self.st = torch.zeros(rows * (k // group), dtype=torch.int16, device="cuda")
        self.zt = torch.zeros(rows * (k // group), dtype=torch.uint8, device="cuda") if zeros else None
        if not half:
            self.tile(self, 0)

    def tile(self, into, part):
        _lib.check(LIB.fh_op_tile_weight_w4(du.ptr(self.dev["p"]), du.ptr(self.dev["s"]), du.ptr(self.dev["z"]),
                                            du.ptr(into.wt), du.ptr(into.st), du.ptr(into.zt), self.n, self.k, self.group,
                                            part, du.stream()))

    def exact(self):
        z = self.z.astype(np.float64) if self.z is not None else np.full(self.s.shape, 8.0)
        rep = lambda a: np.repeat(a, self.group, 1)  # noqa: E731
        return rep(widen(self.s)) * (self.q.astype(np.float64) - rep(z))

    def off(self, x):
        """The bound on the FP32 error of x W^T (see above), x in 64 bits [m][k]."""
        m, groups = x.shape[0], self.k // self.group
        xg = x.reshape(m, groups, self.group)
        zero = 16 + (self.z.astype(np.float64) if self.z is not None else 8.0)
        runs = np.abs(np.cumsum(xg, 2)).max(2)  # [m][groups]
        most = 2 * (31 + np.max(zero)) * runs + 16 * np.abs(xg).max(2) * np.sqrt(self.group)
        return (2.0 ** -24) * (2 * self.group + 40) * (most @ np.abs(widen(self.s)).T)


def activations(r, m, k, whole, junk=True):
    """Row-major bits, and the tile order with rows past m full of NaN."""
    x = r.integers(-8, 9, (m, k)).astype(np.float32) if whole else r.standard_normal((m, k)).astype(np.float32)
    bits = orc.f32_to_bf16(x.reshape(-1)).reshape(m, k)
    full = np.full((32, k), 0x7FC0 if junk else 0, np.uint16)
    full[:m] = bits
    return bits, du.to_dev(np.ascontiguousarray(full.reshape(2, 16, k // 32, 4, 8).transpose(2, 0, 3, 1, 4)).reshape(-1))


def call(xt, w, m, n, epi, out, ldo, splits=1, residual=None, err=None, stream=None):
    _lib.check(LIB.fh_op_gemm_w4(du.ptr(xt), du.ptr(w.wt), du.ptr(w.st), du.ptr(w.zt), m, n, w.k, w.group, epi, splits,
                                 du.ptr(residual), du.ptr(out), ldo, du.ptr(err), stream or du.stream()))


SHAPES = [(16, 128), (32, 256), (48, 384), (1040, 128), (4096, 1024), (64, 12288), (8192, 512), (16, 4096 + 128)]


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("m", [1, 2, 8, 15, 16, 17, 32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_whole_numbers_are_exact(n, k, m, group):
    r = np.random.default_rng(n + k + m + group)
    w = Weight(r, n, k, group, zeros=(n + m) % 2 == 1 or m == 8)
    x, xt = activations(r, m, k, whole=True)
    want = widen(x) @ w.exact().T
    ldo = n + 5
    out = torch.full(((m + 1) * ldo,), 7.5, dtype=torch.float32, device="cuda")
    call(xt, w, m, n, F32, out, ldo)
    got = du.to_host(out, np.float32).reshape(m + 1, ldo)
    assert np.array_equal(got[:m, :n], want)
    assert np.all(got[:m, n:] == 7.5) and np.all(got[m] == 7.5)  # nothing else is written
    out = du.to_dev(np.full((m + 1) * n, 0x1234, np.uint16))
    call(xt, w, m, n, BF16, out, n)
    got = du.to_host(out, np.uint16).reshape(m + 1, n)
    assert np.array_equal(got[:m], narrow(want)) and np.all(got[m] == 0x1234)


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("m", [1, 20])
def test_split_slabs_add_up_exactly(splits, m):
    r = np.random.default_rng(splits)
    n, k = 96, 1024
    w = Weight(r, n, k, 64, True)
    x, xt = activations(r, m, k, whole=True)
    slab = 32 * n
    out = torch.full((splits * slab + n,), 7.5, dtype=torch.float32, device="cuda")
    call(xt, w, m, n, PARTIAL, out, n, splits)
    got = du.to_host(out, np.float32)
    assert np.all(got[splits * slab:] == 7.5)
    slabs = got[:splits * slab].reshape(splits, 32, n)
    assert np.array_equal(slabs[:, :m].astype(np.float64).sum(0), widen(x) @ w.exact().T)
    assert np.all(slabs[:, m:] == 7.5)


@pytest.mark.parametrize("m", [1, 9, 32])
@pytest.mark.parametrize("alias", [False, True])
def test_residual(m, alias):
    r = np.random.default_rng(m)
    n, k = 112, 384
    w = Weight(r, n, k, 128, False)
    x, xt = activations(r, m, k, whole=True)
    res = orc.f32_to_bf16(r.integers(-99, 99, m * n).astype(np.float32))
    dres = du.to_dev(res)
    out = dres if alias else du.empty(m * n, np.uint16)
    call(xt, w, m, n, RESIDUAL, out, n, residual=dres)
    want = widen(x) @ w.exact().T + widen(res).reshape(m, n)
    assert np.array_equal(du.to_host(out, np.uint16).reshape(m, n), narrow(want))


@pytest.mark.parametrize("m", [1, 16, 17, 32])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_random_values_are_within_the_roundings(m, group, zeros):
    r = np.random.default_rng(m + group)
    n, k = 528, 2048
    s = orc.f32_to_bf16((r.random(n * (k // group)) * 0.01 + 1e-3).astype(np.float32))
    w = Weight(r, n, k, group, zeros, scales=s)
    x, xt = activations(r, m, k, whole=False)
    want, off = widen(x) @ w.exact().T, w.off(widen(x))
    out = torch.zeros(m * n, dtype=torch.float32, device="cuda")
    call(xt, w, m, n, F32, out, n)
    got = du.to_host(out, np.float32).reshape(m, n).astype(np.float64)
    assert np.all(np.abs(got - want) <= off)
    # All roundings of a group taken as independent: 2^-25 * 24 / 4.6 * sqrt(128) = 1.8e-6 of the result's norm.
    assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)
    out = du.empty(m * n, np.uint16)
    call(xt, w, m, n, BF16, out, n)
    got = widen(du.to_host(out, np.uint16).reshape(m, n))
    assert np.all(np.abs(got - want) <= off + 2.0 ** -8 * (np.abs(want) + off))


@pytest.mark.parametrize("m", [1, 7, 16, 18, 32])
@pytest.mark.parametrize("zeros", [False, True])
def test_swiglu_of_interleaved_halves_feeds_the_next_projection(m, zeros):
    r = np.random.default_rng(m)
    width, k, group = 256, 512, 64
    scale = lambda a, b: orc.f32_to_bf16((r.random(a * b) * 0.01 + 2e-3).astype(np.float32))  # noqa: E731
    gate = Weight(r, width, k, group, zeros, scales=scale(width, k // group), half=True)
    up = Weight(r, width, k, group, zeros, scales=scale(width, k // group), half=True)
    gate.tile(gate, 1)
    up.tile(gate, 2)
    x, xt = activations(r, m, k, whole=False)
    out, err = du.to_dev(np.full(32 * width, 0x2222, np.uint16)), du.empty(1, np.uint32)
    call(xt, gate, m, 2 * width, SWIGLU, out, width, err=err)
    assert du.to_host(err, np.uint32)[0] == 0
    tiled = du.to_host(out, np.uint16).reshape(width // 32, 2, 4, 16, 8).transpose(1, 3, 0, 2, 4).reshape(32, width)
    assert np.all(tiled[m:] == 0x2222)
    g, u = widen(x) @ gate.exact().T, widen(x) @ up.exact().T
    # Half a step of bf16 for gate, up and the product, the FP32 sums before them; |d silu / dg| <= 1.1.
    dg, du_ = gate.off(widen(x)) + 2.0 ** -8 * np.abs(g), up.off(widen(x)) + 2.0 ** -8 * np.abs(u)
    silu = g / (1 + np.exp(-g))
    want, off = silu * u, 1.1 * dg * (np.abs(u) + du_) + np.abs(silu) * du_
    assert np.all(np.abs(widen(tiled[:m]) - want) <= (off + 2.0 ** -8 * (np.abs(want) + off)) * 1.001 + 1e-30)
    # The tile-ordered output is the next projection's operand as it is.
    down = Weight(r, 48, width, 128, zeros)
    y = torch.zeros(m * 48, dtype=torch.float32, device="cuda")
    call(out, down, m, 48, F32, y, 48)
    a = widen(tiled[:m])
    got = du.to_host(y, np.float32).reshape(m, 48)
    assert np.all(np.abs(got - a @ down.exact().T) <= down.off(a))


def test_swiglu_reports_nonfinite_rows_below_m_only():
    r = np.random.default_rng(0)
    w = Weight(r, 32, 128, 32, False)
    _, xt = activations(r, 3, 128, whole=True)  # rows 3.. are NaN
    out, err = du.empty(32 * 16, np.uint16), du.empty(1, np.uint32)
    # 16 output columns are half a tile column of the next operand: the buffer holds 32 x 32.
    out = du.empty(32 * 32, np.uint16)
    call(xt, w, 3, 32, SWIGLU, out, 16, err=err)
    assert du.to_host(err, np.uint32)[0] == 0
    call(xt, w, 4, 32, SWIGLU, out, 16, err=err)
    assert du.to_host(err, np.uint32)[0] == 1


@pytest.mark.parametrize("width", [16, 48, 80])
@pytest.mark.parametrize("m", [1, 17])
def test_swiglu_of_half_a_block_of_columns_stays_in_its_blocks(width, m):
    """n / 2 an odd multiple of 16: out holds ceil(n / 64) blocks of 32 x 32, nothing behind them or in the last
    block's other columns is written."""
    r = np.random.default_rng(width + m)
    gate = Weight(r, width, 128, 64, True, half=True)
    up = Weight(r, width, 128, 64, True, half=True)
    gate.tile(gate, 1)
    up.tile(gate, 2)
    x, xt = activations(r, m, 128, whole=True)
    blocks = -(-width // 32)
    out = du.to_dev(np.full(1024 * blocks + 1024, 0x2222, np.uint16))
    call(xt, gate, m, 2 * width, SWIGLU, out, width)
    got = du.to_host(out, np.uint16)
    assert np.all(got[1024 * blocks:] == 0x2222)
    tiled = got[:1024 * blocks].reshape(blocks, 2, 4, 16, 8).transpose(1, 3, 0, 2, 4).reshape(32, 32 * blocks)
    assert np.all(tiled[m:] == 0x2222) and np.all(tiled[:, width:] == 0x2222)
    # Exact sums narrowed to bf16; the exponential, a quotient and two products round in FP32, together less than
    # 2^-20, then half a step of bf16 (results below the normal numbers, 2^-126, aside).
    g, u = (widen(narrow(widen(x) @ w.exact().T)) for w in (gate, up))
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-g)) * u
    assert np.all(np.abs(widen(tiled[:m, :width]) - want) <= (2.0 ** -8 + 2.0 ** -20) * np.abs(want) + 1e-30)


def test_extremes_of_weights_and_scales():
    """All weights at the ends, scales at the ends of bf16, zero scales, zero points 0 and 15."""
    r = np.random.default_rng(1)
    n, k, m = 16, 256, 4
    w = Weight(r, n, k, 32, True)
    w.q[:8] = 0
    w.q[8:] = 15
    w.z[:, 0::2] = 0
    w.z[:, 1::2] = 15
    w.s[:] = 0x3F80
    w.s[3] = 0
    w.s[5] = 0x0080  # the smallest normal number
    packed = w.q[:, 0::2] | (w.q[:, 1::2] << 4)
    w.dev = dict(p=torch.from_numpy(packed.copy()).cuda(), s=du.to_dev(w.s), z=torch.from_numpy(w.z).cuda())
    w.tile(w, 0)
    x, xt = activations(r, m, k, whole=True)
    out = torch.zeros(m * n, dtype=torch.float32, device="cuda")
    call(xt, w, m, n, F32, out, n)
    assert np.array_equal(du.to_host(out, np.float32).reshape(m, n), widen(x) @ w.exact().T)


@pytest.mark.parametrize("n,k,group", [(1, 128, 32), (3, 256, 64), (33, 1152, 128), (1000, 384, 32)])
def test_quantize_is_the_stated_rounding(n, k, group):
    r = np.random.default_rng(n)
    x = r.standard_normal((n, k)).astype(np.float32) * 0.02
    x[0, :group] = 0  # a group of zeros
    if n > 1:
        x[1, :group] = 1e-39  # below the smallest normal number
        x[-1, -group:] = r.integers(-7, 8, group)  # ties and ends
    bits = orc.f32_to_bf16(x.reshape(-1))
    w = widen(bits).astype(np.float32).reshape(n, k // group, group)
    packed, scales = torch.zeros(n * k // 2 + 4, dtype=torch.uint8, device="cuda"), du.empty(n * (k // group) + 1, np.uint16)
    err = du.empty(1, np.uint32)
    src = du.to_dev(bits)
    _lib.check(LIB.fh_op_quantize_w4(du.ptr(src), du.ptr(packed), du.ptr(scales), n, k, group, du.ptr(err), du.stream()))
    s = orc.f32_to_bf16((np.abs(w).max(2) / np.float32(7)).reshape(-1))
    got = du.to_host(scales, np.uint16)
    assert np.array_equal(got[:-1], s) and got[-1] == 0 and du.to_host(err, np.uint32)[0] == 0
    f = widen(s).astype(np.float32).reshape(n, -1, 1)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(f > 0, np.clip(np.rint(w / f), -8, 7), 0).astype(np.int64) + 8
    q = q.reshape(n, k).astype(np.uint8)
    p = packed.cpu().numpy()
    assert np.array_equal(p[:n * k // 2].reshape(n, k // 2), q[:, 0::2] | (q[:, 1::2] << 4)) and not p[n * k // 2:].any()


def test_quantize_reports_nonfinite_weights():
    for bad in (0x7F80, 0xFF80, 0x7FC0):
        bits = np.full(128, 0x3F80, np.uint16)
        bits[77] = bad
        src, err = du.to_dev(bits), du.empty(1, np.uint32)
        packed, scales = torch.zeros(64, dtype=torch.uint8, device="cuda"), du.empty(2, np.uint16)
        _lib.check(LIB.fh_op_quantize_w4(du.ptr(src), du.ptr(packed), du.ptr(scales), 1, 128, 64, du.ptr(err), du.stream()))
        assert du.to_host(err, np.uint32)[0] == 1


def test_two_streams_and_a_replayed_graph():
    r = np.random.default_rng(8)
    n, k, m = 2048, 1024, 5
    w = Weight(r, n, k, 128, True)
    x, xt = activations(r, m, k, whole=True)
    want = (widen(x) @ w.exact().T).astype(np.float32)
    outs = [torch.zeros(m * n, dtype=torch.float32, device="cuda") for _ in range(3)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for s, o in zip(streams, outs):
        call(xt, w, m, n, F32, o, n, stream=s.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(xt, w, m, n, F32, outs[2], n)
    for _ in range(3):
        outs[2].fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert np.array_equal(du.to_host(o, np.float32).reshape(m, n), want)


# ---- every form of workgroup -------------------------------------------------------

def on_device(w):
    """W in 64 bits on the device, [n][k]."""
    rep = lambda a: a.repeat_interleave(w.group, 1)  # noqa: E731
    s = torch.from_numpy(widen(w.s)).cuda()
    z = torch.from_numpy(w.z).cuda().double() if w.z is not None else torch.full_like(s, 8.0)
    return rep(s) * (torch.from_numpy(w.q).cuda().double() - rep(z))


def product(x, w):
    return (torch.from_numpy(widen(x)).cuda() @ on_device(w).t()).cpu().numpy()


# Both sides of the sizes from which workgroups have 2 and 4 weight tiles and 4 waves instead of 16, an odd number of
# 32-column pairs, and widths whose blocks of 128 columns the waves take in several turns, the last one short.
FORMS = [(8192, 4224, (1, 8, 16, 17, 32)), (8208, 1152, (1, 16, 17, 32)), (16368, 1152, (2, 18)),
         (16384, 1152, (1, 8, 9, 16, 17, 32)), (16416, 1152, (8, 9, 17, 32)), (65536, 640, (1, 8, 9, 32)),
         (65568, 640, (1, 9, 32)), (4096, 6528, (16, 17, 32))]


@pytest.mark.parametrize("n,k,rows", FORMS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_every_form_is_exact_on_whole_numbers(n, k, rows, group, zeros):
    r = np.random.default_rng(n + group)
    w = Weight(r, n, k, group, zeros)
    for m in rows:
        x, xt = activations(r, m, k, whole=True)
        want = product(x, w)
        out = torch.full(((m + 1) * n,), 7.5, dtype=torch.float32, device="cuda")
        call(xt, w, m, n, F32, out, n)
        got = du.to_host(out, np.float32).reshape(m + 1, n)
        assert np.array_equal(got[:m], want) and np.all(got[m] == 7.5), m
        res = orc.f32_to_bf16(r.integers(-99, 99, m * n).astype(np.float32))
        dres, out = du.to_dev(res), du.to_dev(np.full((m + 1) * n, 0x1234, np.uint16))
        call(xt, w, m, n, RESIDUAL, out, n, residual=dres)
        got = du.to_host(out, np.uint16).reshape(m + 1, n)
        assert np.array_equal(got[:m], narrow(want + widen(res).reshape(m, n))) and np.all(got[m] == 0x1234), m


@pytest.mark.parametrize("n", [4096, 4112])
@pytest.mark.parametrize("m", [1, 9, 32])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_split_slabs_of_wide_weights_add_up_exactly(n, m, group, zeros):
    r = np.random.default_rng(n + m)
    k, splits = 2176, 4  # 17 blocks of 128 columns: 5, 5, 5 and 2
    w = Weight(r, n, k, group, zeros)
    x, xt = activations(r, m, k, whole=True)
    out = torch.full(((splits * 32 + 1) * n,), 7.5, dtype=torch.float32, device="cuda")
    call(xt, w, m, n, PARTIAL, out, n, splits)
    got = du.to_host(out, np.float32).reshape(-1, n)
    slabs = got[:splits * 32].reshape(splits, 32, n)
    assert np.array_equal(slabs[:, :m].astype(np.float64).sum(0), product(x, w))
    assert np.all(slabs[:, m:] == 7.5) and np.all(got[-1] == 7.5)


@pytest.mark.parametrize("n,m", [(8192, 17), (16352, 1), (16384, 1), (16384, 9), (16384, 17), (16416, 32), (24576, 1),
                                 (24576, 32), (65536, 1), (65536, 8)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, True), (128, False)])
def test_swiglu_of_every_form(n, m, group, zeros):
    """Exact sums (scales are powers of two) narrowed to bf16; the exponential, a quotient and two products round in
    FP32, together less than 2^-20, then half a step of bf16."""
    r = np.random.default_rng(n + m)
    width, k = n // 2, 640
    scale = lambda: orc.f32_to_bf16((2.0 ** r.integers(-9, -6, width * (k // group))).astype(np.float32))  # noqa: E731
    gate = Weight(r, width, k, group, zeros, scales=scale(), half=True)
    up = Weight(r, width, k, group, zeros, scales=scale(), half=True)
    gate.tile(gate, 1)
    up.tile(gate, 2)
    x, xt = activations(r, m, k, whole=True)
    blocks = -(-width // 32)
    out, err = du.to_dev(np.full(1024 * blocks + 1024, 0x2222, np.uint16)), du.empty(1, np.uint32)
    call(xt, gate, m, n, SWIGLU, out, width, err=err)
    assert du.to_host(err, np.uint32)[0] == 0
    got = du.to_host(out, np.uint16)
    tiled = got[:1024 * blocks].reshape(blocks, 2, 4, 16, 8).transpose(1, 3, 0, 2, 4).reshape(32, 32 * blocks)
    assert np.all(got[1024 * blocks:] == 0x2222) and np.all(tiled[m:] == 0x2222) and np.all(tiled[:, width:] == 0x2222)
    g, u = (widen(narrow(product(x, w))) for w in (gate, up))
    want = g / (1 + np.exp(-g)) * u
    assert np.all(np.abs(widen(tiled[:m, :width]) - want) <= (2.0 ** -8 + 2.0 ** -20) * np.abs(want) + 1e-30)

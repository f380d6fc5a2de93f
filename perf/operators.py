"""What the operators for many continuations of one prompt are measured on: copies of KV pages (fork, compaction),
decode attention of a batch whose rows share a prefix, and projections with 4-bit weights.

The plain forms are elementary torch operations in 32 bits, rounded once at the end; with `own` set, `run` calls the
kernel roots of the C ABI (include/ferric_hip.h) instead, on the same inputs. Head counts and projection sizes are
those of Qwen3-8B and Qwen3-0.6B; lengths are generic.
"""

from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

PAGE, DIM = 16, 128
HEADS = {"8b": (32, 8), "0.6b": (16, 8)}  # query heads, KV heads
LAYERS = {"8b": 36, "0.6b": 28}
EPILOGUES = {"bf16": 0, "swiglu": 2, "f32": 3}


def listed():
    return [
        # One user's sequence is forked once: its last, partly filled page is copied in every layer (latency).
        dict(name="fork-0.6b-1", kind="copy", model="0.6b", pages=64, moves=1, lo=5, hi=5, fan=True),
        # 31 samples of one prompt: one partly filled page to 31 new ones.
        dict(name="fork-8b-31", kind="copy", model="8b", pages=256, moves=31, lo=9, hi=9, fan=True),
        # Compaction of a long-running pool: whole pages from its end into the holes below.
        dict(name="compact-8b-1111", kind="copy", model="8b", pages=2500, moves=1111, lo=16, hi=16, fan=False),
        # A few samples of a short prompt.
        dict(name="prefix-8b-b4", kind="prefix", model="8b", rows=4, groups=1, single=0, prefix=1488, lo=1, hi=100, per=1),
        # A full decode batch over one document, ragged continuations.
        dict(name="prefix-8b-b32", kind="prefix", model="8b", rows=32, groups=1, single=0, prefix=8192, lo=1, hi=500, per=1),
        # Two system prompts and a sequence of its own, the small model.
        dict(name="prefix-0.6b-b29", kind="prefix", model="0.6b", rows=29, groups=2, single=1, prefix=2000, lo=30, hi=900, per=1),
        # A speculative verify over one document: five rows a sequence.
        dict(name="prefix-8b-32x5", kind="prefix", model="8b", rows=160, groups=1, single=0, prefix=4096, lo=5, hi=300, per=5),
        # The largest: a full decode batch over a very long document.
        dict(name="prefix-8b-b32-long", kind="prefix", model="8b", rows=32, groups=1, single=0, prefix=32000, lo=1, hi=700, per=1),
        # One user, one token: the smallest projection, the largest of a layer, and the LM head of a small batch.
        dict(name="w4-0.6b-o-m1", kind="w4", n=1024, k=2048, m=1, group=128, zeros=0, epilogue="bf16"),
        dict(name="w4-8b-gateup-m1", kind="w4", n=24576, k=4096, m=1, group=128, zeros=0, epilogue="swiglu"),
        dict(name="w4-8b-head-m7", kind="w4", n=151936, k=4096, m=7, group=64, zeros=1, epilogue="f32"),
        # A full decode batch through the down projection, small groups with zero points.
        dict(name="w4-8b-down-m32", kind="w4", n=4096, k=12288, m=32, group=32, zeros=1, epilogue="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["copy", "prefix", "prefix", "w4", "w4"])
    model = rng.choice(["8b", "8b", "0.6b"])
    if kind == "copy":
        moves = _log(rng, 1, 1100)
        lo, hi = rng.choice([(16, 16), (1, 16), (rng.randint(1, 15),) * 2])
        return dict(kind=kind, model=model, pages=2 * moves + rng.randint(2, 200), moves=moves, lo=lo, hi=hi,
                    fan=rng.random() < 0.5)
    if kind == "prefix":
        per = rng.choice([1, 1, 1, rng.randint(2, 8)])
        rows = per * _log(rng, 1, 160 // per if per > 1 else 32)
        most = min(32000, 900000 // rows)  # the plain form reads every row's prefix
        prefix = PAGE * _log(rng, 1, most // PAGE)
        hi = max(per, _log(rng, 1, 2000))
        single = rng.choice([0, 0, 1]) if rows // per > 1 else 0
        groups = rng.randint(1, max(1, min(4, rows // per - single)))
        return dict(kind=kind, model=model, rows=rows, groups=groups, single=single, prefix=prefix,
                    lo=max(per, hi // rng.choice([2, 8, 1000])), hi=hi, per=per)
    n, k = rng.choice([(6144, 4096), (4096, 4096), (24576, 4096), (4096, 12288), (4096, 1024), (1024, 2048),
                       (6144, 1024), (32 * _log(rng, 1, 1000), 128 * _log(rng, 1, 64)), (151936, rng.choice([1024, 4096]))])
    case = dict(kind=kind, n=n, k=k, m=_log(rng, 1, 32), group=rng.choice([32, 64, 128, 128]),
                zeros=rng.choice([0, 1]), epilogue="f32" if n == 151936 else rng.choice(["bf16", "swiglu", "f32"]))
    if case["epilogue"] == "swiglu":  # the next projection's operand comes in whole blocks of 32 columns
        case["n"] += n % 64
    return case


# ---- inputs ---------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)


def _plan(case, seed):
    """Rows of a shared-prefix batch: (groups [first row, rows, prefix pages], page table, positions, physical pages).

    Rows of a group are whole sequences of `per` rows at consecutive positions; the `single` rows at the end share nothing."""
    rng = random.Random(seed)
    per, rows = case["per"], case["rows"]
    sequences = rows // per
    shared = sequences - case["single"]
    cuts = sorted(rng.sample(range(1, shared), case["groups"] - 1)) if case["groups"] > 1 else []
    cuts = [0] + cuts + [shared]
    prefix_pages = [case["prefix"] // PAGE if i == 0 else max(1, case["prefix"] // PAGE // (i + 1))
                    for i in range(case["groups"])]
    own_len = [rng.randint(case["lo"], case["hi"]) for _ in range(sequences)]
    own_len[0] = case["hi"]  # the longest length is there
    lengths, group_of = [], []
    for s in range(sequences):
        g = next((i for i in range(case["groups"]) if cuts[i] <= s < cuts[i + 1]), None)
        group_of.append(g)
        lengths.append((prefix_pages[g] * PAGE if g is not None else 0) + own_len[s])
    stride = max((n + PAGE - 1) // PAGE for n in lengths)
    order = list(range(sum(prefix_pages) + sum((n + PAGE - 1) // PAGE for n in own_len)))
    physical = len(order) + 3
    rng.shuffle(order)
    take = iter(order)
    prefixes = [[next(take) for _ in range(n)] for n in prefix_pages]
    table = np.full((rows, stride), 0xFFFFFFFF, np.uint32)
    positions = np.zeros(rows, np.uint32)
    for s in range(sequences):
        pages = list(prefixes[group_of[s]]) if group_of[s] is not None else []
        pages += [next(take) for _ in range((own_len[s] + PAGE - 1) // PAGE)]
        for i in range(per):
            table[s * per + i, :len(pages)] = pages
            positions[s * per + i] = lengths[s] - per + i
    groups = np.array([[cuts[i] * per, (cuts[i + 1] - cuts[i]) * per, prefix_pages[i]] for i in range(case["groups"])],
                      np.uint32)
    return groups, table, positions, physical


def _tile_weight(q):
    """4-bit weights [n][k] in their tile order: a tile is 16 rows x 128 columns, lane = row + 16 * (column % 32 // 8),
    four words a lane (32 columns apart), element e of 8 at bit 4 * (e // 2) + 16 * (e % 2)."""
    n, k = q.shape
    t = q.view(n // 16, 16, k // 128, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5)  # tile, lane group, row, word, parity, pair
    t = t.contiguous().view(-1, 4, 2)  # bytes of a word: nibbles 2 b and 2 b + 1
    t = t.view(-1, 2)
    return (t[:, 0] | (t[:, 1] << 4)).contiguous()


def _tile_rows(x, n):
    """Per-row, per-group values [n][groups] in their tile order [n / 16][groups][16]."""
    return x.view(n // 16, 16, -1).permute(0, 2, 1).contiguous()


def _interleave(x):
    """Tile rows of gate (first half) and up (second half) in turn: even tile rows gate, odd ones up."""
    half = x.shape[0] // 2
    return torch.stack([x[:half].reshape(half // 16, 16, -1), x[half:].reshape(half // 16, 16, -1)], 1).reshape(x.shape)


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "copy":
        kvh = HEADS[case["model"]][1]
        rng = np.random.default_rng(seed)
        order = rng.permutation(case["pages"])
        moves = np.empty((case["moves"], 3), np.uint32)
        moves[:, 0] = order[-1] if case["fan"] else order[case["moves"]:2 * case["moves"]]
        moves[:, 1] = order[:case["moves"]]
        moves[:, 2] = rng.integers(case["lo"], case["hi"] + 1, case["moves"])
        return dict(kind="copy", caches=_normal(g, 2 * LAYERS[case["model"]], case["pages"], PAGE, kvh, DIM), moves=moves)
    if case["kind"] == "prefix":
        qh, kvh = HEADS[case["model"]]
        groups, table, positions, physical = _plan(case, seed)
        context = table.shape[1] * PAGE
        state = dict(kind="prefix", qh=qh, kvh=kvh, groups=groups, context=context, physical=physical,
                     table=torch.from_numpy(table.view(np.int32)).cuda(),
                     positions=torch.from_numpy(positions.view(np.int32)).cuda(),
                     # Normalised queries and keys; the query norm's weights sharpen the softmax.
                     q=_normal(g, case["rows"], qh, DIM) * 2,
                     k=_normal(g, physical, PAGE, kvh, DIM), v=_normal(g, physical, PAGE, kvh, DIM),
                     out=torch.empty((case["rows"], qh, DIM), dtype=torch.bfloat16, device="cuda"),
                     error=torch.zeros(1, dtype=torch.int32, device="cuda"))
        return state
    n, k, m, group = case["n"], case["k"], case["m"], case["group"]
    q = torch.randint(0, 16, (n, k), dtype=torch.uint8, device="cuda", generator=g)
    # Scales of weights of standard deviation 0.02: a group's largest over 7, with some spread.
    scales = (torch.rand((n, k // group), device="cuda", generator=g) * 0.006 + 0.004).bfloat16()
    zeros = torch.randint(5, 11, (n, k // group), dtype=torch.uint8, device="cuda", generator=g) if case["zeros"] else None
    x = _normal(g, m, k)
    full = torch.zeros((32, k), dtype=torch.bfloat16, device="cuda")
    full[:m] = x
    wide = case["epilogue"] == "swiglu"
    lay = _interleave if wide else (lambda t: t)
    state = dict(kind="w4", n=n, k=k, m=m, group=group, epilogue=case["epilogue"], x=x, scales=scales, zeros=zeros,
                 packed=q[:, 0::2] | (q[:, 1::2] << 4),  # [n][k / 2], even columns in the low half
                 # As the weight and the activations lie in a running program: in tile order.
                 x_tiled=full.view(2, 16, k // 32, 4, 8).permute(2, 0, 3, 1, 4).contiguous(),
                 w_tiled=_tile_weight(lay(q)), scales_tiled=_tile_rows(lay(scales), n),
                 zeros_tiled=_tile_rows(lay(zeros), n) if zeros is not None else None,
                 error=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if wide:  # the next projection's operand: 32 rows in tile order, those past m as they were
        state["out"] = torch.zeros((-(-n // 64), 2, 4, 16, 8), dtype=torch.bfloat16, device="cuda")
    else:
        state["out"] = torch.empty((m, n), dtype=torch.float32 if case["epilogue"] == "f32" else torch.bfloat16,
                                   device="cuda")
    return state


# ---- one pass ---------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "copy":
        return _plain_copy(state)
    if state["kind"] == "prefix":
        return _plain_prefix(state)
    return _plain_w4(state)


def _plain_copy(state):
    caches, moves = state["caches"], torch.from_numpy(state["moves"].astype(np.int64)).cuda()
    src, dst, slots = moves[:, 0], moves[:, 1], moves[:, 2]
    kept = torch.arange(PAGE, device="cuda")[None, :] < slots[:, None]
    caches[:, dst] = torch.where(kept[None, :, :, None, None], caches[:, src], caches[:, dst])
    return caches


def _plain_prefix(state):
    qh, kvh, rows = state["qh"], state["kvh"], state["q"].shape[0]
    table = state["table"].long().clamp(min=0)
    seen = torch.arange(table.shape[1] * PAGE, device="cuda")[None, :] <= state["positions"].long()[:, None]
    q = state["q"].float().view(rows, kvh, qh // kvh, DIM) * DIM ** -0.5
    k = state["k"][table].float().view(rows, -1, kvh, DIM).permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(q, k).masked_fill(~seen[:, None, None, :], -math.inf)
    del k
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = state["v"][table].float().view(rows, -1, kvh, DIM).permute(0, 2, 1, 3).contiguous()
    return torch.matmul(p, v).reshape(rows, qh, DIM).bfloat16()


def _plain_w4(state):
    n, k, m, group = state["n"], state["k"], state["m"], state["group"]
    packed = state["packed"]
    q = torch.stack([packed & 15, packed >> 4], -1).view(n, k // group, group).float()
    z = state["zeros"].float()[..., None] if state["zeros"] is not None else 8.0
    w = ((q - z) * state["scales"].float()[..., None]).view(n, k)
    y = torch.matmul(state["x"].float(), w.t())
    if state["epilogue"] == "f32":
        return y
    if state["epilogue"] == "bf16":
        return y.bfloat16()
    gate, up = y[:, :n // 2].bfloat16().float(), y[:, n // 2:].bfloat16().float()
    full = torch.zeros((32, n // 2), dtype=torch.bfloat16, device="cuda")
    full[:m] = (gate / (1 + torch.exp(-gate)) * up).bfloat16()
    return full.view(2, 16, n // 64, 4, 8)


class _Api:
    """The library and its argument types, loaded at the first use."""

    lib = None

    @classmethod
    def get(cls):
        if cls.lib is None:
            import ferric_amd

            cls.lib = ferric_amd.load()
        return cls.lib


def _done(status):
    if status != 0:
        raise RuntimeError("status %d: %s" % (status, _Api.get().fh_last_error(None)))


def _run_own(state):
    lib, stream = _Api.get(), torch.cuda.current_stream().cuda_stream
    if state["kind"] == "copy":
        caches, moves = state["caches"], state["moves"]
        count, pages, _, kvh, _ = caches.shape
        _done(lib.fh_op_kv_copy_pages(caches.data_ptr(), count, pages * PAGE * kvh * DIM, moves.ctypes.data, len(moves),
                                      kvh, pages, stream))
        return caches
    if state["kind"] == "prefix":
        rows, qh, kvh, groups = state["q"].shape[0], state["qh"], state["kvh"], state["groups"]
        if "scratch" not in state:  # a program keeps it for the batch
            state["bytes"] = lib.fh_prefix_attention_scratch_bytes(groups.ctypes.data, len(groups), rows, qh, kvh,
                                                                   state["context"])
            state["scratch"] = torch.empty(state["bytes"], dtype=torch.uint8, device="cuda")
        _done(lib.fh_op_prefix_attention(
            state["q"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(), state["positions"].data_ptr(),
            state["table"].data_ptr(), groups.ctypes.data, len(groups), state["out"].data_ptr(), 0,
            state["scratch"].data_ptr(), state["bytes"], rows, qh, kvh, state["table"].shape[1], state["physical"],
            state["context"], state["error"].data_ptr(), stream))
        return state["out"]
    n, k, m, out = state["n"], state["k"], state["m"], state["out"]
    zeros = state["zeros_tiled"]
    wide = state["epilogue"] == "swiglu"
    _done(lib.fh_op_gemm_w4(state["x_tiled"].data_ptr(), state["w_tiled"].data_ptr(), state["scales_tiled"].data_ptr(),
                            zeros.data_ptr() if zeros is not None else None, m, n, k, state["group"],
                            EPILOGUES[state["epilogue"]], 1, None, out.data_ptr(), n // 2 if wide else n,
                            state["error"].data_ptr(), stream))
    return out.permute(1, 3, 0, 2, 4) if wide else out


# ---- what a pass needs, and what it should give ------------------------------

def work(case):
    if case["kind"] == "copy":
        slots = case["moves"] * (case["lo"] + case["hi"]) / 2
        read = case["hi"] if case["fan"] else slots
        return {"bytes": (slots + read) * HEADS[case["model"]][1] * DIM * 2 * 2 * LAYERS[case["model"]], "flops": 0}
    if case["kind"] == "prefix":
        qh, kvh = HEADS[case["model"]]
        groups, table, positions, _ = _plan(case, 0)
        per = case["per"]
        tokens = int(sum(int(g[2]) * PAGE for g in groups))
        shared = np.zeros(case["rows"], np.int64)
        for first, rows, pages in groups:
            shared[first:first + rows] = pages * PAGE
        tokens += int((positions.astype(np.int64) + 1 - shared)[per - 1::per].sum())
        return {"bytes": tokens * kvh * DIM * 4 + 2 * case["rows"] * qh * DIM * 2,
                "flops": 4 * DIM * qh * int((positions.astype(np.int64) + 1).sum())}
    n, k, m = case["n"], case["k"], case["m"]
    out = m * n * (4 if case["epilogue"] == "f32" else 1 if case["epilogue"] == "swiglu" else 2)
    return {"bytes": n * k / 2 + n * (k // case["group"]) * (3 if case["zeros"] else 2) + m * k * 2 + out,
            "flops": 2 * m * n * k}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "copy":
        caches = state["caches"]
        for src, dst, slots in state["moves"].tolist():
            caches[:, dst, :slots] = caches[:, src, :slots]
        return caches
    if case["kind"] == "prefix":
        qh, kvh = state["qh"], state["kvh"]
        out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
        for r, (pages, last) in enumerate(zip(state["table"].cpu().numpy(), state["positions"].tolist())):
            pages = torch.from_numpy(pages[:last // PAGE + 1].astype(np.int64)).cuda()
            for h in range(kvh):
                k = state["k"][pages, :, h].reshape(-1, DIM)[:last + 1].double()
                v = state["v"][pages, :, h].reshape(-1, DIM)[:last + 1].double()
                q = state["q"][r, h * (qh // kvh):(h + 1) * (qh // kvh)].double()
                w = torch.softmax(q @ k.t() / math.sqrt(DIM), -1)
                out[r, h * (qh // kvh):(h + 1) * (qh // kvh)] = w @ v
        return out
    n, k, m, group = case["n"], case["k"], case["m"], case["group"]
    y = torch.empty((m, n), dtype=torch.float64, device="cuda")
    x = state["x"].double()
    for at in range(0, n, 16384):
        rows = slice(at, min(n, at + 16384))
        packed = state["packed"][rows]
        w = torch.empty((packed.shape[0], k), dtype=torch.float64, device="cuda")
        w[:, 0::2] = packed.bitwise_and(15).double()
        w[:, 1::2] = packed.bitwise_right_shift(4).double()
        z = state["zeros"][rows].double() if state["zeros"] is not None else torch.full_like(state["scales"][rows], 8).double()
        w -= z.repeat_interleave(group, 1)
        w *= state["scales"][rows].double().repeat_interleave(group, 1)
        y[:, rows] = x @ w.t()
    if case["epilogue"] != "swiglu":
        return y
    # Gate and up are narrowed to bf16 by definition, the product once more at the end.
    gate, up = y[:, :n // 2].bfloat16().double(), y[:, n // 2:].bfloat16().double()
    full = torch.zeros((32, n // 2), dtype=torch.float64, device="cuda")
    full[:m] = gate * torch.sigmoid(gate) * up
    return full.view(2, 16, n // 64, 4, 8)

"""Attention over the paged cache with capped scores, a bias by distance, a
window with sink tokens, prefix and document masks: decode (single tokens and
drafted runs), fused append and decode, and chunked prefill, against float64.

Tolerance, per element, with u = eps/2 of the output type and ``spread`` the
softmax-weighted sum of |v|:  u |ref| + 2^-10 spread (+ fp16's smallest step).
The kernels hold P in fp16 (relative 2^-11) or in two bf16 parts (2^-17), which
moves the numerator by that share of ``spread``; the other 2^-11 allows the
scores an absolute error of 2^-12, twice (numerator and row sum): fp32 dot
products of up to 128 terms of size 4 sum to errors below 128 * 2^-24 * 16, the
cap's tanh is within 1e-6 of 50, the bias within 2^-24 of its size where the
key still counts (below 100), the exponential within 2^-22."""
import ctypes

import numpy as np
import pytest
import torch

from mlxz_b200 import _native, ops
from mlxz_b200._native import DeviceError
from oracle import rng
from oracle import score_mod as osm
from tests.gpu_util import TORCH, random_paged_case, to_bits, to_dev

gpu = pytest.mark.gpu


def _check(out, want, what=""):
    ref, spread = want
    u = 0.0 if out.dtype == torch.float32 else torch.finfo(out.dtype).eps / 2
    tiny = 2.0 ** -25 if out.dtype == torch.float16 else 0.0
    o = out.detach().float().cpu().numpy().astype(np.float64).reshape(ref.shape)
    tol = u * np.abs(ref) + 2.0 ** -10 * spread + tiny
    bad = ~(np.abs(o - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(o - ref)[bad].max()))


MODS = {
    "cap": dict(softcap=20.0),
    "slopes": dict(slopes=True),
    "window": dict(window=37),
    "window1": dict(window=1),
    "window_sink": dict(window=64, sink=4),
    "window_sinks": dict(window=16, sink=33),
    "far_sink": dict(window=5, sink=5000),
    "docs": dict(docs=50),
    "prefix": dict(prefix=29, window=20),
    "all": dict(softcap=50.0, slopes=True, window=100, sink=3, docs=130, prefix=10),
}


def _mod_args(mod, Hq, ctx, q_len, per_row, cuda):
    """(keyword arguments of ops, of the oracle) for a mod of MODS."""
    kw, ow = {}, {}
    if mod.get("softcap"):
        kw["softcap"] = ow["softcap"] = mod["softcap"]
    if mod.get("slopes"):
        s = (2.0 ** (-8.0 * (np.arange(Hq) + 1) / Hq)).astype(np.float32)
        kw["alibi_slopes"], ow["slopes"] = torch.from_numpy(s).to(cuda), s
    if mod.get("window"):
        kw["window"] = ow["window"] = mod["window"]
        kw["sink_tokens"] = ow["sink"] = mod.get("sink", 0)
    if mod.get("prefix"):
        # ragged: 0, the full length and beyond among them
        p = np.array([(mod["prefix"] * (b % 4)) for b in range(len(ctx))], dtype=np.int32)
        kw["prefix_lens"], ow["prefix"] = torch.from_numpy(p).to(cuda), p
    if mod.get("docs"):
        d = mod["docs"]
        if per_row:
            f = np.concatenate([np.arange(c - n, c) // d * d for c, n in zip(ctx, q_len)] or
                               [np.zeros(0)]).astype(np.int32)
            kw["first_keys"], ow["first"] = torch.from_numpy(f).to(cuda), f
        else:
            f = np.array([max(0, c - n) // d * d for c, n in zip(ctx, q_len)], dtype=np.int32)
            kw["first_keys"] = torch.from_numpy(f).to(cuda)
            ow["first"] = np.repeat(f, q_len)
    return kw, ow


def _dev(case, dtype, cuda):
    return (to_dev(case["kp"], dtype, cuda), to_dev(case["vp"], dtype, cuda),
            torch.from_numpy(case["tables"]).to(cuda), torch.from_numpy(case["ctx"]).to(cuda))


# --- decode ---------------------------------------------------------------------------

CTX = [300, 1, 15, 16, 17, 63, 64, 65, 0, 1000, 37, 129]


@gpu
@pytest.mark.parametrize("mod", MODS)
@pytest.mark.parametrize("dtype,D,G,bs,nq", [("bf16", 128, 4, 16, 1), ("f16", 64, 4, 32, 3),
                                             ("bf16", 64, 1, 48, 16), ("f16", 128, 16, 16, 1),
                                             ("bf16", 128, 2, 64, 5)])
def test_decode_vs_oracle(cuda, mod, dtype, D, G, bs, nq):
    Hkv, B = 2, len(CTX)
    case = random_paged_case(11 + D + nq, B, Hkv, D, bs, CTX, dtype, nq=nq, G=G)
    kp, vp, tables, ctx = _dev(case, dtype, cuda)
    q = to_dev(case["q"], dtype, cuda)
    q_len = np.full(B, nq)
    kw, ow = _mod_args(MODS[mod], Hkv * G, CTX, q_len, False, cuda)
    out = ops.paged_decode(q, kp, vp, tables, ctx, causal=True, out_dtype=torch.float32, **kw)
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    rows = case["q"].reshape(B * nq, Hkv * G, D)
    _check(out, osm.paged(rows, case["kp"], case["vp"], case["tables"], np.arange(B) * nq, q_len,
                          case["ctx"], dtype, **ow), mod)


@gpu
@pytest.mark.parametrize("num_warps", [0, 4, 8, 64])
@pytest.mark.parametrize("mod", ["window_sink", "all", "cap"])
def test_decode_split_over_warps(cuda, num_warps, mod):
    """Long contexts cut into pieces: some rows see nothing of some pieces."""
    dtype, D, G, nq, ctx = "bf16", 128, 4, 4, [5000, 3, 2047, 700]
    case = random_paged_case(3, 4, 2, D, 16, ctx, dtype, nq=nq, G=G)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    q = to_dev(case["q"], dtype, cuda)
    q_len = np.full(4, nq)
    m = dict(MODS[mod], window=2000) if mod == "all" else MODS[mod]
    kw, ow = _mod_args(m, 8, ctx, q_len, False, cuda)
    out = ops.paged_decode(q, kp, vp, tables, c, causal=True, num_warps=num_warps, **kw)
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    _check(out, osm.paged(case["q"].reshape(16, 8, D), case["kp"], case["vp"], case["tables"],
                          np.arange(4) * nq, q_len, case["ctx"], dtype, **ow), mod)


@gpu
def test_causal_without_mods_is_a_drafted_run(cuda):
    """Row i of a drafted run is the plain decode over its own prefix."""
    dtype, D, G, nq = "bf16", 64, 4, 4
    ctx = [200, 33, 4]
    case = random_paged_case(8, 3, 2, D, 16, ctx, dtype, nq=nq, G=G)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    q = to_dev(case["q"], dtype, cuda)
    out = ops.paged_decode(q, kp, vp, tables, c, causal=True)
    _check(out, osm.paged(case["q"].reshape(12, 8, D), case["kp"], case["vp"], case["tables"],
                          np.arange(3) * nq, np.full(3, nq), case["ctx"], dtype))
    one = ops.paged_decode(q[:, -1], kp, vp, tables, c)
    assert torch.equal(ops.paged_decode(q[:, -1], kp, vp, tables, c, causal=True), one)


@gpu
@pytest.mark.parametrize("nq", [1, 3])
def test_rows_that_see_nothing_are_zero(cuda, nq):
    """Documents that start behind the token; more drafted tokens than context."""
    dtype, D, ctx = "f16", 128, [40, 2, 100, 0]
    case = random_paged_case(5, 4, 2, D, 16, ctx, dtype, nq=nq, G=4)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    first = torch.tensor([40, 0, 1 << 30, 0], dtype=torch.int32, device=cuda)
    q = to_dev(case["q"], dtype, cuda)
    out = torch.full_like(q, 7.0)
    ops.paged_decode(q, kp, vp, tables, c, causal=True, first_keys=first, out=out)
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    assert not out[0].any() and not out[2].any() and not out[3].any()
    assert not out[1, :max(0, nq - 2)].any() and out[1, -1].any()


@gpu
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 6e4])
def test_decode_hidden_blocks_may_be_anything(cuda, fill):
    """What the window leaves out may be NaN, infinite or gone: blocks behind it
    lose their table entries, the rest of a partly seen tile holds ``fill``."""
    dtype, D, G, ctx, window, sink = "f16", 64, 4, [500, 130, 77], 70, 5
    case = random_paged_case(6, 3, 2, D, 16, ctx, dtype, G=G)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    q = to_dev(case["q"][:, 0], dtype, cuda)
    want = ops.paged_decode(q, kp, vp, tables, c, window=window, sink_tokens=sink)
    for b, n in enumerate(ctx):
        for t in range(sink, n - window):
            blk = int(tables[b, t // 16])
            kp[blk, :, t % 16] = fill
            vp[blk, :, t % 16] = fill
        for j in range(1, (n - window) // 16):
            tables[b, j] = -1 if j % 2 else 1 << 30
    got = ops.paged_decode(q, kp, vp, tables, c, window=window, sink_tokens=sink)
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("batch_invariant", [False, True])
@pytest.mark.parametrize("mod", ["cap", "window_sink", "docs", "all"])
def test_append_decode_vs_oracle(cuda, batch_invariant, mod):
    """The new token is written to its slot and attended in the same launch."""
    dtype, D, G, Hkv = "bf16", 128, 4, 2
    ctx = [300, 1, 16, 17, 2000, 129]
    B = len(ctx)
    case = random_paged_case(21, B, Hkv, D, 16, ctx, dtype, G=G)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    q = to_dev(case["q"][:, 0], dtype, cuda)
    kn, vn = (rng.normal(22, (B, Hkv, D), dtype, stream=s) for s in (1, 2))
    kw, ow = _mod_args(MODS[mod], Hkv * G, ctx, np.ones(B, dtype=int), False, cuda)
    out = ops.paged_append_decode(q, kp, vp, to_dev(kn, dtype, cuda), to_dev(vn, dtype, cuda),
                                  tables, c, batch_invariant=batch_invariant, **kw)
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    for b, n in enumerate(ctx):
        blk, at = case["tables"][b, (n - 1) // 16], (n - 1) % 16
        case["kp"][blk, :, at], case["vp"][blk, :, at] = kn[b], vn[b]
    assert np.array_equal(to_bits(kp), case["kp"]) and np.array_equal(to_bits(vp), case["vp"])
    _check(out, osm.paged(case["q"][:, 0], case["kp"], case["vp"], case["tables"], np.arange(B),
                          np.ones(B, dtype=int), case["ctx"], dtype, **ow), mod)


@gpu
@pytest.mark.parametrize("dtype,D,G,ctx,mod", [
    ("bf16", 128, 4, [5000], "cap"), ("f16", 64, 8, [9001], "slopes"),
    ("bf16", 64, 1, [6000, 3], "docs"), ("f16", 128, 2, [3333, 0, 70], "far_sink"),
    ("bf16", 128, 16, [4100], "prefix"), ("bf16", 128, 8, [16000], "cap")])
def test_decode_of_few_long_sequences(cuda, dtype, D, G, ctx, mod):
    """Pairs cut into many pieces: their merge, and warps left without a share."""
    B, Hkv = len(ctx), 2
    case = random_paged_case(25, B, Hkv, D, 16, ctx, dtype, G=G)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    q = to_dev(case["q"][:, 0], dtype, cuda)
    kw, ow = _mod_args(MODS[mod], Hkv * G, ctx, np.ones(B, dtype=int), False, cuda)
    want = osm.paged(case["q"][:, 0], case["kp"], case["vp"], case["tables"], np.arange(B),
                     np.ones(B, dtype=int), case["ctx"], dtype, **ow)
    first = None
    for _ in range(3):
        out = ops.paged_decode(q, kp, vp, tables, c, out_dtype=torch.float32, **kw)
        torch.cuda.synchronize()
        ops.check_device_errors(0)
        _check(out, want, mod)
        assert first is None or torch.equal(out, first)
        first = out


@gpu
def test_batch_invariant_bytes_with_a_window(cuda):
    """A sequence's bytes do not depend on the batch around it."""
    dtype, D, G, Hkv, ctx = "bf16", 64, 4, 2, [3000, 40, 900]
    case = random_paged_case(23, 3, Hkv, D, 16, ctx, dtype, G=G)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    q = to_dev(case["q"][:, 0], dtype, cuda)
    kn = to_dev(rng.normal(24, (3, Hkv, D), dtype), dtype, cuda)
    kw = dict(window=1500, sink_tokens=4, softcap=30.0, batch_invariant=True)
    out = ops.paged_append_decode(q, kp, vp, kn, kn, tables, c, **kw)
    for b in range(3):
        s = slice(b, b + 1)
        one = ops.paged_append_decode(q[s], kp, vp, kn[s], kn[s], tables[s].contiguous(), c[s], **kw)
        assert torch.equal(one[0], out[b])


@gpu
def test_decode_graph_and_two_streams(cuda):
    """Captured launches with their own workspaces on two streams at once, and
    lengths that change between replays."""
    dtype, D, G, ctx = "bf16", 128, 4, [900, 70]
    case = random_paged_case(31, 2, 2, D, 16, [1000, 90], dtype, G=G)
    kp, vp, tables, _ = _dev(case, dtype, cuda)
    c = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    q = to_dev(case["q"][:, 0], dtype, cuda)
    kw = dict(window=128, sink_tokens=4, softcap=30.0)
    graphs, outs, streams = [], [], []
    for _ in range(2):
        ws = ops.decode_workspace(2, 2, G, D, 0, shared=False)
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.paged_decode(q, kp, vp, tables, c, workspace=ws, **kw)
            with torch.cuda.graph(g, stream=s):
                outs.append(ops.paged_decode(q, kp, vp, tables, c, workspace=ws, **kw))
        graphs.append((g, ws))
        streams.append(s)
    torch.cuda.synchronize()
    for lens in ([900, 70], [1000, 90], [40, 1]):
        c.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for (g, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want = osm.paged(case["q"][:, 0], case["kp"], case["vp"], case["tables"], np.arange(2),
                         np.ones(2, dtype=int), np.array(lens), dtype, softcap=30.0, window=128,
                         sink=4)
        for o in outs:
            _check(o, want, lens)
    ops.check_device_errors(0)


# --- prefill --------------------------------------------------------------------------

def _prefill_case(seed, ctx, qlen, dtype, D, G, bs, Hkv):
    case = random_paged_case(seed, len(ctx), Hkv, D, bs, ctx, dtype, G=G)
    T = sum(qlen)
    case["qp"] = rng.normal(seed, (max(T, 1), Hkv * G, D), dtype, stream=9)[:T]
    case["q_start"] = np.cumsum([0] + qlen[:-1]).astype(np.int32)
    case["q_len"] = np.array(qlen, dtype=np.int32)
    return case


def _prefill(case, dtype, cuda, kw, out_dtype=None, out=None, pools=None):
    kp, vp, tables, ctx = pools or _dev(case, dtype, cuda)
    i = {k: torch.from_numpy(case[k]).to(cuda) for k in ("q_start", "q_len")}
    res = ops.paged_prefill(to_dev(case["qp"], dtype, cuda), kp, vp, tables, i["q_start"],
                            i["q_len"], ctx, int(case["q_len"].max()), out_dtype=out_dtype,
                            out=out, **kw)
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    return res


PREFILL = [
    # dtype, D, G, bs, ctx (chunk included), q_len
    ("bf16", 128, 8, 16, [100, 300, 17, 64, 513], [100, 37, 1, 0, 200]),
    ("f16", 64, 1, 16, [1000, 129], [513, 129]),
    ("bf16", 64, 16, 32, [77, 40, 300], [30, 40, 299]),
    ("f16", 128, 4, 64, [2000, 5], [200, 5]),
    ("bf16", 128, 2, 48, [16, 33, 1, 385], [16, 33, 1, 385]),
]


@gpu
@pytest.mark.parametrize("mod", MODS)
@pytest.mark.parametrize("dtype,D,G,bs,ctx,qlen", PREFILL)
def test_prefill_vs_oracle(cuda, mod, dtype, D, G, bs, ctx, qlen):
    Hkv = 2
    case = _prefill_case(40 + D + G, ctx, qlen, dtype, D, G, bs, Hkv)
    kw, ow = _mod_args(MODS[mod], Hkv * G, ctx, qlen, True, cuda)
    out = _prefill(case, dtype, cuda, kw, torch.float32)
    _check(out, osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                          case["q_len"], case["ctx"], dtype, **ow), mod)


@gpu
@pytest.mark.parametrize("window,sink", [(128, 0), (129, 4), (500, 128), (1000, 200), (4000, 4)])
def test_prefill_long_window(cuda, window, sink):
    """Windows that leave out whole key tiles, at and off their borders."""
    case = _prefill_case(50, [3000, 900], [260, 130], "bf16", 128, 4, 16, 1)
    out = _prefill(case, "bf16", cuda, dict(window=window, sink_tokens=sink))
    _check(out, osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                          case["q_len"], case["ctx"], "bf16", window=window, sink=sink))


@gpu
def test_prefill_prefix_ahead_of_the_chunk(cuda):
    """A first chunk inside its prefix sees keys that lie ahead of it, several
    key tiles on."""
    ctx, qlen, pre = [700, 700, 300], [40, 700, 100], np.array([650, 650, 900], dtype=np.int32)
    case = _prefill_case(51, ctx, qlen, "bf16", 64, 2, 16, 2)
    for kw in ({}, dict(window=30), dict(softcap=20.0)):
        out = _prefill(case, "bf16", cuda, dict(kw, prefix_lens=torch.from_numpy(pre).to(cuda)))
        _check(out, osm.paged(case["qp"], case["kp"], case["vp"], case["tables"],
                              case["q_start"], case["q_len"], case["ctx"], "bf16", prefix=pre,
                              **kw), kw)


@gpu
def test_prefill_empty_rows_and_rows_of_no_sequence(cuda):
    """Rows that see nothing are zero; rows behind the last sequence stay."""
    case = _prefill_case(52, [300, 140], [200, 130], "f16", 128, 4, 16, 2)
    T = 330
    first = np.zeros(T + 9, dtype=np.int32)
    first[50:180] = 1 << 30      # more than a whole query block of empty rows
    first[200:330] = np.arange(130) + 10 - 3
    case["qp"] = rng.normal(52, (T + 9, 8, 128), "f16", stream=9)
    out = torch.full((T + 9, 8, 128), 7.0, dtype=torch.float16, device=cuda)
    _prefill(case, "f16", cuda, dict(first_keys=torch.from_numpy(first).to(cuda)), out=out)
    assert not out[50:180].any() and (out[T:] == 7).all()
    want = osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                     case["q_len"], case["ctx"], "f16", first=first)
    _check(out[:T], (want[0][:T], want[1][:T]))


@gpu
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_prefill_hidden_blocks_may_be_anything(cuda, fill):
    ctx, qlen, window, sink = [900, 400], [100, 40], 150, 20
    case = _prefill_case(53, ctx, qlen, "bf16", 128, 4, 16, 2)
    kw = dict(window=window, sink_tokens=sink)
    want = _prefill(case, "bf16", cuda, kw)
    kp, vp, tables, c = _dev(case, "bf16", cuda)
    for b, (n, m) in enumerate(zip(ctx, qlen)):
        lo = n - m - window + 1  # the first row's lowest key
        for t in range(sink, lo):
            blk = int(tables[b, t // 16])
            kp[blk, :, t % 16] = fill
            vp[blk, :, t % 16] = fill
        for j in range(-(-sink // 16), lo // 16):
            tables[b, j] = -1
    got = _prefill(case, "bf16", cuda, kw, pools=(kp, vp, tables, c))
    # G = 4: a query block is 32 tokens, the later ones' hidden keys include seen ones
    assert torch.equal(got, want)


# Few query blocks over long tables: their keys are shared out over clusters of 8, 4,
# 2 and 1 blocks, or (many query blocks, or short tables) not at all.
FEW = [
    ("bf16", 128, 4, 16, 2, [4500], [5]),
    ("f16", 64, 8, 32, 1, [4490, 4100, 70], [1, 20, 16]),
    ("f16", 128, 2, 16, 2, [2100, 300, 40], [70, 64, 0]),
    ("bf16", 64, 4, 64, 3, [1100, 65, 1], [33, 65, 1]),
    ("bf16", 128, 16, 16, 5, [600, 590, 513], [30, 1, 9]),
    ("bf16", 64, 4, 16, 8, [650] * 6 + [70] * 4, [40] * 9 + [0]),
]


@gpu
@pytest.mark.parametrize("mod", ["cap", "slopes", "window_sinks", "docs", "prefix", "all"])
@pytest.mark.parametrize("dtype,D,G,bs,Hkv,ctx,qlen", FEW)
def test_prefill_of_few_rows(cuda, mod, dtype, D, G, bs, Hkv, ctx, qlen):
    case = _prefill_case(60 + D + G, ctx, qlen, dtype, D, G, bs, Hkv)
    kw, ow = _mod_args(MODS[mod], Hkv * G, ctx, qlen, True, cuda)
    for out_dtype in (torch.float32, TORCH[dtype]):
        out = _prefill(case, dtype, cuda, kw, out_dtype)
        _check(out, osm.paged(case["qp"], case["kp"], case["vp"], case["tables"],
                              case["q_start"], case["q_len"], case["ctx"], dtype, **ow), mod)


@gpu
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_prefill_of_few_rows_with_hidden_blocks_and_empty_rows(cuda, fill):
    """A window over part of the keys, whose other blocks may be anything; rows
    that see nothing; rows behind the last sequence."""
    ctx, qlen, window, sink = [5000, 3100], [40, 9], 3000, 20
    case = _prefill_case(61, ctx, qlen, "bf16", 128, 4, 16, 1)
    case["qp"] = rng.normal(61, (60, 4, 128), "bf16", stream=9)
    first = np.zeros(60, dtype=np.int32)
    first[3:36] = 1 << 30  # but for the sinks; the second query block sees more
    kp, vp, tables, c = _dev(case, "bf16", cuda)
    for b, (n, m) in enumerate(zip(ctx, qlen)):
        lo = n - m - window + 1
        for t in range(sink, lo):
            blk = int(tables[b, t // 16])
            kp[blk, :, t % 16] = fill
            vp[blk, :, t % 16] = fill
        for j in range(-(-sink // 16), lo // 16):
            tables[b, j] = -1
    for s in (sink, 0):
        if s == 0:
            kp[tables[:, 0].long()] = fill
            kp[tables[:, 1].long()] = fill
        out = torch.full((60, 4, 128), 7.0, dtype=torch.bfloat16, device=cuda)
        _prefill(case, "bf16", cuda, dict(window=window, sink_tokens=s,
                                          first_keys=torch.from_numpy(first).to(cuda)),
                 out=out, pools=(kp, vp, tables, c))
        assert (out[49:] == 7).all() and (s > 0 or not out[3:36].any())
        want = osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                         case["q_len"], case["ctx"], "bf16", first=first, window=window, sink=s)
        _check(out[:49], (want[0][:49], want[1][:49]))


@gpu
def test_prefill_of_few_rows_in_a_graph_and_with_a_bad_sequence(cuda):
    """Lengths that change between replays, one stream next to another; a
    sequence in error leaves its rows and the others' results alone."""
    ctx, qlen = [4300, 4300], [6, 4]
    case = _prefill_case(62, ctx, qlen, "f16", 128, 4, 16, 2)
    kp, vp, tables, c = _dev(case, "f16", cuda)
    i = {k: torch.from_numpy(case[k]).to(cuda) for k in ("q_start", "q_len")}
    q = to_dev(case["qp"], "f16", cuda)
    kw = dict(softcap=25.0, first_keys=torch.full((10,), 3, dtype=torch.int32, device=cuda))
    runs = []
    for _ in range(2):
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call = lambda: ops.paged_prefill(q, kp, vp, tables, i["q_start"], i["q_len"], c, 6, **kw)
            call()
            with torch.cuda.graph(g, stream=s):
                runs.append((g, s, call()))
    torch.cuda.synchronize()
    for lens in ([4300, 4300], [6, 4], [200, 4001]):
        c.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s, _ in runs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        ops.check_device_errors(0)
        want = osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                         case["q_len"], np.array(lens), "f16", softcap=25.0,
                         first=np.full(10, 3))
        for _, _, out in runs:
            _check(out, want, lens)
    c.copy_(torch.tensor([2, 4001], dtype=torch.int32))  # fewer tokens than query rows
    out = torch.full_like(runs[0][2], 7.0)
    ops.paged_prefill(q, kp, vp, tables, i["q_start"], i["q_len"], c, 6, out=out, **kw)
    with pytest.raises(DeviceError, match="context length"):
        ops.check_device_errors(0)
    assert (out[:6] == 7).all()
    _check(out[6:], (want[0][6:], want[1][6:]))


@gpu
def test_prefill_last_row_equals_decode(cuda):
    case = _prefill_case(54, [700, 250], [64, 9], "f16", 128, 8, 16, 1)
    kw = dict(softcap=30.0, window=200, sink_tokens=4)
    out = _prefill(case, "f16", cuda, kw, torch.float32)
    kp, vp, tables, ctx = _dev(case, "f16", cuda)
    last = case["q_start"] + case["q_len"] - 1
    dec = ops.paged_decode(to_dev(case["qp"][last], "f16", cuda), kp, vp, tables, ctx,
                           out_dtype=torch.float32, **kw)
    want = osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                     case["q_len"], case["ctx"], "f16", softcap=30.0, window=200, sink=4)
    rows = (want[0][last], want[1][last])
    _check(out[torch.from_numpy(last).long()], rows)
    _check(dec, rows)


@gpu
def test_decode_with_every_key_hidden_reads_no_table_entry(cuda):
    """A token that sees no key needs no valid block: zeros and no error."""
    q, kp, vp, tables, _ = (t.to(cuda) for t in _host())
    q += 1
    vp[:] = float("nan")
    tables[0] = torch.tensor([-1, 1 << 20])
    tables[1] = torch.tensor([2, 3])
    vp[2:] = 0.5
    ctx = torch.tensor([32, 32], dtype=torch.int32, device=cuda)
    first = torch.tensor([32, 31], dtype=torch.int32, device=cuda)
    out = ops.paged_decode(q, kp, vp, tables, ctx, first_keys=first)
    ops.check_device_errors(0)
    assert (out[0] == 0).all() and (out[1] == 0.5).all()


@gpu
def test_drafted_tokens_before_the_sequence_see_the_prefix(cuda):
    """Two cached tokens and four query tokens: those at positions below 0 see
    the prefix alone, and nothing without one.  Values are exact: V is 1."""
    q, kp, vp, tables, _ = (t.to(cuda) for t in _host(nq=4))
    vp[:] = 1
    ctx = torch.full((2,), 2, dtype=torch.int32, device=cuda)
    prefix = torch.tensor([1, 0], dtype=torch.int32, device=cuda)
    out = ops.paged_decode(q, kp, vp, tables, ctx, causal=True, prefix_lens=prefix)
    ops.check_device_errors(0)
    assert (out[0] == 1).all() and (out[1, :2] == 0).all() and (out[1, 2:] == 1).all()


@gpu
def test_context_beyond_2_to_30_without_a_window(cuda):
    """No window hides nothing, however long the context.  All but the first
    block of the table are one block of zero keys (score 0, value 0); the first
    block's first key scores 64, so its value 1 has weight 1 / (1 + n e^-64),
    n = 2^30 + 32, which is 1 to 2e-19 and exact in bf16."""
    D, bs, blocks = 64, 256, (1 << 22) + 1
    kp = torch.zeros(2, 1, bs, D, dtype=torch.bfloat16, device=cuda)
    vp = torch.zeros_like(kp)
    kp[1, 0, 0], vp[1, 0, 0] = 1, 1
    q = torch.ones(1, 2, D, dtype=torch.bfloat16, device=cuda)
    tables = torch.zeros(1, blocks, dtype=torch.int32, device=cuda)
    tables[0, 0] = 1
    ctx = torch.tensor([(1 << 30) + 32], dtype=torch.int32, device=cuda)
    slopes = torch.zeros(2, device=cuda)
    out = ops.paged_decode(q, kp, vp, tables, ctx, scale=1.0, alibi_slopes=slopes)
    ops.check_device_errors(0)
    assert (out == 1).all()


# --- refusals -------------------------------------------------------------------------

def _host(B=2, Hq=8, Hkv=2, D=64, nq=None):
    q = torch.zeros(B, Hq, D, dtype=torch.bfloat16) if nq is None else \
        torch.zeros(B, nq, Hq, D, dtype=torch.bfloat16)
    pool = torch.zeros(4, Hkv, 16, D, dtype=torch.bfloat16)
    return q, pool, pool, torch.zeros(B, 2, dtype=torch.int32), torch.ones(B, dtype=torch.int32)


BAD = [(dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
       (dict(window=-1), "window"), (dict(window=3, sink_tokens=-1), "sink"),
       (dict(alibi_slopes=torch.zeros(8, dtype=torch.float64)), "alibi_slopes"),
       (dict(alibi_slopes=torch.zeros(2)), "alibi_slopes"),
       (dict(prefix_lens=torch.zeros(3, dtype=torch.int32)), "prefix_lens"),
       (dict(prefix_lens=torch.zeros(2, dtype=torch.int64)), "prefix_lens"),
       (dict(first_keys=torch.zeros(5, dtype=torch.int32)), "first_keys")]


@pytest.mark.parametrize("kw,text", BAD)
def test_refusals_on_the_host(kw, text):
    q, kp, vp, tables, ctx = _host()
    with pytest.raises(ValueError, match=text):
        ops.paged_decode(q, kp, vp, tables, ctx, **kw)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=text):
        ops.paged_append_decode(q, kp, vp, k, k, tables, ctx, **kw)
    with pytest.raises(ValueError, match=text):
        ops.paged_prefill(q, kp, vp, tables, ctx, ctx, ctx, 1, **kw)


@gpu
def test_tensors_off_the_pools_device_are_refused(cuda):
    on = [t.to(cuda) for t in _host()]
    q, kp, vp, tables, ctx = on
    far = torch.empty(q.shape, dtype=q.dtype)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="out must be on the pools' device"):
        ops.paged_decode(*on, window=4, out=far)
    with pytest.raises(ValueError, match="workspace must be on the pools' device"):
        ops.paged_decode(*on, window=4, workspace=torch.zeros(1 << 20, dtype=torch.uint8))
    with pytest.raises(ValueError, match="q must be on the pools' device"):
        ops.paged_decode(torch.zeros(2, 2, 8, 64, dtype=q.dtype), *on[1:], causal=True)
    with pytest.raises(ValueError, match="out must be on the pools' device"):
        ops.paged_append_decode(q, kp, vp, k.to(cuda), k.to(cuda), tables, ctx, window=4, out=far)
    with pytest.raises(ValueError, match="v_new must be on the pools' device"):
        ops.paged_append_decode(q, kp, vp, k.to(cuda), k, tables, ctx, window=4)
    with pytest.raises(ValueError, match="out must be on the pools' device"):
        ops.paged_prefill(q, kp, vp, tables, ctx, ctx, ctx, 1, window=4, out=far)


def test_several_tokens_need_causal():
    q, kp, vp, tables, ctx = _host(nq=3)
    with pytest.raises(ValueError, match="causal"):
        ops.paged_decode(q, kp, vp, tables, ctx, window=4)


def test_c_abi_argument_errors():
    lib = _native.lib()
    p = ctypes.c_void_p(64)  # never read: every call below is refused first

    def prefill(mod, D=64):
        return lib.mz_paged_prefill_mod(p, 1, 512, 64, p, 512, 64, 4, p, p, 4, p, p, p, 2, p, 1, 8,
                                        2, D, 16, 4, 0.125, mod, 1, None, None)

    def append(mod):
        return lib.mz_paged_append_decode_mod(p, 1, 512, 64, p, 512, 64, p, p, p, p, 128, 64, p, 2,
                                              p, 1, 8, 2, 64, 16, 4, 0.125, mod, 1, 0, 0, p, 0,
                                              None, None)

    inv, ali = _native.MZ_ERR_INVALID_ARG, _native.MZ_ERR_ALIGNMENT
    for fields, rc in ((dict(softcap=-2.0), inv), (dict(softcap=float("inf")), inv),
                       (dict(window=-1), inv), (dict(sink_tokens=-3), inv),
                       (dict(alibi_slopes=66), ali), (dict(prefix_lens=65), ali),
                       (dict(first_keys=67), ali)):
        assert append(ctypes.byref(_native.ScoreMod(**fields))) == rc, fields
    assert prefill(None) == inv and append(None) == inv
    ok = ctypes.byref(_native.ScoreMod(softcap=3.0))
    assert prefill(ok, D=96) == _native.MZ_ERR_UNSUPPORTED


def test_oracle_masks():
    """The visibility rule on a case small enough to read."""
    v = osm.visible(np.array([5]), 8, window=2, sink=1)[0]
    assert v.tolist() == [True, False, False, False, True, True, False, False]
    v = osm.visible(np.array([1, 5]), 8, window=2, prefix=3, first=np.array([0, 5]))
    assert v[0].tolist() == [True] * 3 + [False] * 5
    assert v[1].tolist() == [True] * 3 + [False] * 2 + [True] + [False] * 2


@gpu
def test_default_workspaces_of_two_streams_and_of_two_graphs(cuda):
    """Calls that bring no workspace, at once on two streams, and two captured
    graphs replayed at once."""
    dtype, D, G, ctx = "bf16", 128, 4, [3000, 70, 900]
    case = random_paged_case(33, 3, 2, D, 16, ctx, dtype, G=G)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    q = to_dev(case["q"][:, 0], dtype, cuda)
    kw = dict(window=2000, sink_tokens=4, softcap=30.0)
    want = osm.paged(case["q"][:, 0], case["kp"], case["vp"], case["tables"], np.arange(3),
                     np.ones(3, dtype=int), case["ctx"], dtype, softcap=30.0, window=2000, sink=4)
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(ops.paged_decode(q, kp, vp, tables, c, **kw))
            graphs.append(g)
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                outs.append(ops.paged_decode(q, kp, vp, tables, c, **kw))
                g.replay()
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    for o in outs:
        _check(o, want)


@gpu
@pytest.mark.parametrize("softcap", [1e-6, 0.5, 1500.0, 3e4, 1e29, 1e32])
def test_caps_of_every_size(cuda, softcap):
    """From caps that bind every score to those that touch none, with scores near
    and far beyond half the cap in the same tile."""
    dtype, D, G, ctx, qlen = "bf16", 64, 4, [130, 300], [70, 9]
    case = _prefill_case(60, ctx, qlen, dtype, D, G, 16, 2)
    # scores of standard deviation 8
    case["qp"] = to_bits(8 * to_dev(case["qp"], dtype, "cpu"))
    want = osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                     case["q_len"], case["ctx"], dtype, softcap=softcap)
    _check(_prefill(case, dtype, cuda, dict(softcap=softcap)), want)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    last = case["q_start"] + case["q_len"] - 1
    out = ops.paged_decode(to_dev(case["qp"][last], dtype, cuda), kp, vp, tables, c,
                           softcap=softcap)
    _check(out, (want[0][last], want[1][last]))
    ops.check_device_errors(0)


@gpu
def test_nan_keys_and_queries_reach_their_rows_only(cuda):
    """A NaN key poisons the rows that see it, a NaN query its own row."""
    dtype, D, ctx = "bf16", 64, [40, 40]
    case = _prefill_case(61, ctx, [40, 40], dtype, D, 2, 16, 1)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    kp[int(tables[0, 2]), :, 3] = float("nan")  # key 35 of the first request
    q = to_dev(case["qp"], dtype, cuda)
    q[40 + 7, 1] = float("nan")
    i = {k: torch.from_numpy(case[k]).to(cuda) for k in ("q_start", "q_len")}
    kw = dict(window=4, softcap=20.0)
    out = ops.paged_prefill(q, kp, vp, tables, i["q_start"], i["q_len"], c, 40, **kw)
    bad = out.isnan().all(-1)
    want = torch.zeros(80, 2, dtype=torch.bool)
    want[35:39] = True
    want[47, 1] = True
    assert torch.equal(bad.cpu(), want) and torch.equal(out.isnan().any(-1), bad)
    dec = ops.paged_decode(q[[38, 47]].contiguous(), kp, vp, tables, c - 1, **kw)
    assert dec[0].isnan().all() and dec[1, 1].isnan().all() and not dec[1, 0].isnan().any()


def test_caps_that_overflow_and_tables_too_wide_are_refused():
    lib = _native.lib()
    p = ctypes.c_void_p(64)

    def append(width=2, **mod):
        return lib.mz_paged_append_decode_mod(
            p, 1, 512, 64, p, 512, 64, p, p, p, p, 128, 64, p, width, p, 1, 8, 2, 64, 16, 4, 0.125,
            ctypes.byref(_native.ScoreMod(**mod)), 1, 0, 0, p, 0, None, None)

    assert append(softcap=1e-40) == _native.MZ_ERR_INVALID_ARG
    assert append(width=1 << 27, window=3) == _native.MZ_ERR_UNSUPPORTED


@gpu
@pytest.mark.parametrize("softcap", [20.0, 3e4, 1e29])
def test_capped_prefill_ignores_what_lies_behind_the_last_key(cuda, softcap):
    """The last tile's rows behind the sequence are whatever the block holds:
    huge values there change no byte."""
    dtype, D, G, ctx, qlen = "bf16", 64, 4, [130, 300], [70, 9]
    case = _prefill_case(62, ctx, qlen, dtype, D, G, 16, 2)
    want = _prefill(case, dtype, cuda, dict(softcap=softcap))
    kp, vp, tables, c = _dev(case, dtype, cuda)
    for b, n in enumerate(ctx):
        for fill in (3e38, float("nan"), float("-inf")):
            blk = int(tables[b, (n - 1) // 16])
            kp[blk, :, n % 16:] = fill
            vp[blk, :, n % 16:] = fill
            got = _prefill(case, dtype, cuda, dict(softcap=softcap), pools=(kp, vp, tables, c))
            assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("softcap", [0.0, 5.0, 30.0])
def test_negative_slopes_raise_far_scores(cuda, softcap):
    """Slopes below 0: scores grow with the distance, beyond the cap."""
    dtype, D, G, ctx, qlen = "bf16", 64, 2, [700, 130], [90, 130]
    case = _prefill_case(63, ctx, qlen, dtype, D, G, 16, 2)
    s = np.array([-0.25, -0.01, 0.0, 0.5], dtype=np.float32)
    kw = dict(softcap=softcap, alibi_slopes=torch.from_numpy(s).to(cuda))
    want = osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                     case["q_len"], case["ctx"], dtype, softcap=softcap, slopes=s)
    _check(_prefill(case, dtype, cuda, kw), want)
    kp, vp, tables, c = _dev(case, dtype, cuda)
    last = case["q_start"] + case["q_len"] - 1
    out = ops.paged_decode(to_dev(case["qp"][last], dtype, cuda), kp, vp, tables, c, **kw)
    _check(out, (want[0][last], want[1][last]))


def _torch_pools(cuda, seed, n_blocks, Hkv, bs, D, dtype=torch.bfloat16):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(n_blocks, Hkv, bs, D, generator=g, device=cuda).to(dtype) for _ in range(2))


@gpu
@pytest.mark.parametrize("D,G,kw", [(128, 4, dict(softcap=30.0)), (64, 8, dict(window=3400)),
                                    (128, 1, dict(softcap=30.0)), (64, 16, dict(softcap=30.0)),
                                    (128, 4, {}), (64, 8, {}), (128, 16, {}), (64, 16, {})])
def test_batch_invariant_bytes_with_many_merges_a_warp(cuda, D, G, kw):
    """A sequence's bytes do not depend on the batch around it, nor on the run,
    where its pieces are many (3500 tokens: seven) and a warp merges more pairs
    than its list of eight holds (24 sequences of 4 KV heads on 8 warps)."""
    B, Hkv, bs = 24, 4, 16
    ctx = [3500 - 7 * b for b in range(B)]
    width = -(-max(ctx) // bs)
    kp, vp = _torch_pools(cuda, 71, B * width, Hkv, bs, D)
    tables = torch.randperm(B * width, generator=torch.Generator().manual_seed(72)).int()
    tables = tables.reshape(B, width).to(cuda)
    c = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(73)
    q = torch.randn(B, Hkv * G, D, generator=g, device=cuda).to(kp.dtype)
    kn, vn = (torch.randn(B, Hkv, D, generator=g, device=cuda).to(kp.dtype) for _ in range(2))
    kw = dict(kw, batch_invariant=True, num_warps=8, out_dtype=torch.float32)
    runs = [ops.paged_append_decode(q, kp, vp, kn, vn, tables, c, **kw) for _ in range(4)]
    for b in range(0, B, 3):
        s = slice(b, b + 1)
        one = ops.paged_append_decode(q[s], kp, vp, kn[s], vn[s], tables[s].contiguous(), c[s], **kw)
        for out in runs:
            assert torch.equal(one[0], out[b]), b
    ops.check_device_errors(0)


@gpu
@pytest.mark.parametrize("ctx", [[300, 130, 4300], [4300, 1, 4300]])
@pytest.mark.parametrize("n", [(1 << 31) - 1, (1 << 31) - 16, 1 << 30, 301])
def test_prefill_reports_a_length_of_any_size(cuda, ctx, n):
    """A sequence whose query length on the device exceeds its context, up to
    2^31 - 1, is reported; the sequences behind it are computed all the same."""
    qlen = [20, 1, 33]
    case = _prefill_case(64, ctx, qlen, "bf16", 64, 4, 16, 2)
    kp, vp, tables, c = _dev(case, "bf16", cuda)
    c[0] = 300
    lens = torch.tensor([n, 1, 33], dtype=torch.int32, device=cuda)
    starts = torch.from_numpy(case["q_start"]).to(cuda)
    out = torch.full((54, 8, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    ops.paged_prefill(to_dev(case["qp"], "bf16", cuda), kp, vp, tables, starts, lens, c, 33,
                      softcap=20.0, out=out)
    with pytest.raises(DeviceError, match="context length"):
        ops.check_device_errors(0)
    assert (out[:20] == 7).all()
    want = osm.paged(case["qp"], case["kp"], case["vp"], case["tables"], case["q_start"],
                     case["q_len"], case["ctx"], "bf16", softcap=20.0)
    _check(out[20:], (want[0][20:], want[1][20:]))


@gpu
@pytest.mark.parametrize("window", [1, 100, 4000])
@pytest.mark.parametrize("ctx", [(1 << 31) - 2048, (1 << 31) - 2048 - 1000])
def test_window_over_the_longest_context(cuda, window, ctx):
    """The widest table that is taken (2^31 - 2048 tokens): the block ids that are
    loaded ahead end behind the last key, and past 2^31.  All its entries are
    one block of 1024 tokens, so a short cache of the same block has the same
    keys in the window."""
    D, bs, G, n = 64, 1024, 2, 3
    case = random_paged_case(65, 1, 1, D, bs, [bs], "bf16", n_blocks=1, G=G)
    kp, vp = (to_dev(case[k], "bf16", cuda) for k in ("kp", "vp"))
    case["qp"] = rng.normal(65, (n, G, D), "bf16", stream=9)
    q = to_dev(case["qp"], "bf16", cuda)
    tables = torch.zeros(1, (1 << 21) - 2, dtype=torch.int32, device=cuda)
    short = 8192 - ((1 << 31) - ctx) % bs
    want = osm.paged(case["qp"], case["kp"], case["vp"], np.zeros((1, 8), dtype=np.int32),
                     np.array([0]), np.array([n]), np.array([short]), "bf16", window=window)
    c = torch.tensor([ctx], dtype=torch.int32, device=cuda)
    i = [torch.tensor([x], dtype=torch.int32, device=cuda) for x in (0, n)]
    out = ops.paged_prefill(q, kp, vp, tables, *i, c, n, window=window)
    ops.check_device_errors(0)
    _check(out, want)
    out = ops.paged_decode(q[None], kp, vp, tables, c, window=window, causal=True)
    ops.check_device_errors(0)
    _check(out[0], want)


@pytest.mark.parametrize("softcap", [1e-50, 1e-40, 5e-324])
def test_caps_below_float32_are_refused(softcap):
    """Rounded to float32 they would be 0, which stands for no cap."""
    q, kp, vp, tables, ctx = _host()
    with pytest.raises(ValueError, match="softcap"):
        ops.paged_decode(q, kp, vp, tables, ctx, softcap=softcap)
    with pytest.raises(ValueError, match="softcap"):
        ops.paged_prefill(q, kp, vp, tables, ctx, ctx, ctx, 1, softcap=softcap)


@gpu
def test_caps_beyond_float32_are_none(cuda):
    q, kp, vp, tables, ctx = (t.to(cuda) for t in _host())
    q, kp, ctx = torch.randn_like(q), torch.randn_like(kp), ctx + 20
    tables[:] = torch.arange(4, device=cuda).reshape(2, 2)
    vp = torch.randn_like(vp)
    slopes = torch.zeros(8, device=cuda)
    a, b = (ops.paged_decode(q, kp, vp, tables, ctx, softcap=c, alibi_slopes=slopes)
            for c in (1e300, 0.0))
    ops.check_device_errors(0)
    assert torch.equal(a, b)

"""Step metadata on the GPU (ops.paged_plan / mz_paged_plan) against a walk over
the sequences on the host, with the block order of BlockManager.allocate.  All
outputs are whole numbers and must be equal."""
import ctypes
import random

import pytest
import torch

from mlxz_b200 import _native, ops
from mlxz_b200._native import DeviceError
from mlxz_b200.paged_attention import BlockManager

gpu = pytest.mark.gpu


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _host_plan(bm, tables, ctx, q, held, bs, n_rows):
    """The same step on the host: tables grow through the BlockManager."""
    tables = [list(t) for t in tables]
    q_start, positions, slots, new = [], [], [], []
    for b, (c, n) in enumerate(zip(ctx, q)):
        need = max(0, -(-(c + n) // bs) - held[b])
        got = bm.allocate(need)
        new += got
        tables[b] += got
        q_start.append(len(positions))
        for pos in range(c, c + n):
            positions.append(pos)
            slots.append(tables[b][pos // bs] * bs + pos % bs)
    pad = n_rows - len(positions)
    return tables, q_start, positions + [0] * pad, slots + [-1] * pad, new


def _case(seed, ctx, q, bs, slack=0, extra=0):
    """Random tables (``extra`` blocks beyond need held) from one BlockManager."""
    r = random.Random(seed)
    held = [-(-c // bs) + (r.randint(0, extra) if extra else 0) for c in ctx]
    need = sum(max(0, -(-(c + n) // bs) - h) for c, n, h in zip(ctx, q, held))
    bm = BlockManager(sum(held) + need + slack + 1, bs)
    r.shuffle(bm._free_list)
    tables = [bm.allocate(h) for h in held]
    return bm, tables, held


def _dev_tables(tables, width, dev):
    t = torch.full((len(tables), width), -1, dtype=torch.int32)
    for i, row in enumerate(tables):
        t[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
    return t.to(dev)


def _check(dev, ctx, q, bs, pad=0, extra=0, give_held=True, seed=0):
    bm, tables, held = _case(seed, ctx, q, bs, extra=extra)
    n_blocks = bm.total_blocks
    n_rows = sum(q) + pad
    width = max([1] + [max(h, -(-(c + n) // bs)) for c, n, h in zip(ctx, q, held)]) + 1
    t_dev = _dev_tables(tables, width, dev)
    want_t, want_start, want_pos, want_slots, new = _host_plan(bm, tables, ctx, q, held, bs, n_rows)
    p = ops.paged_plan(t_dev, _i32(ctx, dev), _i32(q, dev), n_rows, bs, n_blocks,
                       new_ids=_i32(new, dev) if new else None,
                       held=_i32(held, dev) if give_held else None)
    torch.cuda.synchronize()
    ops.check_device_errors(0)
    assert torch.equal(t_dev.cpu(), _dev_tables(want_t, width, "cpu"))
    assert p.q_start.tolist() == want_start
    assert p.positions.tolist() == want_pos
    assert p.slots.tolist() == want_slots
    assert p.lengths.tolist() == [c + n for c, n in zip(ctx, q)]
    assert p.held.tolist() == [len(t) for t in want_t]
    assert p.n_new.tolist() == [len(new)]


CASES = [
    # ctx, q, bs
    ([0], [1], 16),
    ([0], [0], 16),
    ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1], 16),
    ([5, 0, 100, 7], [0, 40, 0, 3], 16),
    ([0, 0, 0], [1023, 1, 1025], 16),        # sequences that start at the 1024-row boundary
    ([3, 0, 9], [1024, 1024, 1], 48),
    ([0], [5000], 64),                       # one sequence over several blocks of rows
    ([7, 1], [2, 3], 1),                     # one token per block
    ([1000, 2, 77], [1, 64, 13], 128),
]


@gpu
@pytest.mark.parametrize("ctx,q,bs", CASES)
@pytest.mark.parametrize("pad", [0, 3])
def test_plan_matches_host(cuda, ctx, q, bs, pad):
    _check(cuda, ctx, q, bs, pad=pad)


@gpu
def test_plan_default_held_and_spare_blocks(cuda):
    _check(cuda, [15, 16, 0, 40], [1, 1, 20, 0], 16, give_held=False)
    # tables that hold more blocks than their tokens need
    _check(cuda, [15, 16, 0, 40], [1, 33, 20, 9], 16, extra=3, seed=4)


@gpu
@pytest.mark.parametrize("B", [2047, 2048, 2049, 5000])
def test_plan_many_sequences(cuda, B):
    """More sequences than one round of the scan; runs of empty ones."""
    r = random.Random(B)
    q = [r.choice([0, 0, 1, 1, 1, 7]) for _ in range(B)]
    q[B // 3:B // 2] = [0] * (B // 2 - B // 3)
    _check(cuda, [r.randint(0, 50) for _ in range(B)], q, 16, pad=5, seed=B)


@gpu
@pytest.mark.parametrize("seed", range(6))
def test_plan_random(cuda, seed):
    r = random.Random(seed)
    B = r.randint(1, 300)
    top = r.choice([1, 5, 200, 1500])
    _check(cuda, [r.randint(0, 600) for _ in range(B)], [r.randint(0, top) for _ in range(B)],
           r.choice([16, 32, 48]), pad=r.randint(0, 2000), extra=r.randint(0, 2), seed=seed)


@gpu
def test_plan_no_rows_and_no_sequences(cuda):
    _check(cuda, [3, 0], [0, 0], 16)
    p = ops.paged_plan(torch.empty(0, 4, dtype=torch.int32, device=cuda), _i32([], cuda),
                       _i32([], cuda), 5, 16, 9)
    assert p.slots.tolist() == [-1] * 5 and p.positions.tolist() == [0] * 5
    assert p.n_new.tolist() == [0] and p.q_start.numel() == 0


@gpu
def test_plan_in_a_graph_and_on_a_side_stream(cuda):
    """A captured plan follows lengths that change in place between replays."""
    bs, B = 16, 3
    tables = torch.full((B, 8), -1, dtype=torch.int32, device=cuda)
    ids = torch.arange(20, dtype=torch.int32, device=cuda)
    ctx, q = _i32([0, 0, 0], cuda), _i32([20, 1, 3], cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.paged_plan(tables, ctx, q, 32, bs, 20, new_ids=ids)
        with torch.cuda.graph(g, stream=side):
            p = ops.paged_plan(tables, ctx, q, 32, bs, 20, new_ids=ids)
    torch.cuda.current_stream().wait_stream(side)
    q.copy_(_i32([1, 17, 2], cuda))
    tables.fill_(-1)
    g.replay()
    torch.cuda.synchronize()
    assert tables[:, :2].tolist() == [[0, -1], [1, 2], [3, -1]]
    assert p.slots[:20].tolist() == [0] + list(range(16, 33)) + [48, 49]
    assert p.slots[20:].tolist() == [-1] * 12
    ops.check_device_errors(0)


@gpu
def test_plan_reports_bad_lengths_and_ids(cuda):
    def run(ctx, q, n_rows, ids, held=None, tables=None, n_blocks=8):
        t = tables if tables is not None else torch.full((len(ctx), 4), -1, dtype=torch.int32)
        t = t.to(cuda)
        p = ops.paged_plan(t, _i32(ctx, cuda), _i32(q, cuda), n_rows, 16, n_blocks,
                           new_ids=_i32(ids, cuda), held=None if held is None else _i32(held, cuda))
        torch.cuda.synchronize()
        return t.cpu(), p

    def raises(text):
        with pytest.raises(DeviceError, match=text):
            ops.check_device_errors(0)

    # beyond the table (4 blocks of 16), negative, and a table short of its tokens
    for ctx, q, held in (([60], [5], None), ([-1], [1], None), ([0], [-2], None), ([20], [1], [1])):
        t, p = run(ctx + [0], q + [1], 8, [3, 4], held=None if held is None else held + [0])
        raises("context length")
        # the sequence behind it is planned as if the bad one brought nothing
        assert p.q_start.tolist() == [0, 0] and p.slots[0].item() == 3 * 16
        assert p.lengths[0].item() == ctx[0] and t[1, 0].item() == 3
    # more rows than given: the sequence that does not fit gets none
    t, p = run([0, 0], [3, 6], 8, [1, 2])
    raises("rows")
    assert p.slots.tolist() == [16, 17, 18, -1, -1, -1, -1, -1] and p.lengths.tolist() == [3, 0]
    # new ids run out: the first block is there, the second's slots are skipped
    t, p = run([0], [20], 20, [5])
    raises("new blocks")
    assert t[0].tolist() == [5, -1, -1, -1]
    assert p.slots.tolist() == list(range(80, 96)) + [-1] * 4
    assert p.n_new.item() == 2 and p.held.item() == 1
    # ids outside the pool, new and held
    t, p = run([0], [1], 1, [8])
    raises("block id")
    assert p.slots.item() == -1
    t, p = run([1], [1], 1, [0], tables=torch.tensor([[99, -1, -1, -1]], dtype=torch.int32))
    raises("block id")
    assert p.slots.item() == -1


def test_plan_refusals_on_the_host():
    t = torch.zeros(2, 4, dtype=torch.int32)
    v = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_plan(t, v, v, 4, 16, 8)
    with pytest.raises(ValueError, match="max_blocks"):
        ops.paged_plan(v, v, v, 4, 16, 8)
    with pytest.raises(ValueError, match="ctx_lens"):
        ops.paged_plan(t, v.long(), v, 4, 16, 8)
    with pytest.raises(ValueError, match="q_lens"):
        ops.paged_plan(t, v, v[:1], 4, 16, 8)
    with pytest.raises(ValueError, match="held"):
        ops.paged_plan(t, v, v, 4, 16, 8, held=v[:1])
    with pytest.raises(ValueError, match="n_rows"):
        ops.paged_plan(t, v, v, -1, 16, 8)
    with pytest.raises(ValueError, match="max_blocks"):
        ops.paged_plan(t[:, :0], v, v, 4, 16, 8)


def test_plan_c_abi_argument_errors():
    lib = _native.lib()
    p = ctypes.c_void_p(64)  # never read: every call below is refused first

    def call(width=4, n_new=0, B=2, rows=4, bs=16, n_blocks=8, tables=p, n_used=p, slots=p):
        return lib.mz_paged_plan(tables, width, p, p, None, None, n_new, B, rows, bs, n_blocks, p,
                                 p, slots, p, p, n_used, None, None)

    for kw in (dict(width=0), dict(B=-1), dict(rows=-1), dict(bs=0), dict(n_blocks=0),
               dict(tables=None), dict(n_used=None), dict(slots=None), dict(n_new=3)):
        assert call(**kw) == _native.MZ_ERR_INVALID_ARG, kw
    assert call(width=1 << 28, bs=16) == _native.MZ_ERR_UNSUPPORTED
    assert call(width=1 << 20, B=1 << 12) == _native.MZ_ERR_UNSUPPORTED


# --- entry points by number ----------------------------------------------------------------

def test_packed_calls_refuse_what_is_no_call():
    lib = _native.lib()
    slots = bytes(8 * 64)
    assert lib.mz_call_packed(99, slots, 19) == _native.MZ_ERR_INVALID_ARG
    assert lib.mz_call_packed(-1, slots, 19) == _native.MZ_ERR_INVALID_ARG
    assert "no entry point" in _native.last_error()[1]
    assert lib.mz_call_packed(0, slots, 18) == _native.MZ_ERR_INVALID_ARG
    assert "takes 19 arguments" in _native.last_error()[1]
    assert lib.mz_call_packed(0, None, 19) == _native.MZ_ERR_INVALID_ARG
    wide = [0] * 19
    wide[7] = 1 << 32  # n_seqs is 32 bits wide
    with pytest.raises(ValueError, match="out of its type's range"):
        _native.call_packed("mz_paged_plan", *wide)


@pytest.mark.parametrize("name", sorted(_native._PACKED))
def test_packed_calls_take_their_arguments_in_order(name):
    """Every argument arrives: each changed one by one from a set that is
    refused for its sizes gives the status of the plain call."""
    lib, types = _native.lib(), _native._SIGNATURES[name]
    assert _native._PACKED[name][2] == len(types)
    for i in range(-1, len(types)):
        args = [0.0 if t is ctypes.c_float else 0 for t in types]
        if i >= 0 and types[i] not in (ctypes.c_void_p, ctypes.c_size_t) and \
                not issubclass(types[i], ctypes._Pointer):
            args[i] = -3
        # pointers stay null and sizes 0 or below: nothing can be launched
        plain = getattr(lib, name)(*[None if a == 0 and issubclass(
            t, (ctypes.c_void_p, ctypes._Pointer)) else max(a, 0) if t is ctypes.c_uint32 else a
            for a, t in zip(args, types)])
        said = _native.last_error()
        args = [max(a, 0) if t is ctypes.c_uint32 else a for a, t in zip(args, types)]
        op, pack, n = _native._PACKED[name]
        assert lib.mz_call_packed(op, pack(*args), n) == plain != 0
        assert _native.last_error() == said

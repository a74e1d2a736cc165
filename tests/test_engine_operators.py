"""The operators together, as a server runs them: step metadata, norm and
rotation with the append, masked attention of prompt chunks, then decode steps
whose tables grow on the GPU, eagerly and from a captured graph."""
import numpy as np
import pytest
import torch

from mlxz_b200 import ops
from mlxz_b200.engine import (PagedDecodeStep, PagedKVStore, PagedPrefillStep, QKNormRope,
                              QuantizedPagedDecodeStep, QuantizedPagedKVStore)
from mlxz_b200.engine.sharding import PeerAllGather
from oracle import rng
from oracle import score_mod as osm
from tests.gpu_util import to_bits, to_dev

gpu = pytest.mark.gpu
L, HKV, G, D, BS, DT = 2, 2, 4, 128, 16, "bf16"
HQ = HKV * G


def _ropes(cuda, axes=None):
    inv = 10000.0 ** (-torch.arange(D // 2, device=cuda, dtype=torch.float32) / (D // 2))
    out = []
    for l in range(L):
        w = [(1 + 0.2 * torch.randn(D, generator=torch.Generator().manual_seed(10 * l + i)))
             .to(torch.bfloat16).to(cuda) for i in range(2)]
        out.append(QKNormRope(inv, w[0], w[1], eps=1e-6, interleaved=l == 1, freq_axes=axes))
    return out


def _tokens(n, seed):
    """Projected q, k, v of n tokens of every layer (bits)."""
    return [rng.normal(seed, (L, n, h, D), DT, stream=i) for i, h in enumerate((HQ, HKV, HKV))]


def _reference(ropes, toks, l, pos_from, cuda, positions=None, **mod):
    """Attention of tokens pos_from.. over the whole sequence, from the turned
    heads of the operator (tested by itself) in 64 bits."""
    q, k, v = (to_dev(t[l], DT, cuda) for t in toks)
    n = q.shape[0]
    pos = torch.arange(n, dtype=torch.int32, device=cuda) if positions is None else positions
    q, k = ropes[l].apply(q, k, pos)
    f = [rng.to_f32(to_bits(x), DT).transpose(1, 0, 2) for x in (q, k, v)]
    o, s = osm.attention(f[0][:, pos_from:], f[1], f[2], np.arange(pos_from, n), D ** -0.5, **mod)
    return o.transpose(1, 0, 2), s.transpose(1, 0, 2), to_bits(k)


def _check(out, ref, spread):
    """The attention tests' tolerance: bf16 store and 2^-10 of the spread."""
    o = out.float().cpu().numpy().astype(np.float64)
    assert (np.abs(o - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -10 * spread).all()


@gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("mod", [{}, dict(window=40, sink_tokens=4), dict(softcap=20.0)])
def test_prompt_chunks_then_decode(cuda, graph, mod):
    prompts, steps = {"a": 90, "b": 17, "c": 47}, 20
    omod = {("sink" if k == "sink_tokens" else k): v for k, v in mod.items()}
    ropes = _ropes(cuda)
    store = PagedKVStore(L, 64, HKV, D, BS, torch.bfloat16, cuda)
    toks = {s: _tokens(n + steps, 100 + i) for i, (s, n) in enumerate(prompts.items())}
    for s in prompts:
        store.add_sequence(s)
    done = dict.fromkeys(prompts, 0)
    while any(done[s] < n for s, n in prompts.items()):
        chunks = [(s, min(33, n - done[s])) for s, n in prompts.items()]
        step = PagedPrefillStep(store, chunks, HQ, rope=ropes, **mod)
        for l in range(L):
            q, k, v = (to_dev(np.concatenate([toks[s][i][l, done[s]:done[s] + n]
                                              for s, n in chunks]), DT, cuda) for i in range(3))
            out = step.layer(l, q, k, v)
            row = 0
            for s, n in chunks:
                part = [t[:, :done[s] + n] for t in toks[s]]
                if n:
                    o, sp, _ = _reference(ropes, part, l, done[s], cuda, **omod)
                    _check(out[row:row + n], o, sp)
                row += n
        step.finish()
        for s, n in chunks:
            done[s] += n
    ids = list(prompts)
    dec = PagedDecodeStep(store, ids, HQ, max_blocks=8, rope=ropes, **mod)
    if graph:
        dec.capture()
    for t in range(steps):
        q, k, v = (to_dev(np.stack([toks[s][i][:, prompts[s] + t] for s in ids], 1), DT, cuda)
                   for i in range(3))
        out = dec.replay(q, k, v) if graph else dec.step(q, k, v)
        for l in range(L):
            for b, s in enumerate(ids):
                p = prompts[s] + t
                o, sp, kb = _reference(ropes, [x[:, :p + 1] for x in toks[s]], l, p, cuda, **omod)
                _check(out[l, b:b + 1], o, sp)
        dec.advance()
        # the device's tables are the host's
        for b, s in enumerate(ids):
            tb = store.tables[s]
            assert dec.tables[b].tolist() == tb + [-1] * (8 - len(tb))
        assert dec.positions.tolist() == [store.offsets[s] for s in ids]
        assert dec.lengths.tolist() == [store.offsets[s] + 1 for s in ids]
    # the cache holds the turned keys, bit for bit
    for s in ids:
        n = prompts[s] + steps
        _, _, kb = _reference(ropes, toks[s], 0, n - 1, cuda)
        tb = torch.tensor(store.tables[s], device=cuda)
        got = store.pools[0, 0][tb].transpose(1, 2).reshape(-1, HKV, D)[:n]
        assert np.array_equal(to_bits(got), kb)
    torch.cuda.synchronize()
    ops.check_device_errors(0)


@gpu
def test_image_positions_prefix_and_documents(cuda):
    """Three position axes for an image prefix that all tokens see, and packed
    documents behind it."""
    n, pre = 80, 24
    axes = (torch.arange(D // 2) % 3).int().to(cuda)
    ropes = _ropes(cuda, axes)
    pos = torch.arange(n, dtype=torch.int32).repeat(3, 1)
    pos[0, :pre], pos[1, :pre] = 3, torch.arange(pre, dtype=torch.int32) // 6
    pos[2, :pre] = torch.arange(pre, dtype=torch.int32) % 6
    pos = pos.to(cuda)
    first = torch.tensor([0] * 50 + [50] * 30, dtype=torch.int32)
    toks = _tokens(n, 7)
    store = PagedKVStore(L, 8, HKV, D, BS, torch.bfloat16, cuda)
    store.add_sequence("x")
    step = PagedPrefillStep(store, [("x", n)], HQ, rope=ropes, rope_positions=pos,
                            prefix_lens=[pre], first_keys=first.to(cuda))
    for l in range(L):
        out = step.layer(l, *(to_dev(t[l], DT, cuda) for t in toks))
        o, sp, _ = _reference(ropes, toks, l, 0, cuda, positions=pos, prefix=pre,
                              first=first.numpy())
        _check(out, o, sp)
    ops.check_device_errors(0)


@gpu
def test_quantised_store_with_rope_and_window(cuda):
    """Over a quantised store the turned keys are quantised: the same codes as
    from heads turned beforehand, and the same attention bytes."""
    n = 50
    ropes, toks = _ropes(cuda), _tokens(n + 1, 9)
    outs, codes = [], []
    for ahead in (False, True):
        store = QuantizedPagedKVStore(L, 8, HKV, D, BS, 8, device=cuda)
        store.add_sequence("x")
        pos = torch.arange(n + 1, dtype=torch.int32, device=cuda)
        step = PagedPrefillStep(store, [("x", n)], HQ, rope=None if ahead else ropes, window=16,
                                sink_tokens=2)
        got = []
        for l in range(L):
            q, k, v = (to_dev(t[l, :n], DT, cuda) for t in toks)
            if ahead:
                q, k = ropes[l].apply(q, k, pos[:n])
            got.append(step.layer(l, q, k, v))
        step.finish()
        dec = QuantizedPagedDecodeStep(store, ["x"], HQ, rope=None if ahead else ropes)
        q, k, v = (to_dev(t[:, n:], DT, cuda) for t in toks)
        if ahead:
            q, k = (torch.stack(x) for x in zip(*(ropes[l].apply(q[l], k[l], pos[n:])
                                                  for l in range(L))))
        got.append(dec.step(q, k, v))
        outs.append(got)
        codes.append(store.codes.clone())
    assert torch.equal(codes[0], codes[1])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    ops.check_device_errors(0)


@gpu
def test_advance_with_blocks_from_outside_and_outgrown_tables(cuda):
    """Blocks that a table got between steps go up with the whole tables; a
    table wider than the step is refused as before."""
    store = PagedKVStore(1, 32, HKV, D, BS, torch.bfloat16, cuda)
    store.add_sequence("a", 15)
    store.add_sequence("b", 40)
    step = PagedDecodeStep(store, ["a", "b"], HQ, max_blocks=4)
    store.ensure_capacity("b", 20)  # a fourth block, unknown to the device
    step.advance()                  # "a" grows
    for i, s in enumerate(("a", "b")):
        tb = store.tables[s]
        assert step.tables[i].tolist() == tb + [-1] * (4 - len(tb))
    with pytest.raises(ValueError, match="outgrew"):
        for _ in range(30):
            step.advance()


@gpu
def test_advance_with_offsets_from_outside(cuda):
    """Offsets that moved between steps go up with the next block."""
    store = PagedKVStore(1, 32, HKV, D, BS, torch.bfloat16, cuda)
    store.add_sequence("a", 15)
    store.add_sequence("b", 3)
    step = PagedDecodeStep(store, ["a", "b"], HQ, max_blocks=4)
    store.offsets["b"] += 4
    step.advance()  # "a" grows
    assert step.positions.tolist() == [16, 8] and step.lengths.tolist() == [17, 9]
    for i, s in enumerate(("a", "b")):
        tb = store.tables[s]
        assert step.tables[i].tolist() == tb + [-1] * (4 - len(tb))

@gpu
def test_advance_with_blocks_exchanged_from_outside(cuda):
    """Blocks that were exchanged between steps (a copy on write by another
    path, a request put in another's place) go up with the next block."""
    store = PagedKVStore(1, 64, HKV, D, BS, torch.bfloat16, cuda)
    store.add_sequence("a", 14)
    store.add_sequence("b", 40)
    step = PagedDecodeStep(store, ["a", "b"], HQ, max_blocks=4)
    store.tables["b"][1] = store.bm.allocate(1)[0]

    def same():
        for i, s in enumerate(("a", "b")):
            tb = store.tables[s]
            assert step.tables[i].tolist() == tb + [-1] * (4 - len(tb))
        assert step.positions.tolist() == [store.offsets[s] for s in ("a", "b")]

    step.advance()
    step.advance()  # "a" grows
    assert len(store.tables["a"]) == 2
    same()
    store.free_sequence("b")
    store.bm.allocate(1)
    store.add_sequence("b", 42)  # as many tokens in as many blocks, but others
    while store.offsets["b"] < 48:
        step.advance()  # "b" grows
    assert len(store.tables["b"]) == 4
    same()
    torch.cuda.synchronize()
    ops.check_device_errors(0)

@gpu
def test_prefill_metadata_is_done_when_the_step_is_made(cuda, monkeypatch):
    """A step made on one stream may run its layers on another at once: what it
    holds on the device is complete, like the uploads of its tables."""
    plan = ops.paged_plan

    def late(*args, **kw):
        torch.cuda._sleep(200_000_000)  # about 0.1 s ahead of the launch
        return plan(*args, **kw)

    store = PagedKVStore(1, 8, HKV, D, BS, torch.bfloat16, cuda)
    store.add_sequence("x")
    made = torch.cuda.Stream()
    with torch.cuda.stream(made):
        PagedPrefillStep(store, [("x", 40)], HQ)  # the kernel's first launch may wait by itself
        monkeypatch.setattr(ops, "paged_plan", late)
        step = PagedPrefillStep(store, [("x", 40)], HQ)
        assert made.query()
    q, k, v = (to_dev(t[0], DT, cuda) for t in _tokens(40, 3))
    out = step.layer(0, q, k, v)
    ops.check_device_errors(0)
    f = [rng.to_f32(to_bits(x), DT).transpose(1, 0, 2) for x in (q, k, v)]
    o, sp = osm.attention(*f, np.arange(40), D ** -0.5)
    _check(out, o.transpose(1, 0, 2), sp.transpose(1, 0, 2))


def test_fused_all_gather_takes_plain_steps_only():
    class Step:
        plain = False

    with pytest.raises(ValueError, match="plain"):
        PeerAllGather.launch(object.__new__(PeerAllGather), Step(), 0, None, None, None)


def test_one_rope_or_one_per_layer():
    from mlxz_b200.engine.qk_rope import per_layer

    r = QKNormRope(torch.ones(4))
    assert per_layer(None, 3) == [None] * 3 and per_layer(r, 2) == [r, r]
    assert per_layer([r, r], 2) == [r, r]
    with pytest.raises(ValueError, match="per layer"):
        per_layer([r], 2)

"""Cases of the serving operators around the paged KV cache, with their plain forms.

Four operators, in the order in which a step of a server runs them:

  plan     block tables, slot maps and positions of a step, built on the GPU from the
           requests' lengths (``ops.paged_plan``);
  rope     RMS norm of every query and key head, the rotation by position (one position
           axis or several) and, with pools given, the write of K and V to their slots
           (``ops.qk_norm_rope``, ``ops.qk_norm_rope_append``);
  prefill  attention of chunks of new tokens over the paged cache with capped scores, a bias
           by distance, a sliding window with sink tokens, a prefix mask and a document mask
           (``ops.paged_prefill`` with those arguments);
  decode   the same for single tokens and for short runs of drafted tokens
           (``ops.paged_decode`` with those arguments).

``run`` computes them in elementary torch operations in 32 bits (angles in 64), or, where
``own`` is true, by the framework's calls.  Lengths follow from a case alone (its ``lens`` is
the seed of their pattern); values follow from ``prepare``'s seed.
"""
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --- cases -------------------------------------------------------------------------------------

def _attn(name, op, dtype, B, q, ctx_lo, ctx_hi, Hq=32, Hkv=8, D=128, bs=16, ragged=True,
          softcap=0.0, slopes=False, window=0, sink=0, prefix=0, docs=0, lens=1):
    return {"name": name, "op": op, "dtype": dtype, "B": B, "q": q, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "Hq": Hq, "Hkv": Hkv, "D": D, "bs": bs, "ragged": ragged,
            "softcap": softcap, "slopes": slopes, "window": window, "sink": sink,
            "prefix": prefix, "docs": docs, "lens": lens}


def _rope(name, dtype, T, Hq=32, Hkv=8, D=128, rot=128, axes=1, paired=False, norm=True,
          append=True, far=8192, bs=16):
    return {"name": name, "op": "rope", "dtype": dtype, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D,
            "rot": rot, "axes": axes, "paired": paired, "norm": norm, "append": append,
            "far": far, "bs": bs}


def _plan(name, B, q_lo, q_hi, ctx_hi, bs=16, pad=0, lens=1):
    return {"name": name, "op": "plan", "B": B, "q_lo": q_lo, "q_hi": q_hi, "ctx_hi": ctx_hi,
            "bs": bs, "pad": pad, "lens": lens}


def listed():
    return [
        # the metadata of one decode step of 64 live requests: one new token each
        _plan("plan-step-64", B=64, q_lo=1, q_hi=1, ctx_hi=8192),
        # a step that admits 256 ragged prompts, some empty, padded to a fixed row count
        _plan("plan-prompts-256", B=256, q_lo=0, q_hi=1024, ctx_hi=4096, pad=333),
        # queries, keys and values of one decode step of 64 requests, written to the cache
        _rope("rope-step-64", "bf16", T=64),
        # one layer of a 16384-token prompt step, written to the cache
        _rope("rope-prompt-16k", "bf16", T=16384),
        # text, image and video tokens with (time, height, width) positions, adjacent pairs,
        # keys returned dense, far positions, an odd token count
        _rope("rope-three-axes", "f16", T=8191, D=64, rot=64, axes=3, paired=True, append=False,
              far=1_000_000),
        # eight 512-token chunks at offset 3584 with scores capped at 50
        _attn("prefill-softcap", "prefill", "bf16", B=8, q=512, ctx_lo=4096, ctx_hi=4096,
              ragged=False, softcap=50.0),
        # a 4096-token chunk late in a long prompt, sliding window with sink tokens
        _attn("prefill-window", "prefill", "bf16", B=1, q=4096, ctx_lo=16384, ctx_hi=16384,
              ragged=False, window=4096, sink=4),
        # small ragged prompts with a bias by distance
        _attn("prefill-slopes", "prefill", "f16", B=5, q=333, ctx_lo=37, ctx_hi=700, D=64,
              slopes=True, lens=3),
        # packed documents behind a shared prefix that every token sees both ways
        _attn("prefill-documents", "prefill", "bf16", B=4, q=1500, ctx_lo=1500, ctx_hi=2100,
              prefix=257, docs=400, lens=4),
        # one decode step, 64 requests of 512 to 8192 tokens: capped scores in a window with sinks
        _attn("decode-window", "decode", "bf16", B=64, q=1, ctx_lo=512, ctx_hi=8192,
              softcap=50.0, window=4096, sink=4, lens=5),
        # the smallest step: four short requests, a bias by distance
        _attn("decode-slopes", "decode", "f16", B=4, q=1, ctx_lo=37, ctx_hi=511, D=64,
              slopes=True, lens=6),
        # four drafted tokens of 32 requests scored over their caches, causally
        _attn("decode-drafts", "decode", "bf16", B=32, q=4, ctx_lo=512, ctx_hi=8192, lens=7),
    ]


def _log(rng, lo, hi):
    """A whole number, spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "rope", "prefill", "prefill", "decode", "decode"])
    if op == "plan":
        B = _log(rng, 1, 1024)
        top = max(1, min(2048, 131072 // B))
        q_hi = rng.choice([1, _log(rng, 1, top)])
        c = _plan("", B, rng.choice([0, 1]) if q_hi > 1 else 1, q_hi, _log(rng, 1, 8192),
                  bs=rng.choice([16, 32, 64]), pad=rng.choice([0, _log(rng, 1, 200)]),
                  lens=rng.randrange(1 << 20))
    elif op == "rope":
        D = rng.choice([64, 128, 128])
        c = _rope("", rng.choice(["bf16", "f16", "f32"]), _log(rng, 1, 8192),
                  Hq=rng.choice([8, 32]), Hkv=rng.choice([1, 4, 8]), D=D,
                  rot=rng.choice([D, D, D // 2]), axes=rng.choice([1, 1, 3]),
                  paired=rng.random() < 0.4, norm=rng.random() < 0.8,
                  append=rng.random() < 0.6, far=_log(rng, 512, 1_000_000),
                  bs=rng.choice([16, 32]))
    else:
        Hkv = rng.choice([1, 2, 4, 8])
        G = rng.choice([1, 2, 4])
        few = op == "decode"
        q = rng.choice([1, 1, rng.randint(2, 4)]) if few else _log(rng, 1, 2048)
        lo = _log(rng, 16, 512)
        c = _attn("", op, rng.choice(["bf16", "f16"]), _log(rng, 1, 64 if few else 8), q,
                  max(lo, q), max(lo, q) + _log(rng, 1, 7168), Hq=Hkv * G, Hkv=Hkv,
                  D=rng.choice([64, 128]), bs=rng.choice([16, 32, 64]),
                  ragged=rng.random() < 0.8, softcap=rng.choice([0.0, 20.0, 50.0]),
                  slopes=rng.random() < 0.4, lens=rng.randrange(1 << 20))
        if rng.random() < 0.5:
            c["window"] = _log(rng, 8, 4096)
            c["sink"] = rng.choice([0, 4])
        if rng.random() < 0.3:
            c["docs"] = _log(rng, 50, 1000)
        if not few and rng.random() < 0.3:
            c["prefix"] = _log(rng, 5, 500)
        if not few and not (c["window"] or c["docs"] or c["prefix"] or c["softcap"]):
            c["slopes"] = True
    del c["name"]
    return c


# --- lengths: from the case alone -----------------------------------------------------------------

def _plan_lens(c):
    r = random.Random(c["lens"])
    q = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["B"])]
    if sum(q) == 0:
        q[0] = 1
    ctx = [r.randint(0, c["ctx_hi"]) for _ in range(c["B"])]
    return q, ctx


def _attn_lens(c):
    """New tokens and tokens in the cache (the new ones among them) of every request."""
    r = random.Random(c["lens"])
    q, ctx = [], []
    for b in range(c["B"]):
        n = c["q"]
        if c["ragged"] and c["op"] == "prefill" and b:
            n = r.randint(1, c["q"])
        t = r.randint(c["ctx_lo"], c["ctx_hi"]) if c["ragged"] else c["ctx_hi"]
        q.append(n)
        ctx.append(max(t, n))
    return q, ctx


def _doc_starts(c, length):
    """First position of the document that each position of a packed request belongs to."""
    starts = np.arange(0, length, c["docs"])
    return starts[np.searchsorted(starts, np.arange(length), side="right") - 1]


def _row_limits(c, n, t):
    """Per new token of a request of t tokens: how many keys from the first on it sees in any
    case, and the first and one past the last key of the range that it sees besides."""
    p = np.arange(t - n, t)
    lo = _doc_starts(c, t)[p] if c["docs"] else np.zeros(n, dtype=np.int64)
    if c["window"]:
        lo = np.maximum(lo, p - c["window"] + 1)
    return np.maximum(min(c["prefix"], t), np.minimum(c["sink"], p + 1)), lo, p + 1


# --- work: what a pass cannot do without ------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "plan":
        q, ctx = _plan_lens(c)
        bs, rows = c["bs"], sum(q) + c["pad"]
        blocks = sum(-(-(n + t) // bs) - t // bs for n, t in zip(q, ctx) if n)
        fresh = sum(-(-(n + t) // bs) - -(-t // bs) for n, t in zip(q, ctx))
        # lengths and held counts read; starts, lengths, held written; positions, slots written
        return {"bytes": 24 * c["B"] + 12 * rows + 4 * blocks + 4 * fresh, "flops": 0}
    if c["op"] == "rope":
        es = 4 if c["dtype"] == "f32" else 2
        heads = c["Hq"] + c["Hkv"]
        moved = 2 * c["T"] * (heads + (c["Hkv"] if c["append"] else 0)) * c["D"] * es
        return {"bytes": moved + c["T"] * (4 * c["axes"] + (8 if c["append"] else 0)),
                "flops": c["T"] * heads * (4 * c["D"] + 3 * c["rot"])}
    pairs, keys, rows = 0, 0, 0
    for n, t in zip(*_attn_lens(c)):
        head, lo, hi = _row_limits(c, n, t)
        lo = np.maximum(lo, head)
        pairs += int((head + np.maximum(hi - lo, 0)).sum())
        keys += int(head.max() + max(0, hi.max() - max(lo.min(), head.max())))
        rows += n
    return {"bytes": 4 * rows * c["Hq"] * c["D"] + 4 * keys * c["Hkv"] * c["D"],
            "flops": 4 * pairs * c["Hq"] * c["D"]}


# --- inputs -----------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).to("cuda")


def _tables(g, counts, width, n_blocks):
    """Block tables of `counts` blocks each, drawn without repetition, -1 behind them."""
    perm = torch.randperm(n_blocks, generator=g, device="cuda").int()
    n = _i32(counts)[:, None]
    base = torch.cumsum(n, 0) - n
    j = torch.arange(width, device="cuda")[None, :]
    at = (base + j).clamp(max=n_blocks - 1)
    return torch.where(j < n, perm[at], -1).int(), perm[int(sum(counts)):]


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] == "plan":
        q, ctx = _plan_lens(c)
        bs = c["bs"]
        held = [-(-t // bs) for t in ctx]
        fresh = sum(-(-(n + t) // bs) - h for n, t, h in zip(q, ctx, held))
        width = max(-(-(n + t) // bs) for n, t in zip(q, ctx)) + 2
        s["n_blocks"] = int((sum(held) + fresh) * 1.1) + 2
        s["tables"], rest = _tables(g, held, width, s["n_blocks"])
        s["new_ids"] = rest[:max(1, fresh)].contiguous()
        s["held"], s["ctx"], s["q"] = _i32(held), _i32(ctx), _i32(q)
        s["rows"] = sum(q) + c["pad"]
        return s
    dt = DTYPES[c["dtype"]]
    if c["op"] == "rope":
        T, Hq, Hkv, D, bs = c["T"], c["Hq"], c["Hkv"], c["D"], c["bs"]
        # the projection's output: queries, keys and values side by side
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device="cuda").to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        pos = torch.randint(0, c["far"], (c["axes"], T), generator=g, device="cuda").int()
        s["pos"] = pos if c["axes"] > 1 else pos[0]
        half = c["rot"] // 2
        s["inv_freq"] = 500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float32) / half)
        s["freq_axes"] = (torch.arange(half, device="cuda") * c["axes"] // half).int() \
            if c["axes"] > 1 else None
        s["qw"] = s["kw"] = None
        if c["norm"]:
            s["qw"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dt)
            s["kw"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dt)
        s["eps"] = 1e-6 if c["norm"] else None
        if c["append"]:
            blocks = -(-T // bs)
            n = int(blocks * 1.1) + 2
            ids = torch.randperm(n, generator=g, device="cuda")[:blocks]
            t = torch.arange(T, device="cuda")
            s["slots"] = ids[t // bs] * bs + t % bs
            s["k_pool"] = torch.zeros(n, Hkv, bs, D, dtype=dt, device="cuda")
            s["v_pool"] = torch.zeros(n, Hkv, bs, D, dtype=dt, device="cuda")
        return s
    q, ctx = _attn_lens(c)
    bs, D = c["bs"], c["D"]
    counts = [-(-t // bs) for t in ctx]
    n_blocks = int(sum(counts) * 1.1) + 2
    s["tables"], _ = _tables(g, counts, max(counts), n_blocks)
    shape = (n_blocks, c["Hkv"], bs, D)
    s["k_pool"] = torch.randn(shape, generator=g, device="cuda", dtype=dt)
    s["v_pool"] = torch.randn(shape, generator=g, device="cuda", dtype=dt)
    rows = sum(q)
    # capped scores only matter where some come near the cap
    wide = 4.0 if c["softcap"] else 1.0
    x = (wide * torch.randn(rows, c["Hq"], D, generator=g, device="cuda")).to(dt)
    s["x"] = x.view(c["B"], c["q"], c["Hq"], D) if c["op"] == "decode" else x
    if c["op"] == "decode" and c["q"] == 1:
        s["x"] = s["x"][:, 0]
    s["q"], s["ctx"], s["max_q"] = _i32(q), _i32(ctx), max(q)
    s["q_start"] = _i32([sum(q[:b]) for b in range(c["B"])])
    s["slopes"] = s["prefix"] = s["first"] = None
    if c["slopes"]:
        h = torch.arange(c["Hq"], device="cuda", dtype=torch.float32)
        s["slopes"] = 2.0 ** (-8.0 * (h + 1) / c["Hq"])
    if c["prefix"]:
        s["prefix"] = _i32([min(c["prefix"], t) for t in ctx])
    if c["docs"]:
        firsts = [_doc_starts(c, t)[t - n:] for n, t in zip(q, ctx)]
        # a run of drafted tokens is one document: its first token's
        s["first"] = _i32([int(f[0]) for f in firsts] if c["op"] == "decode"
                          else np.concatenate(firsts).tolist())
    return s


# --- one pass ---------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "rope": _own_rope, "prefill": _own_prefill,
                "decode": _own_decode}[op](state)
    return {"plan": _plain_plan, "rope": _plain_rope, "prefill": _plain_prefill,
            "decode": _plain_decode}[op](state)


def _own_plan(s):
    from mlxz_b200 import ops
    p = ops.paged_plan(s["tables"], s["ctx"], s["q"], s["rows"], s["case"]["bs"], s["n_blocks"],
                       new_ids=s["new_ids"], held=s["held"])
    return [s["tables"], p.q_start, p.positions, p.slots, p.lengths, p.held, p.n_new]


def _plain_plan(s):
    bs, tables, ctx, q, held = s["case"]["bs"], s["tables"], s["ctx"], s["q"], s["held"]
    dev = tables.device
    end = ctx + q
    need = ((end + bs - 1) // bs - held).clamp(min=0)
    base = torch.cumsum(need, 0) - need
    j = torch.arange(tables.shape[1], device=dev)[None, :] - held[:, None]
    at = (base[:, None] + j).clamp(0, s["new_ids"].numel() - 1)
    fresh = (j >= 0) & (j < need[:, None])
    tables.copy_(torch.where(fresh, s["new_ids"][at], tables))
    total = torch.cumsum(q, 0)
    start = total - q
    row = torch.arange(s["rows"], device=dev)
    seq = torch.searchsorted(total, row, right=True).clamp(max=q.numel() - 1)
    live = row < total[-1]
    pos = torch.where(live, ctx[seq] + row - start[seq], 0)
    slots = torch.where(live, tables[seq, pos // bs].long() * bs + pos % bs, -1)
    return [tables, start.int(), pos.int(), slots, end, held + need, need.sum(dtype=torch.int32).view(1)]


def _own_rope(s):
    from mlxz_b200 import ops
    kw = dict(q_weight=s["qw"], k_weight=s["kw"], eps=s["eps"], interleaved=s["case"]["paired"],
              freq_axes=s["freq_axes"])
    if not s["case"]["append"]:
        return list(ops.qk_norm_rope(s["q"], s["k"], s["pos"], s["inv_freq"], **kw))
    q = ops.qk_norm_rope_append(s["q"], s["k"], s["v"], s["pos"], s["inv_freq"], s["k_pool"],
                                s["v_pool"], s["slots"], **kw)
    return [q, s["k_pool"], s["v_pool"]]


def _angles(s):
    pos = s["pos"].double()
    pos = pos[s["freq_axes"].long()].t() if s["freq_axes"] is not None else pos[:, None]
    return pos * s["inv_freq"].double()


def _plain_rope(s):
    c = s["case"]
    a = _angles(s)
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    rot = c["rot"]

    def turned(x, w):
        y = x.float()
        if c["norm"]:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * w.float()
        r = y[..., :rot]
        if c["paired"]:
            u, v = r[..., 0::2], r[..., 1::2]
            r = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
        else:
            u, v = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
        return torch.cat([r, y[..., rot:]], -1).to(x.dtype)

    q, k = turned(s["q"], s["qw"]), turned(s["k"], s["kw"])
    if not c["append"]:
        return [q, k]
    blk, at = s["slots"] // c["bs"], s["slots"] % c["bs"]
    s["k_pool"][blk, :, at] = k
    s["v_pool"][blk, :, at] = s["v"]
    return [q, s["k_pool"], s["v_pool"]]


def _own_prefill(s):
    from mlxz_b200 import ops
    c = s["case"]
    return ops.paged_prefill(s["x"], s["k_pool"], s["v_pool"], s["tables"], s["q_start"], s["q"],
                             s["ctx"], s["max_q"], softcap=c["softcap"], alibi_slopes=s["slopes"],
                             window=c["window"], sink_tokens=c["sink"], prefix_lens=s["prefix"],
                             first_keys=s["first"])


def _own_decode(s):
    from mlxz_b200 import ops
    c = s["case"]
    return ops.paged_decode(s["x"], s["k_pool"], s["v_pool"], s["tables"], s["ctx"], causal=True,
                            softcap=c["softcap"], alibi_slopes=s["slopes"], window=c["window"],
                            sink_tokens=c["sink"], first_keys=s["first"])


def _attend(s, q, pos, first):
    """q [B, Q, Hq, D] at positions pos [B, Q] over the paged cache, in 32 bits."""
    c = s["case"]
    B, Q, Hq, D = q.shape
    Hkv, G = c["Hkv"], Hq // c["Hkv"]

    def cached(pool):  # [B, Hkv, S, D]
        t = pool[s["tables"].clamp(min=0).long()].float()
        return t.transpose(1, 2).reshape(B, Hkv, -1, D)

    k = cached(s["k_pool"])
    x = q.float().view(B, Q, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Q, D)
    x = (x @ k.transpose(-1, -2)).view(B, Hkv, G, Q, -1).mul_(D ** -0.5)
    del k
    if c["softcap"]:
        x = x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    t = torch.arange(x.shape[-1], device=q.device)[None, None, :]
    p = pos[:, :, None]
    if c["slopes"]:
        far = (p - t).abs().float()
        x.sub_(s["slopes"].view(1, Hkv, G, 1, 1) * far[:, None, None])
    lo = torch.zeros_like(p)
    if first is not None:
        lo = torch.maximum(lo, first[:, :, None])
    if c["window"]:
        lo = torch.maximum(lo, p - c["window"] + 1)
    seen = (t <= p) & ((t >= lo) | (t < c["sink"]))
    if c["prefix"]:
        seen = seen | (t < s["prefix"][:, None, None])
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top.isinf(), 0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = x.view(B, Hkv, G * Q, -1) @ cached(s["v_pool"])
    o = o.view(B, Hkv, G, Q, D) / torch.where(total == 0, 1, total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, D)


def _plain_prefill(s):
    x, n = s["x"], s["q"]
    T, i = x.shape[0], torch.arange(s["max_q"], device=x.device)[None, :]
    at = (s["q_start"][:, None] + i).clamp(max=T - 1)
    pos = s["ctx"][:, None] - n[:, None] + i
    o = _attend(s, x[at], pos, s["first"][at] if s["first"] is not None else None)
    row = torch.arange(T, device=x.device)
    seq = torch.searchsorted(torch.cumsum(n, 0), row, right=True)
    return o[seq, row - s["q_start"][seq]].to(x.dtype)


def _plain_decode(s):
    x = s["x"]
    q = x[:, None] if x.dim() == 3 else x
    pos = s["ctx"][:, None] - q.shape[1] + torch.arange(q.shape[1], device=x.device)[None, :]
    first = s["first"][:, None].expand(pos.shape) if s["first"] is not None else None
    return _attend(s, q, pos, first).to(x.dtype).view(x.shape)


# --- the definitions in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_rope(s) if case["op"] == "rope" else _exact_attention(s)


def _exact_rope(s):
    c = s["case"]
    T, D, half = c["T"], c["D"], c["rot"] // 2
    pos = s["pos"].double().view(c["axes"], T)
    theta = torch.stack([pos[0 if s["freq_axes"] is None else int(s["freq_axes"][i])]
                         * float(s["inv_freq"][i]) for i in range(half)], -1)
    # complex rotation of the pairs (first, second)
    turn = torch.polar(torch.ones_like(theta), theta)[:, None]
    first = torch.arange(half, device="cuda") * (2 if c["paired"] else 1)
    second = first + (1 if c["paired"] else half)

    def turned(x, w):
        y = x.double()
        if c["norm"]:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / D + s["eps"]) * w.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turned(s["q"], s["qw"]), turned(s["k"], s["kw"])
    if not c["append"]:
        return [q, k]
    pools = []
    for rows in (k, s["v"].double()):
        pool = torch.zeros(s["k_pool"].shape, dtype=torch.float64, device="cuda")
        flat = pool.transpose(1, 2).reshape(-1, c["Hkv"], D)
        flat[s["slots"]] = rows
        pools.append(flat.view(pool.shape[0], c["bs"], c["Hkv"], D).transpose(1, 2).contiguous())
    return [q, *pools]


def _exact_attention(s):
    c = s["case"]
    D, G, bs = c["D"], c["Hq"] // c["Hkv"], c["bs"]
    x = s["x"].reshape(-1, c["Hq"], D)
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, t) in enumerate(zip(*_attn_lens(c))):
        ids = s["tables"][b, :-(-t // bs)].long()
        pos = np.arange(t - n, t)
        lo = np.zeros(n, dtype=np.int64)
        if c["docs"]:
            lo = _doc_starts(c, t)[pos] if c["op"] == "prefill" else \
                np.full(n, _doc_starts(c, t)[pos[0]])
        if c["window"]:
            lo = np.maximum(lo, pos + 1 - c["window"])
        lo, p = (torch.from_numpy(v).to("cuda")[:, None] for v in (lo, pos))
        j = torch.arange(t, device="cuda")[None]
        hidden = ((j > p) | ((j < lo) & (j >= c["sink"]))) & (j >= c["prefix"])
        empty = hidden.all(-1, keepdim=True)
        for h in range(c["Hkv"]):
            k = s["k_pool"][ids, h].reshape(-1, D)[:t].double()
            v = s["v_pool"][ids, h].reshape(-1, D)[:t].double()
            for g in range(h * G, (h + 1) * G):
                a = (x[row:row + n, g].double() @ k.t()) / D ** 0.5
                if c["softcap"]:
                    a = c["softcap"] * torch.tanh(a / c["softcap"])
                if c["slopes"]:
                    a = a - float(s["slopes"][g]) * (p - j).abs()
                a = torch.softmax(a.masked_fill(hidden, float("-inf")), -1)
                out[row:row + n, g] = torch.where(empty, 0.0, a) @ v
        row += n
    return out.view(s["x"].shape)

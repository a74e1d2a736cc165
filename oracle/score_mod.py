"""numpy restatement of attention with modified scores and masks (oracle; test
infrastructure).

The reference's attention call takes a mask and leaves scores to its models
(src/mlxz/paged_attention/attention.py:40-42); the definition is the one of
mz_score_mod: for a token at position p and a key at position t,
x = scale q.k, capped by softcap tanh(x / softcap), minus slope |p - t|; the key
is seen iff t < prefix or (t <= p and (t >= max(first, p - window + 1) or t < sink)).
"""
from __future__ import annotations

import numpy as np

from .paged import gather


def visible(pos: np.ndarray, T: int, window: int = 0, sink: int = 0, prefix: int = 0,
            first: np.ndarray | int = 0) -> np.ndarray:
    """[n, T] truth values: token i (position pos[i]) sees key t."""
    p = np.asarray(pos, dtype=np.int64)[:, None]
    t = np.arange(T)[None, :]
    lo = np.broadcast_to(np.asarray(first, dtype=np.int64).reshape(-1, 1), p.shape)
    if window:
        lo = np.maximum(lo, p - window + 1)
    return (t < prefix) | ((t <= p) & ((t >= lo) | (t < sink)))


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, pos: np.ndarray, scale: float,
              softcap: float = 0.0, slopes: np.ndarray | None = None, window: int = 0,
              sink: int = 0, prefix: int = 0, first: np.ndarray | int = 0
              ) -> tuple[np.ndarray, np.ndarray]:
    """q (Hq, n, D), k / v (Hkv, T, D) floats: (out, spread), both float64
    (Hq, n, D).  ``spread`` is the same weighted sum over |v|: what a relative
    change of the weights can move the output by."""
    Hq, n, D = q.shape
    Hkv, T, _ = k.shape
    G = Hq // Hkv
    out, spread = np.zeros((Hq, n, D)), np.zeros((Hq, n, D))
    if T == 0 or n == 0:
        return out, spread
    seen = visible(pos, T, window, sink, prefix, first)
    used = seen.any(axis=0)  # keys that no token sees may hold anything
    far = np.abs(np.asarray(pos, dtype=np.float64)[:, None] - np.arange(T)[None, :])
    for h in range(Hq):
        kk = np.where(used[:, None], k[h // G], 0).astype(np.float64)
        vv = np.where(used[:, None], v[h // G], 0).astype(np.float64)
        x = q[h].astype(np.float64) @ kk.T * scale
        if softcap:
            x = softcap * np.tanh(x / softcap)
        if slopes is not None:
            x = x - float(slopes[h]) * far
        x = np.where(seen, x, -np.inf)
        top = x.max(axis=-1, keepdims=True)
        e = np.exp(x - np.where(np.isinf(top), 0, top))
        total = e.sum(axis=-1, keepdims=True)
        e /= np.where(total == 0, 1, total)
        out[h], spread[h] = e @ vv, e @ np.abs(vv)
    return out, spread


def paged(q: np.ndarray, k_pool: np.ndarray, v_pool: np.ndarray, tables: np.ndarray,
          q_start: np.ndarray, q_len: np.ndarray, ctx_lens: np.ndarray, dtype: str,
          scale: float | None = None, first: np.ndarray | None = None,
          prefix: np.ndarray | None = None, **mod) -> tuple[np.ndarray, np.ndarray]:
    """Batched form: sequence b's q_len[b] rows of q (T, Hq, D; uint16 bits of
    ``dtype``) from row q_start[b] are its last tokens (positions below 0 see the
    prefix alone); ``first`` per row.  (out, spread) in float64, zeros elsewhere."""
    from .rng import to_f32

    bs, D = k_pool.shape[2], q.shape[2]
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(len(q_len)):
        n, c, r0 = int(q_len[b]), int(ctx_lens[b]), int(q_start[b])
        if n == 0:
            continue
        kb, vb = gather(k_pool, v_pool, list(tables[b]), c, bs)
        qb = to_f32(q[r0:r0 + n], dtype).transpose(1, 0, 2)
        o, s = attention(qb, to_f32(kb, dtype), to_f32(vb, dtype), np.arange(c - n, c),
                         D ** -0.5 if scale is None else scale,
                         prefix=0 if prefix is None else min(int(prefix[b]), c),
                         first=0 if first is None else first[r0:r0 + n], **mod)
        out[r0:r0 + n], spread[r0:r0 + n] = o.transpose(1, 0, 2), s.transpose(1, 0, 2)
    return out, spread

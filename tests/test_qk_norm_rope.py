"""Head norm, rotation and append in one pass (ops.qk_norm_rope[_append]) against
the definition in 64 bits.

Tolerance, per element, from the roundings the kernel makes:
  eps/2 |ref|          the store in the tensor's type (fp16 also its smallest step),
  32 * 2^-24 (|a|+|b|) fp32 arithmetic on the pair (a, b): the mean square sums at
                       most 16 rounded terms in a chain (half of it through the
                       root: 8 units of 2^-24), rsqrtf 2 ulp (4), three products
                       (3), the angle's rounding to fp32 half turns (2), sine and
                       cosine 2 ulp (4) and the rotation's products and sum (3),
                       rounded up."""
import ctypes

import pytest
import torch

from mlxz_b200 import _native, ops
from mlxz_b200._native import DeviceError

gpu = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def _reference(x, pos, inv_freq, w, eps, offset, interleaved, freq_axes):
    """(result, |a| + |b| of each element's pair) in 64 bits."""
    y = x.double()
    D, half = y.shape[-1], inv_freq.numel()
    if eps is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * (w.double() + offset)
    p = pos.double()
    p = p[None] if p.dim() == 1 else p
    ax = freq_axes.long() if freq_axes is not None else torch.zeros(half, dtype=torch.long,
                                                                     device=x.device)
    th = (p[ax] * inv_freq.double()[:, None]).t()[:, None]
    i = torch.arange(half, device=x.device)
    i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = y[..., i0], y[..., i1]
    out, mag = y.clone(), y.abs()
    out[..., i0] = a * th.cos() - b * th.sin()
    out[..., i1] = b * th.cos() + a * th.sin()
    mag[..., i0] = mag[..., i1] = a.abs() + b.abs()
    return out, mag


def _assert_close(got, want):
    ref, mag = want
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + 32 * 2.0 ** -24 * mag + TINY[got.dtype]
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off"


def _inputs(T, Hq, Hkv, D, rot, dtype, axes=1, far=4000, seed=0, wdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed + T + D)
    dt = DT[dtype]
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device="cuda").to(dt)
    pos = torch.randint(0, far, (axes, T), generator=g, device="cuda").int()
    half = rot // 2
    inv = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float32) / max(half, 1))
    fa = torch.randint(0, axes, (half,), generator=g, device="cuda").int() if axes > 1 else None
    wd = wdtype or dt
    w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(wd) for _ in range(2)]
    return (qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], pos if axes > 1 else pos[0], inv,
            fa, w[0], w[1])


SHAPES = [
    # T, Hq, Hkv, D, rot
    (1, 32, 8, 128, 128),
    (3, 5, 1, 64, 64),
    (37, 8, 2, 128, 64),       # partial rotation
    (9, 7, 3, 96, 96),         # heads that do not fill a warp's groups
    (5, 6, 2, 80, 32),
    (4, 3, 2, 256, 256),
    (11, 2, 2, 16, 16),
    (700, 4, 4, 64, 64),
    (2, 61, 7, 112, 16),
    (6, 4, 2, 48, 0),          # norm alone
    (2500, 33, 3, 128, 128),
]


@gpu
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_dense_matches_definition(cuda, T, Hq, Hkv, D, rot, dtype, interleaved):
    q, k, _, pos, inv, _, qw, kw = _inputs(T, Hq, Hkv, D, rot, dtype)
    qo, ko = ops.qk_norm_rope(q, k, pos, inv, q_weight=qw, k_weight=kw, eps=1e-6,
                              interleaved=interleaved)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        _assert_close(got, _reference(x, pos, inv, w, 1e-6, 0.0, interleaved, None))
    ops.check_device_errors(0)


@gpu
@pytest.mark.parametrize("axes", [2, 3, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_several_axes_and_far_positions(cuda, axes, interleaved):
    """Positions up to 2^31 - 1, where fp32 angles would be off by turns."""
    q, k, _, pos, inv, fa, qw, kw = _inputs(41, 6, 2, 128, 96, "f32", axes=axes, far=2 ** 31 - 1)
    pos[0, :4] = torch.tensor([0, 1, 2 ** 31 - 1, 2 ** 30 + 1], device=cuda, dtype=torch.int32)
    qo, ko = ops.qk_norm_rope(q, k, pos, inv, freq_axes=fa, interleaved=interleaved)
    _assert_close(qo, _reference(q, pos, inv, None, None, 0.0, interleaved, fa))
    _assert_close(ko, _reference(k, pos, inv, None, None, 0.0, interleaved, fa))
    neg, _ = ops.qk_norm_rope(q, k, -pos, inv, freq_axes=fa, interleaved=interleaved)
    _assert_close(neg, _reference(q, -pos, inv, None, None, 0.0, interleaved, fa))


@gpu
@pytest.mark.parametrize("wdtype", ["f32", "bf16", "f16"])
def test_weight_types_offset_and_missing_weights(cuda, wdtype):
    q, k, _, pos, inv, _, qw, kw = _inputs(19, 4, 2, 64, 64, "bf16", wdtype=DT[wdtype])
    qo, ko = ops.qk_norm_rope(q, k, pos, inv, q_weight=qw, k_weight=kw, eps=1e-5,
                              weight_offset=1.0)
    _assert_close(qo, _reference(q, pos, inv, qw, 1e-5, 1.0, False, None))
    _assert_close(ko, _reference(k, pos, inv, kw, 1e-5, 1.0, False, None))
    qo, ko = ops.qk_norm_rope(q, k, pos, inv, q_weight=qw, eps=1e-5, weight_offset=1.0)
    _assert_close(ko, _reference(k, pos, inv, None, 1e-5, 0.0, False, None))


def _pools(T, Hkv, D, bs, dt, seed=0):
    n = -(-T // bs) + 3
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randperm(n, generator=g, device="cuda")
    t = torch.arange(T, device="cuda")
    slots = ids[t // bs] * bs + t % bs
    kp = torch.randn(n, Hkv, bs, D, generator=g, device="cuda").to(dt)
    return kp, torch.randn_like(kp), slots


@gpu
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", [s for s in SHAPES if s[3] in (64, 128, 256, 80)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_writes_slots_and_nothing_else(cuda, T, Hq, Hkv, D, rot, dtype):
    q, k, v, pos, inv, _, qw, kw = _inputs(T, Hq, Hkv, D, rot, dtype)
    bs = 48
    kp, vp, slots = _pools(T, Hkv, D, bs, DT[dtype])
    slots = slots.clone()
    if T > 2:
        slots[1] = -1  # a padded row: its K/V go nowhere, its queries are still turned
    k0, v0 = kp.clone(), vp.clone()
    qo = ops.qk_norm_rope_append(q, k, v, pos, inv, kp, vp, slots, q_weight=qw, k_weight=kw,
                                 eps=1e-6)
    _assert_close(qo, _reference(q, pos, inv, qw, 1e-6, 0.0, False, None))
    # the same keys as the dense form, bit for bit; values copied
    _, kd = ops.qk_norm_rope(q, k, pos, inv, q_weight=qw, k_weight=kw, eps=1e-6)
    live = slots >= 0
    blk, at = slots[live] // bs, slots[live] % bs
    k0[blk, :, at] = kd[live]
    v0[blk, :, at] = v[live]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    ops.check_device_errors(0)


@gpu
def test_in_place_and_strided_outputs(cuda):
    q, k, v, pos, inv, _, qw, kw = _inputs(77, 8, 2, 128, 128, "bf16")
    want_q, want_k = ops.qk_norm_rope(q, k, pos, inv, q_weight=qw, k_weight=kw, eps=1e-6)
    v0 = v.clone()
    room = torch.zeros(77, 2, 8, 128, dtype=q.dtype, device=cuda)
    qo, _ = ops.qk_norm_rope(q, k, pos, inv, q_weight=qw, k_weight=kw, eps=1e-6, q_out=room[:, 1])
    assert torch.equal(qo, want_q) and not room[:, 0].any()
    ops.qk_norm_rope(q, k, pos, inv, q_weight=qw, k_weight=kw, eps=1e-6, q_out=q, k_out=k)
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(v, v0)


@gpu
def test_infinities_stay_in_their_pair_without_a_norm(cuda):
    q, k, v, pos, inv, *_ = _inputs(5, 2, 2, 128, 64, "bf16")
    q[1, 0, 100] = float("inf")   # not rotated
    q[2, 1, 3] = float("nan")     # rotates with dimension 35
    kp, vp, slots = _pools(5, 2, 128, 16, torch.bfloat16)
    v[0, 0, 5] = float("-inf")
    qo = ops.qk_norm_rope_append(q, k, v, pos, inv, kp, vp, slots)
    bad = (~qo.isfinite()).nonzero().tolist()
    assert bad == [[1, 0, 100], [2, 1, 3], [2, 1, 35]]
    assert vp[slots[0] // 16, 0, slots[0] % 16, 5] == float("-inf")


@gpu
def test_graph_replay_and_side_stream(cuda):
    q, k, v, pos, inv, _, qw, kw = _inputs(64, 8, 2, 128, 128, "bf16")
    kp, vp, slots = _pools(64, 2, 128, 16, torch.bfloat16)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.qk_norm_rope_append(q, k, v, pos, inv, kp, vp, slots, qw, kw, eps=1e-6)
        with torch.cuda.graph(g, stream=side):
            qo = ops.qk_norm_rope_append(q, k, v, pos, inv, kp, vp, slots, qw, kw, eps=1e-6)
    torch.cuda.current_stream().wait_stream(side)
    pos.add_(11)
    g.replay()
    torch.cuda.synchronize()
    _assert_close(qo, _reference(q, pos, inv, qw, 1e-6, 0.0, False, None))


@gpu
def test_device_errors(cuda):
    q, k, v, pos, inv, fa, *_ = _inputs(3, 2, 1, 64, 64, "bf16", axes=2)
    fa[0] = 2
    ops.qk_norm_rope(q, k, pos, inv, freq_axes=fa)
    with pytest.raises(DeviceError, match="axis"):
        ops.check_device_errors(0)
    kp, vp, slots = _pools(3, 1, 64, 16, torch.bfloat16)
    slots = slots.clone()
    slots[2] = kp.shape[0] * 16
    k0 = kp.clone()
    ops.qk_norm_rope_append(q, k, v, pos[0].contiguous(), inv, kp, vp, slots)
    with pytest.raises(DeviceError, match="slot"):
        ops.check_device_errors(0)
    assert (kp != k0).any(-1).sum() == 2  # the two good rows


@gpu
def test_misaligned_tensors_are_refused(cuda):
    buf = torch.zeros(4, 2, 136, dtype=torch.bfloat16, device=cuda)
    pos = torch.zeros(4, dtype=torch.int32, device=cuda)
    inv = torch.ones(64, device=cuda)
    with pytest.raises(ValueError, match="16-byte"):
        ops.qk_norm_rope(buf[..., 1:129], buf[..., 8:], pos, inv)
    odd = torch.zeros(4, 2, 132, dtype=torch.bfloat16, device=cuda)[..., :128]
    with pytest.raises(ValueError, match="16-byte"):
        ops.qk_norm_rope(odd, buf[..., 8:], pos, inv)


def test_refusals_on_the_host():
    q, k = torch.zeros(4, 8, 64), torch.zeros(4, 2, 64)
    pos, inv = torch.zeros(4, dtype=torch.int32), torch.ones(32)
    w = torch.ones(64)
    ok = dict(positions=pos, inv_freq=inv)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qk_norm_rope(q, k, **ok)
    for kw, text in ((dict(positions=pos.long(), inv_freq=inv), "positions"),
                     (dict(positions=pos[:3], inv_freq=inv), "positions"),
                     (dict(positions=pos, inv_freq=inv.double()), "inv_freq"),
                     (dict(positions=pos.expand(2, 4).contiguous(), inv_freq=inv), "freq_axes"),
                     (dict(ok, freq_axes=pos), "freq_axes"),
                     (dict(ok, q_weight=w), "eps"),
                     (dict(ok, q_weight=w[:32], eps=1e-6), "weights"),
                     (dict(ok, q_weight=w, k_weight=w.half(), eps=1e-6), "weights"),
                     (dict(ok, q_out=q[:2]), "q_out")):
        with pytest.raises(ValueError, match=text):
            ops.qk_norm_rope(q, k, **kw)
    with pytest.raises(ValueError, match="k must"):
        ops.qk_norm_rope(q, k.half(), **ok)
    pool = torch.zeros(3, 2, 16, 64)
    slots = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="slot_mapping"):
        ops.qk_norm_rope_append(q, k, k, pos, inv, pool, pool, slots.int())
    with pytest.raises(ValueError, match="heads"):
        ops.qk_norm_rope_append(q, q, q, pos, inv, pool, pool, slots)
    with pytest.raises(ValueError, match="dtype"):
        ops.qk_norm_rope_append(q, k, k, pos, inv, pool.half(), pool.half(), slots)


def test_c_abi_argument_errors():
    lib = _native.lib()
    p = ctypes.c_void_p(64)  # never read: every call below is refused first

    def call(T=4, Hq=8, Hkv=2, D=64, rot=64, dtype=1, k_out=p, pools=None, slots=None, axes=1,
             eps=1e-6, qp=p, v=None, ts=640):
        return lib.mz_qk_norm_rope(p, ts, 64, k_out, 640, 64, qp, 640, 64, p, 640, 64, v, 640, 64,
                                   pools, pools, slots, 16, 4, p, 4, axes, p, None, rot, 0, None,
                                   None, 1, 0.0, eps, 1, T, Hq, Hkv, D, dtype, None, None)

    inv, uns, ali = (_native.MZ_ERR_INVALID_ARG, _native.MZ_ERR_UNSUPPORTED,
                     _native.MZ_ERR_ALIGNMENT)
    for kw, rc in ((dict(dtype=9), inv), (dict(T=-1), inv), (dict(Hkv=0), inv),
                   (dict(D=72), uns), (dict(D=272), uns), (dict(rot=24), uns),
                   (dict(rot=80), uns), (dict(axes=5), inv), (dict(axes=2), inv),
                   (dict(eps=-1.0), inv), (dict(eps=float("nan")), inv), (dict(k_out=None), inv),
                   (dict(k_out=None, pools=p), inv), (dict(pools=p, slots=p, v=p), inv),
                   (dict(qp=ctypes.c_void_p(66)), ali), (dict(ts=642), ali)):
        assert call(**kw) == rc, kw
    assert call(T=0) == _native.MZ_OK

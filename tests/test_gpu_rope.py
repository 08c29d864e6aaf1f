"""Norm and rotation of query and key rows against the 64-bit formula.

Tolerance of an f32 result: the norm's factor carries the sum's 13 roundings
halved, the reciprocal root's and two products', the rotation two products, a
sum and the cosine's own rounding: 20 half-steps of 2^-24 of the pair's size
are above all of it.  A bf16 result adds its own 2^-8 of the value, and the
place of an f32 error beside a border is in the first term.
"""
import numpy as np
import pytest

import mx4_ref

pytestmark = pytest.mark.gpu


def make(rows, heads, D, rot, axes, far, seed, dtype, norm=True, pad=0):
    """Projections [rows][heads*D + pad], their rotation, and the same in numpy."""
    import torch
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((rows, heads * D + pad)).astype(np.float32)).cuda().to(dtype)
    half = rot // 2
    freqs = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
    axis = (np.arange(half) * 7 % axes).astype(np.int32)
    pos = rng.integers(max(0, far - 5000), far + 1, (axes, rows)).astype(np.int32)
    w = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in range(2)]
    dev = [None if a is None else torch.from_numpy(a).cuda() for a in (freqs, axis, pos, *w)]
    return x, dict(freqs=freqs, axis=axis, pos=pos, w=w), dev


def check(got, want, x, bf16):
    got = got.float().cpu().numpy().astype(np.float64)
    size = np.abs(want).max(-1, keepdims=True) + 1e-30
    tol = 40 * 2.0 ** -24 * size + (np.abs(want) * 2.0 ** -8 if bf16 else 0)
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {float((np.abs(got - want) / tol).max())}"


@pytest.mark.parametrize("D,rot", [(128, 128), (256, 256), (256, 64), (128, 32), (128, 80), (256, 8), (128, 0)])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("axes,far", [(1, 300), (3, 2000000)])
def test_rope_rows(rkv, ctx, D, rot, adjacent, axes, far):
    import torch
    for rows, qh, kh, src, out, norm in [(1, 24, 4, torch.bfloat16, torch.bfloat16, True),
                                         (37, 5, 1, torch.float32, torch.float32, True),
                                         (300, 16, 2, torch.bfloat16, torch.float32, False)]:
        x, h, (freqs, axis, pos, qw, kw) = make(rows, qh + kh, D, rot, axes, far, rows + D, src, norm)
        rope = rkv.rope_args(rot, freqs, pos, axis, adjacent, qw, kw, eps=1e-6)
        v = x.reshape(rows, qh + kh, D)
        q, k = v[:, :qh], v[:, qh:]
        qo, ko = (torch.full(t.shape, 9.0, dtype=out, device="cuda") for t in (q, k))
        rkv.rope_rows(ctx, rope, q, k, qo, ko)
        ctx.sync()
        for t, o, w in ((q, qo, h["w"][0]), (k, ko, h["w"][1])):
            want = mx4_ref.rope(t.float().cpu().numpy(), h["freqs"], h["pos"], h["axis"], adjacent, w, 1e-6)
            check(o, want, t, out == torch.bfloat16)


def test_far_positions_keep_their_angle(rkv, ctx):
    """Positions up to 2^31 - 1 with frequencies above one radian."""
    import torch
    D, rows = 128, 64
    rng = np.random.default_rng(3)
    x = rng.standard_normal((rows, 1, D)).astype(np.float32)
    freqs = rng.uniform(0, 3, D // 2).astype(np.float32)
    pos = np.concatenate([[0, 2 ** 31 - 1], rng.integers(2 ** 30, 2 ** 31 - 1, rows - 2)]).astype(np.int32)[None]
    q = torch.from_numpy(x).cuda()
    out = torch.empty_like(q)
    rope = rkv.rope_args(D, torch.from_numpy(freqs).cuda(), torch.from_numpy(pos).cuda())
    rkv.rope_rows(ctx, rope, q, None, out, None)
    # the angles' product is exact in f64; its sine is libm's
    check(out, mx4_ref.rope(x, freqs, pos, np.zeros(D // 2, int), False), x, False)
    assert (out[0] == q[0]).all()


@pytest.mark.parametrize("adjacent", [False, True])
def test_in_place_in_a_packed_projection(rkv, ctx, adjacent):
    """q and k turned where they lie; the values beside them stay."""
    import torch
    D, qh, kh, rows = 128, 6, 2, 77
    x, h, (freqs, axis, pos, qw, kw) = make(rows, qh + 2 * kh, D, 96, 2, 5000, 4, torch.bfloat16, pad=64)
    rope = rkv.rope_args(96, freqs, pos, axis, adjacent, qw, kw, eps=1e-5)

    def heads(t):
        v = t[:, :(qh + 2 * kh) * D].unflatten(1, (qh + 2 * kh, D))
        return v[:, :qh], v[:, qh:qh + kh]
    q, k = heads(x)
    qo, ko = torch.empty(q.shape, dtype=x.dtype, device="cuda"), torch.empty(k.shape, dtype=x.dtype, device="cuda")
    rkv.rope_rows(ctx, rope, q, k, qo, ko)
    keep = x.clone()
    rkv.rope_rows(ctx, rope, q, k, q, k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    x[:, :(qh + kh) * D] = keep[:, :(qh + kh) * D]
    assert torch.equal(x, keep)


def test_bf16_weights_and_only_keys(rkv, ctx):
    import torch
    D, rows = 256, 21
    x, h, (freqs, axis, pos, _, kw) = make(rows, 3, D, D, 1, 100, 5, torch.float32)
    k = x.reshape(rows, 3, D)
    out = torch.empty_like(k)
    kb = kw.to(torch.bfloat16)
    rkv.rope_rows(ctx, rkv.rope_args(D, freqs, pos[0].contiguous(), k_norm=kb, eps=0.1), None, k, None, out)
    want = mx4_ref.rope(k.cpu().numpy(), h["freqs"], h["pos"], h["axis"], False, kb.float().cpu().numpy(), 0.1)
    check(out, want, k, False)


def test_zero_and_nonfinite_rows(rkv, ctx):
    """A row of zeros stays zero with eps above 0; NaN stays in its head."""
    import torch
    D = 128
    q = torch.randn(4, 2, D, device="cuda")
    q[1, 0] = 0
    q[2, 1, 5] = float("nan")
    w = torch.ones(D, device="cuda")
    freqs = torch.full((D // 2,), 0.1, device="cuda")
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    rkv.rope_rows(ctx, rkv.rope_args(D, freqs, pos, q_norm=w, eps=1e-6), q, None, out, None)
    assert (out[1, 0] == 0).all() and torch.isnan(out[2, 1]).all()
    assert torch.isfinite(out[2, 0]).all() and torch.isfinite(out[[0, 1, 3]]).all()


def test_bad_axis_is_reported(rkv, ctx):
    import torch
    D = 128
    q = torch.randn(2, 1, D, device="cuda")
    pos = torch.ones(2, 2, dtype=torch.int32, device="cuda")
    axis = torch.full((D // 2,), 7, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    rkv.rope_rows(ctx, rkv.rope_args(D, torch.ones(D // 2, device="cuda"), pos, axis), q, None, out, None)
    with pytest.raises(rkv.RkvError) as e:
        ctx.sync()
    assert e.value.status == rkv.ERR_BAD_BLOCK_TABLE and "0x2" in e.value.message
    ctx.sync()

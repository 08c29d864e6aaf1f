"""Chunked prefill over 4-bit pages against the 64-bit formula: row i of an
entry is the decode of length ctx + i + 1.

Tolerances as in test_gpu_mx4_decode.  A bf16 row's weights have 11 bits, cut
off, and their sum is of the weights as cut: with p (1 - d), 0 <= d < 2^-10, in
the place of p and o the exact row,
  o' - o = sum p (1 - d) (v - o) / sum p (1 - d)
         = sum p (m - d) (v - o) / sum p (1 - d)        for any constant m,
as sum p (v - o) = 0; with m = 2^-11 that is below 2^-11 (1 + 2^-9) times the
mean of |v - o| under p, which is at most the mean of |v| plus |o|.  (A bound by
the row's own largest value, as this file first had it, does not follow: values
of both signs cancel in o and not in |v|.)  The value's own rounding to bf16
adds 2^-8 of it, the f32 terms 8 * 2e-5 of the norm's share.
"""
import math

import numpy as np
import pytest

import mx4_ref
from test_gpu_mx4_decode import Cache, check, query

pytestmark = pytest.mark.gpu


def run(rkv, ctx, c, entries, q, scale, out_dtype=None, seg=0, ws=True, offsets=None, stream=None):
    """entries: (sequence, tokens before the rows, rows)."""
    import torch
    out = torch.full(q.shape, 7.0, dtype=out_dtype or torch.float32, device="cuda")
    seqs, ctxs, rows = ([e[i] for e in entries] for i in range(3))

    def args(w=None):
        return rkv.prefill_args(seqs, ctxs, rows, q, out, scale, q_offsets=offsets, segment_tokens=seg, workspace=w)
    need = rkv.prefill_mx4_workspace_bytes(c.g, args()) if ws else 0
    a = args(torch.full((need,), 255, dtype=torch.uint8, device="cuda") if need else None)
    rkv.prefill_mx4(ctx, c.g, c.pages, c.bt_d, len(c.lens), a)
    ctx.sync()
    return out


def want_of(c, entries, q, scale, size=False):
    out, at = np.zeros(q.shape), 0
    for s, ctx, n in entries:
        k, v = c.kv[s]
        out[at:at + n] = mx4_ref.attend(q[at:at + n], k, np.abs(v) if size else v, scale,
                                        [ctx + 1 + i for i in range(n)])
        at += n
    return out


def close(got, want, bf16, what="", size=None):
    """size: the rows' means of |v| (bf16)."""
    if not bf16:
        return check(got, want, False, what)
    g = got.float().cpu().numpy().astype(np.float64)
    tol = (np.abs(want) * 2.0 ** -8 + 2.0 ** -11 * (1 + 2.0 ** -7) * (size + np.abs(want)) +
           16e-5 * np.linalg.norm(want) / math.sqrt(want.size))
    worst = float((np.abs(g - want) / tol).max())
    print(f"[{what}] worst of tolerance {worst:.3f}", flush=True)
    assert worst <= 1, what


@pytest.mark.parametrize("Hq,Hkv,D,PT", [(16, 2, 256, 64), (8, 2, 128, 32), (24, 4, 256, 32), (3, 1, 128, 256),
                                         (12, 1, 256, 128), (4, 4, 128, 64), (40, 1, 128, 32)])
@pytest.mark.parametrize("bf16", [False, True])
def test_prefill(rkv, ctx, Hq, Hkv, D, PT, bf16):
    import torch
    entries = [(0, 0, 1), (1, 0, 33), (2, 300, 50), (3, 31, 1), (4, 64, 64), (5, 7, 9)]
    c = Cache(rkv, Hkv, D, PT, [a + n for _, a, n in entries], seed=Hq + D)
    q, qn = query((sum(n for _, _, n in entries), Hq, D), 1, True)
    out = run(rkv, ctx, c, entries, q, 1 / math.sqrt(D), torch.bfloat16 if bf16 else None)
    scale = 1 / math.sqrt(D)
    close(out, want_of(c, entries, qn, scale), bf16, f"{Hq}/{Hkv} D{D} PT{PT}", want_of(c, entries, qn, scale, True))


@pytest.mark.parametrize("seg", [-1, 0, 64, 128, 512])
def test_split_ranges(rkv, ctx, seg):
    entries = [(0, 900, 20), (1, 0, 40), (2, 63, 2)]
    c = Cache(rkv, 2, 128, 64, [a + n for _, a, n in entries], seed=2)
    q, qn = query((62, 16, 128), 3, True)
    want = want_of(c, entries, qn, 0.1)
    a = run(rkv, ctx, c, entries, q, 0.1, seg=seg)
    close(a, want, False, f"seg {seg}")
    assert (a == run(rkv, ctx, c, entries, q, 0.1, seg=seg)).all()


def test_rows_of_no_entry_stay(rkv, ctx):
    """Rows between and behind the entries' own keep what they held; an entry
    without rows is fine, and so is one sequence twice."""
    import torch
    c = Cache(rkv, 1, 128, 32, [80, 40], seed=4)
    entries = [(0, 10, 20), (1, 40, 0), (0, 60, 5)]
    q, qn = query((60, 4, 128), 5, True)
    out = run(rkv, ctx, c, entries, q, 0.2, offsets=[3, 40, 41])
    live = np.zeros(60, bool)
    live[3:23] = live[41:46] = True
    assert (out[torch.from_numpy(~live).cuda()] == 7).all()
    want = want_of(c, [(0, 10, 20), (0, 60, 5)], qn[live], 0.2)
    close(out[torch.from_numpy(live).cuda()], want, False)


@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_scale_sign_and_zero(rkv, ctx, scale):
    c = Cache(rkv, 2, 128, 32, [130], seed=6, loud=False)
    q, qn = query((100, 8, 128), 7, True)
    close(run(rkv, ctx, c, [(0, 30, 100)], q, scale), want_of(c, [(0, 30, 100)], qn, scale), False)


@pytest.mark.parametrize("bf16", [False, True])
def test_v_of_any_size(rkv, ctx, bf16):
    import torch
    rng = np.random.default_rng(8)
    base = rng.standard_normal((300, 1, 128))
    vs = [base * 3e-7, base * 100, base * 2.0 ** (-20 + 24 * np.arange(300) / 300)[:, None, None]]
    c = Cache(rkv, 1, 128, 32, [300] * 3, seed=9, v=vs)
    entries = [(s, 200, 100) for s in range(3)]
    q, qn = query((300, 8, 128), 10, True)
    out = run(rkv, ctx, c, entries, q, 0.1, torch.bfloat16 if bf16 else None)
    want = want_of(c, entries, qn, 0.1)
    size = want_of(c, entries, qn, 0.1, True)
    for s in range(3):
        at = slice(100 * s, 100 * s + 100)
        close(out[at], want[at], bf16, f"sequence {s}", size[at])


@pytest.mark.parametrize("seg", [-1, 64])
def test_nan_blocks_stay_with_their_rows(rkv, ctx, seg):
    def edit(c):
        c.v[0][70, 1, 100] = np.nan  # block 3 of kv head 1
        c.k[0][90, 0, 5] = np.inf
        c.v[0][3, 0, 0] = np.inf     # attended by every row: block 0 of kv head 0
    c = Cache(rkv, 2, 128, 32, [120], seed=11, edit=edit)
    q, qn = query((100, 16, 128), 12, True)
    out = run(rkv, ctx, c, [(0, 20, 100)], q, 0.1, seg=seg).cpu().numpy()
    want = want_of(c, [(0, 20, 100)], qn, 0.1)
    nan = np.zeros(out.shape, bool)
    nan[:, :8, :32] = True
    nan[70:, :8] = True
    nan[50:, 8:, 96:] = True
    assert (np.isnan(out) == nan).all()
    assert np.abs(out - want)[~nan].max() < 1e-4


def test_bad_pages_are_reported(rkv, ctx):
    c = Cache(rkv, 1, 128, 32, [100], seed=13)
    q, _ = query((10, 4, 128), 14, True)
    c.bt_d[0, 1] = -1
    with pytest.raises(rkv.RkvError) as e:
        run(rkv, ctx, c, [(0, 90, 10)], q, 0.1)
    assert e.value.status == rkv.ERR_BAD_BLOCK_TABLE
    ctx.sync()


def test_rows_are_the_decodes(rkv, ctx):
    """A chunk's row i against rkv_decode_mx4 of length ctx + i + 1."""
    import torch
    from test_gpu_mx4_decode import run as decode
    L, n = 260, 40
    c = Cache(rkv, 2, 256, 64, [L], seed=15)
    q, qn = query((n, 16, 256), 16, True)
    out = run(rkv, ctx, c, [(0, L - n, n)], q, 1 / 16)
    for i in (0, 1, 17, 39):
        c.lens = np.asarray([L - n + i + 1], np.int32)
        c.lens_d = torch.from_numpy(c.lens).cuda()
        one = decode(rkv, ctx, c, q[i][None, None], 1 / 16)
        check(out[i], one[0, 0].cpu().numpy().astype(np.float64), False, f"row {i}")


def test_captured_and_replayed(rkv, ctx):
    """A split chunk captured once and replayed with other queries, eager calls
    between: every replay bit for bit the eager call's."""
    import torch
    entries = [(0, 1500, 30), (1, 10, 20)]
    c = Cache(rkv, 2, 256, 32, [1530, 30], seed=17)
    q, _ = query((50, 16, 256), 18, True)
    out = torch.empty(q.shape, dtype=torch.bfloat16, device="cuda")

    def args(w=None):
        return rkv.prefill_args([0, 1], [1500, 10], [30, 20], q, out, 0.06, segment_tokens=512, workspace=w)
    need = rkv.prefill_mx4_workspace_bytes(c.g, args())
    assert need > 0
    a = args(torch.full((need,), 255, dtype=torch.uint8, device="cuda"))
    other = args(torch.full((need,), 255, dtype=torch.uint8, device="cuda"))
    rkv.prefill_mx4(ctx, c.g, c.pages, c.bt_d, 2, a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rkv.prefill_mx4(ctx, c.g, c.pages, c.bt_d, 2, a)
    for i in range(4):
        q.copy_(query((50, 16, 256), 30 + i, True)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        rkv.prefill_mx4(ctx, c.g, c.pages, c.bt_d, 2, other)
        ctx.sync()
        assert (out == got).all() and (got != 0).any()


def test_pages_behind_32_bits(rkv, ctx):
    """Pages whose bytes start past 2^32: rows go in, come back, are attended by
    a decode and a chunk, and pages of the same numbers modulo 2^32 stay."""
    import torch
    Hkv, D, PT, Hq, L = 2, 256, 64, 16, 200
    g1 = rkv.geometry(Hkv, D, PT, 1)
    n = (1 << 32) // rkv.mx4_page_bytes(g1) + 16
    g = rkv.geometry(Hkv, D, PT, n)
    rng = np.random.default_rng(19)
    pages = torch.empty(n, rkv.mx4_page_bytes(g), dtype=torch.uint8, device="cuda")
    pages[:40].fill_(9)
    bt = torch.tensor([[n - 1, n - 7, n - 3, n - 12]], dtype=torch.int32, device="cuda")
    x = rng.standard_normal((L, 2 * Hkv, D)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    ids = torch.zeros(L, dtype=torch.int32, device="cuda")
    pos = torch.arange(L, dtype=torch.int32, device="cuda")
    rkv.append_rope(ctx, g, rkv.CACHE_MX4, pages, bt, ids, pos, t[:, :Hkv], t[:, Hkv:])
    k, v = torch.empty(L, Hkv, D, device="cuda"), torch.empty(L, Hkv, D, device="cuda")
    rkv.read_rows(ctx, g, rkv.CACHE_MX4, pages, bt, ids, pos, k, v)
    ctx.sync()
    assert (pages[:40] == 9).all()
    kn, vn = mx4_ref.quantize(x[:, :Hkv], "k")[2], mx4_ref.quantize(x[:, Hkv:], "v")[2]
    assert (k.cpu().numpy() == kn).all() and (v.cpu().numpy() == vn).all()
    q, qn = query((30, Hq, D), 20, True)
    want = mx4_ref.attend(qn, kn, vn, 1 / 16, L - 30 + 1 + np.arange(30))
    out = torch.empty(q.shape, device="cuda")
    rkv.prefill_mx4(ctx, g, pages, bt, 1, rkv.prefill_args([0], [L - 30], [30], q, out, 1 / 16))
    one = torch.empty(1, 1, Hq, D, device="cuda")
    rkv.decode_mx4(ctx, g, pages, bt, torch.tensor([L], dtype=torch.int32, device="cuda"),
                   rkv.decode_args(q[29:][None], one, ids[:1], 1 / 16, L))
    ctx.sync()
    close(out, want, False, "chunk")
    close(one[0, 0][None], want[29:], False, "decode")

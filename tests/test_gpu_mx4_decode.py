"""Attention over 4-bit pages against the 64-bit formula on the pages' values.

Tolerance, relative to the output's 2-norm: products are exact, sums are f32.
A score of D products carries at most D/32 + 2 roundings of 2^-24 of the sum of
their magnitudes, an exponent 2 more; weights carry 2^-22, an output as many
roundings as its waves walk tiles.  With |scale q.k| below about 20 in these
cases that stays under 2e-5; bf16 outputs add their own 2^-8 at each value.
"""
import math

import numpy as np
import pytest

import mx4_ref

pytestmark = pytest.mark.gpu


class Cache:
    """Sequences of the given lengths in shuffled 4-bit pages, packed by the reference."""

    def __init__(self, rkv, Hkv, D, PT, lens, seed=0, loud=True, junk=True, k=None, v=None, edit=None):
        import torch
        rng = np.random.default_rng(seed)
        self.lens = np.asarray(lens, np.int32)
        npg = [-(-int(L) // PT) for L in lens]
        self.num_pages = sum(npg) + 3
        self.bt = np.full((len(lens), max(npg + [1])), -1, np.int32)
        perm = rng.permutation(self.num_pages)
        at = 0
        for s, n in enumerate(npg):
            self.bt[s, :n] = perm[at:at + n]
            at += n
        f = np.ones((Hkv, D))
        if loud:
            f[rng.random((Hkv, D)) < 0.02] = 8
        self.k = [rng.standard_normal((L, Hkv, D)) * f for L in lens] if k is None else k
        self.v = [rng.standard_normal((L, Hkv, D)) * f for L in lens] if v is None else v
        if edit:
            edit(self)
        n = self.num_pages * mx4_ref.page_bytes(Hkv, D, PT)
        # what nobody wrote is anybody's: codes and scales of any value, NaN among them
        pages = rng.integers(0, 256, n).astype(np.uint8) if junk else np.zeros(n, np.uint8)
        for s, L in enumerate(lens):
            mx4_ref.write_rows(pages, Hkv, D, PT, self.bt, [s] * L, range(L), self.k[s], self.v[s])
        self.kv = [(mx4_ref.quantize(a, "k")[2], mx4_ref.quantize(b, "v")[2]) for a, b in zip(self.k, self.v)]
        self.g = rkv.geometry(Hkv, D, PT, self.num_pages)
        self.pages = torch.from_numpy(pages).cuda()
        self.bt_d = torch.from_numpy(self.bt).cuda()
        self.lens_d = torch.from_numpy(self.lens).cuda()

    def want(self, q, scale, seqs=None, q_len=1):
        out = np.zeros(q.shape)
        for b, s in enumerate(range(len(self.lens)) if seqs is None else seqs):
            L = int(self.lens[s])
            out[b] = mx4_ref.attend(q[b], *self.kv[s], scale, [L - q_len + 1 + j for j in range(q_len)])
        return out


def run(rkv, ctx, c, q, scale, q_len=1, seqs=None, out_dtype=None, part=0, longest=None, ws_fill=None):
    import torch
    out = torch.full(q.shape, 7.0, dtype=out_dtype or torch.float32, device="cuda")
    ids = torch.tensor(range(len(c.lens)) if seqs is None else seqs, dtype=torch.int32, device="cuda")
    longest = longest or max(1, int(c.lens.max()))

    def args(ws=None):
        return rkv.decode_args(q, out, ids, scale, longest, q_len=q_len, partition_tokens=part, workspace=ws)
    need = rkv.decode_mx4_workspace_bytes(c.g, args())
    ws = torch.full((max(need, 1),), 255 if ws_fill is None else ws_fill, dtype=torch.uint8, device="cuda")
    a = args(ws if need else None)
    rkv.decode_mx4(ctx, c.g, c.pages, c.bt_d, c.lens_d, a)
    ctx.sync()
    return out


def check(got, want, bf16=False, what=""):
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all(), what
    tol = np.full(want.shape, 2e-5 * max(np.linalg.norm(want) / math.sqrt(want.size), 1e-30))
    if bf16:
        tol = tol + np.abs(want) * 2.0 ** -8
    err = np.abs(got - want)
    print(f"[{what}] rel {np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30):.2e} "
          f"worst of tolerance {float((err / tol).max()):.3f}", flush=True)
    # one value's own error may be several times the norm's share of it
    assert (err <= 8 * tol).all(), what
    if not bf16:
        assert np.linalg.norm(err) <= 2e-5 * max(np.linalg.norm(want), 1e-30), what


def query(shape, seed, bf16):
    import torch
    q = torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32)).cuda()
    q = q.to(torch.bfloat16) if bf16 else q
    return q, q.float().cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("Hq,Hkv,D,PT,q_len", [
    (8, 2, 128, 32, 1), (16, 2, 256, 64, 1), (24, 4, 256, 32, 1), (4, 4, 128, 64, 1), (3, 1, 256, 128, 1),
    (16, 1, 128, 32, 1), (12, 1, 256, 64, 1), (16, 2, 256, 64, 2), (16, 2, 256, 64, 4), (16, 2, 128, 32, 4),
    (5, 1, 128, 256, 3), (28, 2, 256, 32, 2), (32, 1, 256, 64, 1), (32, 1, 128, 64, 1)])
@pytest.mark.parametrize("bf16", [True, False])
def test_decode(rkv, ctx, Hq, Hkv, D, PT, q_len, bf16):
    import torch
    lens = [q_len, 31 + q_len, 32 * 5, 33, 700, 5, 129]
    c = Cache(rkv, Hkv, D, PT, lens, seed=Hq * D + q_len)
    q, qn = query((len(lens), q_len, Hq, D), 3, bf16)
    scale = 1 / math.sqrt(D)
    want = c.want(qn, scale, q_len=q_len)
    for out_dtype in (torch.float32, torch.bfloat16):
        out = run(rkv, ctx, c, q, scale, q_len=q_len, out_dtype=out_dtype)
        check(out, want, out_dtype == torch.bfloat16, f"{Hq}/{Hkv} D{D} PT{PT} q_len{q_len} bf16={bf16}")


@pytest.mark.parametrize("part", [0, 64, 128, 320, 2048])
def test_partitions_agree(rkv, ctx, part):
    """One partition, many, uneven ones; the workspace's contents do not matter."""
    lens = [2000, 0, 64, 1, 1281]
    c = Cache(rkv, 2, 256, 64, lens, seed=4)
    q, qn = query((len(lens), 1, 16, 256), 5, True)
    want = c.want(qn, 1 / 16)
    a = run(rkv, ctx, c, q, 1 / 16, part=part)
    b = run(rkv, ctx, c, q, 1 / 16, part=part, ws_fill=0)
    check(a, want, what=f"part {part}")
    assert (a == b).all() and (a[1] == 0).all()


def test_repeated_and_permuted_entries(rkv, ctx):
    lens = [100, 300, 40]
    c = Cache(rkv, 2, 128, 32, lens, seed=6)
    seqs = [2, 0, 0, 1, 2]
    q, qn = query((5, 1, 8, 128), 7, True)
    check(run(rkv, ctx, c, q, 0.1, seqs=seqs), c.want(qn, 0.1, seqs=seqs))


@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.5])
@pytest.mark.parametrize("heads", [8, 16])
def test_scale_sign_and_zero(rkv, ctx, scale, heads):
    c = Cache(rkv, 1, 128, 32, [77, 600], seed=8, loud=False)
    q, qn = query((2, 1, heads, 128), 9, True)
    q[0, 0, 1] = 0
    qn[0, 0, 1] = 0
    check(run(rkv, ctx, c, q, scale), c.want(qn, scale))


@pytest.mark.parametrize("heads", [4, 16])
def test_v_of_any_size(rkv, ctx, heads):
    """V rising and falling by 2^24 along a sequence, tiny and large throughout."""
    L, D = 700, 128
    rng = np.random.default_rng(10)
    t = np.arange(L)[:, None, None]
    base = rng.standard_normal((L, 1, D))
    vs = [base * 2.0 ** (-20 + 24 * t / L), base * 2.0 ** (4 - 24 * t / L), base * 1e-6, base * 300]
    c = Cache(rkv, 1, D, 32, [L] * 4, seed=11, v=vs)
    q, qn = query((4, 1, heads, D), 12, True)
    want = c.want(qn, 0.3)
    out = run(rkv, ctx, c, q, 0.3)
    for s in range(4):
        check(out[s], want[s], what=f"sequence {s}")


def test_large_scores(rkv, ctx):
    """Scores in the hundreds, rising and falling along the sequence."""
    L, D = 600, 128
    rng = np.random.default_rng(13)
    k = [rng.standard_normal((L, 1, D)) * (1 + np.arange(L)[::d, None, None] / 50) for d in (1, -1)]
    c = Cache(rkv, 1, D, 64, [L, L], seed=14, k=k)
    q, qn = query((2, 1, 8, D), 15, False)
    want = c.want(qn * 8, 1.0)
    got = run(rkv, ctx, c, q * 8, 1.0).cpu().numpy()
    # a score's rounding, 2^-24 of its size, is its weight's relative error
    s = max(float(np.abs(c.kv[i][0][:, 0] @ (qn[i, 0] * 8).T).max()) for i in range(2))
    assert np.abs(got - want).max() <= 16 * s * 2.0 ** -23 * np.abs(want).max()


def test_nan_blocks_stay_with_their_rows(rkv, ctx):
    """A NaN key or value reaches the rows that attend it and no others."""
    def edit(c):
        c.k[0][-1, 0, 3] = np.nan   # the last draft's own key, kv head 0
        c.v[1][-2, 1, 40] = np.inf  # the third draft's value, kv head 1, block 1
    lens = [70, 200, 33]
    c = Cache(rkv, 2, 128, 32, lens, seed=16, edit=edit)
    q, qn = query((3, 4, 16, 128), 17, True)
    out = run(rkv, ctx, c, q, 0.1, q_len=4).cpu().numpy()
    want = c.want(qn, 0.1, q_len=4)
    nan = np.zeros(out.shape, bool)
    nan[0, 3, :8] = True
    nan[1, 2:, 8:, 32:64] = True
    assert (np.isnan(out) == nan).all()
    assert np.abs(out - want)[~nan].max() < 1e-4
    # and through partials
    out = run(rkv, ctx, c, q, 0.1, q_len=4, part=32).cpu().numpy()
    assert (np.isnan(out) == nan).all()


def test_faults_are_reported(rkv, ctx):
    import torch
    c = Cache(rkv, 2, 128, 32, [100, 100], seed=18)
    q, qn = query((2, 1, 8, 128), 19, True)
    good = run(rkv, ctx, c, q, 0.1)
    keep = c.bt_d.clone()
    c.bt_d[0, 1] = c.num_pages
    with pytest.raises(rkv.RkvError) as e:
        run(rkv, ctx, c, q, 0.1)
    assert e.value.status == rkv.ERR_BAD_BLOCK_TABLE and "0x1" in e.value.message
    c.bt_d.copy_(keep)
    for seqs, longest, bit in (([0, 9], None, "0x4"), ([0, -1], None, "0x4"), ([0, 1], 50, "0x2")):
        with pytest.raises(rkv.RkvError) as e:
            run(rkv, ctx, c, q, 0.1, seqs=seqs, longest=longest)
        assert bit in e.value.message
    c.lens_d[1] = 4096
    with pytest.raises(rkv.RkvError):
        run(rkv, ctx, c, q, 0.1, longest=5000)
    c.lens_d[1] = 100
    assert torch.equal(run(rkv, ctx, c, q, 0.1), good)


def test_short_workspace_is_refused(rkv, ctx):
    import torch
    c = Cache(rkv, 1, 128, 32, [900], seed=20)
    q, _ = query((1, 1, 8, 128), 21, True)
    out = torch.empty(q.shape, dtype=torch.float32, device="cuda")
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = rkv.decode_args(q, out, ids, 0.1, 900)
    with pytest.raises(rkv.RkvError) as e:
        rkv.decode_mx4(ctx, c.g, c.pages, c.bt_d, c.lens_d, a)
    assert e.value.status == rkv.ERR_INVALID_ARG and "workspace" in e.value.message


def test_captured_and_replayed(rkv, ctx):
    """Split decode and combine in a graph: every replay has the eager bits."""
    import torch
    lens = [1500, 40, 3000]
    c = Cache(rkv, 2, 256, 64, lens, seed=22)
    q, _ = query((3, 1, 16, 256), 23, True)
    eager = run(rkv, ctx, c, q, 1 / 16)
    out = torch.empty_like(eager)
    ids = torch.arange(3, dtype=torch.int32, device="cuda")
    a = rkv.decode_args(q, out, ids, 1 / 16, 3000)
    ws = torch.empty(rkv.decode_mx4_workspace_bytes(c.g, a), dtype=torch.uint8, device="cuda")
    a = rkv.decode_args(q, out, ids, 1 / 16, 3000, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rkv.decode_mx4(ctx, c.g, c.pages, c.bt_d, c.lens_d, a)
    for i in range(4):
        out.fill_(float(i))
        ws.fill_(i)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(run(rkv, ctx, c, q, 1 / 16), eager)


def test_two_calls_at_once(rkv, ctx):
    """Two streams, a workspace each, on the same pages and context: both give
    the results of a call alone."""
    import torch
    c = Cache(rkv, 2, 256, 64, [3000, 40, 900, 2111], seed=41)
    calls = []
    for i in range(2):
        q, _ = query((4, 1, 16, 256), 50 + i, True)
        out = torch.empty(4, 1, 16, 256, device="cuda")
        ids = torch.arange(4, dtype=torch.int32, device="cuda")
        need = rkv.decode_mx4_workspace_bytes(c.g, rkv.decode_args(q, out, ids, 0.06, 3000))
        assert need > 0
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        calls.append((rkv.decode_args(q, out, ids, 0.06, 3000, workspace=ws), q, out, ids, ws))
    alone = []
    for a, _, out, *_ in calls:
        rkv.decode_mx4(ctx, c.g, c.pages, c.bt_d, c.lens_d, a)
        ctx.sync()
        alone.append(out.clone())
        out.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        for s, (a, *_) in zip(streams, calls):
            rkv.decode_mx4(ctx, c.g, c.pages, c.bt_d, c.lens_d, a, stream=s)
    torch.cuda.synchronize()
    for want, (_, _, out, *_) in zip(alone, calls):
        assert (out == want).all()

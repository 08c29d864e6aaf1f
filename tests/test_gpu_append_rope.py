"""The rotating append against the definition, byte for byte: keys normed and
rotated in 64 bits, rounded to f32 once, quantized (the Q8_0 oracle, or the
plain 4-bit statement), laid out in pages of which every other byte stays."""
import numpy as np
import pytest

import mx4_ref
from test_gpu_rope import check

pytestmark = pytest.mark.gpu


class Call:
    """Rows of several sequences at given positions, in a given order."""

    def __init__(self, Hq, Hkv, D, spans, seed, dtype, rot, norm, axes=1, order=None, PT=32, seqs=None):
        import torch
        rng = np.random.default_rng(seed)
        self.Hq, self.Hkv, self.D, self.PT, self.dtype = Hq, Hkv, D, PT, dtype
        sid = [s for s, (_, n) in enumerate(spans) for _ in range(n)]
        pos = [p + i for p, n in spans for i in range(n)]
        order = np.arange(len(sid)) if order is None else order(rng, len(sid))
        self.seqs = np.asarray(sid, np.int32)[order]
        self.pos = np.asarray(pos, np.int32)[order]
        n = len(sid)
        x = rng.standard_normal((n, Hq + 2 * Hkv, D))
        x[:, :, rng.random(D) < 0.02] *= 8
        self.x = torch.from_numpy(x.astype(np.float32)).cuda().to(dtype)
        self.xn = self.x.float().cpu().numpy()
        half = rot // 2
        self.rot = rot
        self.freqs = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
        self.axis = (np.arange(half) % axes).astype(np.int32)
        self.rpos = self.pos[None] if axes == 1 else rng.integers(0, 9000, (axes, n)).astype(np.int32)
        self.w = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in range(2)]
        W = max(-(-(p + m) // PT) for p, m in spans)
        self.num_pages = W * len(spans) + 2
        self.bt = rng.permutation(self.num_pages)[:W * len(spans)].astype(np.int32).reshape(len(spans), W)

    def rope(self, rkv, adjacent=False, eps=1e-6, own=False):
        import torch
        f, a, p, qw, kw = (None if t is None else torch.from_numpy(t).cuda()
                           for t in (self.freqs, self.axis, self.rpos, *self.w))
        return rkv.rope_args(self.rot, f, None if own else p, a if len(self.rpos) > 1 else None, adjacent, qw, kw, eps)

    def turned(self, which, adjacent=False, eps=1e-6):
        x = self.xn[:, :self.Hq] if which == 0 else self.xn[:, self.Hq:self.Hq + self.Hkv]
        return mx4_ref.rope(x, self.freqs, self.rpos, self.axis, adjacent, self.w[which], eps)

    def parts(self):
        return self.x[:, :self.Hq], self.x[:, self.Hq:self.Hq + self.Hkv], self.x[:, self.Hq + self.Hkv:]

    def pages(self, rkv, rko, fmt, k, v, rule=0, junk=True):
        """Page bytes before (anything) and after the rows."""
        g = rkv.geometry(self.Hkv, self.D, self.PT, self.num_pages)
        n = self.num_pages * (rkv.page_bytes(g) if fmt == rkv.CACHE_Q8 else rkv.mx4_page_bytes(g))
        before = np.random.default_rng(1).integers(0, 256, n).astype(np.uint8) if junk else np.zeros(n, np.uint8)
        after = before.copy()
        k, v = k.astype(np.float32), v.astype(np.float32)
        if fmt == rkv.CACHE_Q8:
            rko.paged_append(rko.layout(self.Hkv, self.D, self.PT, self.num_pages), after, self.bt, self.seqs,
                             self.pos, k, v, rule)
        else:
            mx4_ref.write_rows(after, self.Hkv, self.D, self.PT, self.bt, self.seqs, self.pos, k, v)
        return g, before, after

    def run(self, rkv, ctx, g, fmt, before, rope, q_out=None, rule=0, rows=None):
        import torch
        pages = torch.from_numpy(before).cuda()
        sid, pos = torch.from_numpy(self.seqs).cuda(), torch.from_numpy(self.pos).cuda()
        q, k, v = self.parts()
        bt = torch.from_numpy(self.bt).cuda()
        rkv.append_rope(ctx, g, fmt, pages, bt, sid, pos, k, v, rope, q=q if q_out is not None else None,
                        q_out=q_out, rule=rule)
        ctx.sync()
        self.dev = (pages, bt, sid, pos)
        return pages.cpu().numpy()


SPANS = {
    "one": [(0, 1)],
    "one_deep": [(4099, 1)],
    "drafts": [(30, 4), (8, 4), (61, 4), (3, 4)],
    "odd": [(0, 13), (5, 100), (31, 2), (64, 64), (1, 7)],
    "steps": [(i * 37 % 90, 1) for i in range(40)],
}


def _shuffled(rng, n):
    return rng.permutation(n)


@pytest.mark.parametrize("spans", sorted(SPANS))
@pytest.mark.parametrize("fmt", ["q8", "mx4"])
@pytest.mark.parametrize("D,rot,adjacent,norm,axes", [
    (256, 256, False, True, 1), (128, 128, False, False, 1), (128, 64, True, True, 3), (256, 80, False, True, 2)])
def test_page_bytes(rkv, rko, ctx, spans, fmt, D, rot, adjacent, norm, axes):
    import torch
    fmt = rkv.CACHE_Q8 if fmt == "q8" else rkv.CACHE_MX4
    for dtype, Hq, Hkv, order in ((torch.bfloat16, 8, 2, None), (torch.float32, 3, 1, _shuffled)):
        c = Call(Hq, Hkv, D, SPANS[spans], D + rot, dtype, rot, norm, axes, order)
        v = c.xn[:, Hq + Hkv:]
        g, before, after = c.pages(rkv, rko, fmt, c.turned(1, adjacent), v)
        q_out = torch.full((len(c.pos), Hq, D), 9.0, dtype=dtype, device="cuda")
        got = c.run(rkv, ctx, g, fmt, before, c.rope(rkv, adjacent), q_out)
        assert np.array_equal(got, after), f"{(got != after).sum()} bytes differ"
        check(q_out, c.turned(0, adjacent), None, dtype == torch.bfloat16)


@pytest.mark.parametrize("fmt,PT", [("q8", 16), ("q8", 64), ("mx4", 64), ("mx4", 256)])
def test_long_call_of_odd_lengths(rkv, rko, ctx, fmt, PT):
    """The 32-row workgroups, several kv heads, runs across workgroups."""
    import torch
    fmt = rkv.CACHE_Q8 if fmt == "q8" else rkv.CACHE_MX4
    D, Hkv = 128, 33
    c = Call(2, Hkv, D, [(0, 700), (3, 555), (0, 1), (77, 801)], 5, torch.bfloat16, 128, False, PT=PT)
    c.w = [None, None]
    v = c.xn[:, 2 + Hkv:]
    g, before, after = c.pages(rkv, rko, fmt, c.turned(1), v)
    got = c.run(rkv, ctx, g, fmt, before, c.rope(rkv, own=True))
    assert np.array_equal(got, after), f"{(got != after).sum()} bytes differ"


@pytest.mark.parametrize("rule", [0, 1])
@pytest.mark.parametrize("src", ["bf16", "f32"])
def test_without_rotation_q8_is_append_q8(rkv, rko, ctx, rule, src):
    import torch
    dtype = torch.bfloat16 if src == "bf16" else torch.float32
    c = Call(4, 2, 256, SPANS["odd"], 7, dtype, 0, False)
    q, k, v = c.parts()
    g, before, after = c.pages(rkv, rko, rkv.CACHE_Q8, k.float().cpu().numpy(), v.float().cpu().numpy(), rule)
    got = c.run(rkv, ctx, g, rkv.CACHE_Q8, before, None, rule=rule)
    assert np.array_equal(got, after)
    pages = torch.from_numpy(before).cuda()
    rkv.append_q8(ctx, g, pages, c.dev[1], c.dev[2], c.dev[3], k.contiguous(), v.contiguous(), rule=rule)
    assert np.array_equal(pages.cpu().numpy(), got)
    # and queries pass as they are
    q_out = torch.empty(q.shape, dtype=dtype, device="cuda")
    c.run(rkv, ctx, g, rkv.CACHE_Q8, before, None, q_out, rule=rule)
    assert torch.equal(q_out, q)


def test_row_by_row_is_all_at_once(rkv, rko, ctx):
    """Single tokens appended one call after the other give the chunk's bytes."""
    import torch
    c = Call(1, 2, 128, [(5, 43)], 8, torch.bfloat16, 128, True)
    g, before, after = c.pages(rkv, rko, rkv.CACHE_MX4, c.turned(1), c.xn[:, 3:])
    pages = torch.from_numpy(before).cuda()
    bt = torch.from_numpy(c.bt).cuda()
    _, k, v = c.parts()
    f, w = torch.from_numpy(c.freqs).cuda(), torch.from_numpy(c.w[1]).cuda()
    for i in range(43):
        sid, pos = (torch.tensor([t], dtype=torch.int32, device="cuda") for t in (0, 5 + i))
        rkv.append_rope(ctx, g, rkv.CACHE_MX4, pages, bt, sid, pos, k[i:i + 1], v[i:i + 1],
                        rkv.rope_args(128, f, k_norm=w, eps=1e-6))
    ctx.sync()
    assert np.array_equal(pages.cpu().numpy(), after)


@pytest.mark.parametrize("fmt", ["q8", "mx4"])
def test_bad_rows_are_reported_and_skipped(rkv, rko, ctx, fmt):
    import torch
    fmt = rkv.CACHE_Q8 if fmt == "q8" else rkv.CACHE_MX4
    for what, bit in (("seq", "0x4"), ("pos", "0x2"), ("page", "0x1")):
        c = Call(2, 2, 128, [(0, 40), (6, 30)], 9, torch.bfloat16, 128, False)
        seqs, pos, bt = c.seqs.copy(), c.pos.copy(), c.bt.copy()
        if what == "seq":
            c.seqs[[3, 20]] = [9, -1]
        elif what == "pos":
            c.pos[[0, 33]] = [-1, 32 * c.bt.shape[1]]
        else:
            c.bt[0, 1] = -1
        keep = [i for i in range(70) if 0 <= c.seqs[i] < 2 and 0 <= c.pos[i] < 32 * c.bt.shape[1] and
                0 <= c.bt[c.seqs[i], c.pos[i] // 32] < c.num_pages]
        k = mx4_ref.rope(c.xn[:, 2:4], c.freqs, c.pos[None], c.axis, False)
        full = (c.seqs, c.pos)
        c.seqs, c.pos = c.seqs[keep], c.pos[keep]
        g, before, after = c.pages(rkv, rko, fmt, k[keep], c.xn[keep, 4:])
        c.seqs, c.pos = full
        with pytest.raises(rkv.RkvError) as e:
            c.run(rkv, ctx, g, fmt, before, c.rope(rkv, own=True))
        assert e.value.status == rkv.ERR_BAD_BLOCK_TABLE and bit in e.value.message
        # the pages of the failed call
        pages = torch.from_numpy(before).cuda()
        q, kk, v = c.parts()
        rkv.append_rope(ctx, g, fmt, pages, torch.from_numpy(c.bt).cuda(), torch.from_numpy(c.seqs).cuda(),
                        torch.from_numpy(c.pos).cuda(), kk, v, c.rope(rkv, own=True))
        with pytest.raises(rkv.RkvError):
            ctx.sync()
        assert np.array_equal(pages.cpu().numpy(), after), what
        c.seqs, c.pos, c.bt = seqs, pos, bt


@pytest.mark.parametrize("fmt", ["q8", "mx4"])
@pytest.mark.parametrize("D", [128, 256])
def test_read_rows(rkv, rko, ctx, fmt, D):
    import torch
    fmt = rkv.CACHE_Q8 if fmt == "q8" else rkv.CACHE_MX4
    c = Call(2, 2, D, SPANS["odd"], 10, torch.float32, D, True)
    if fmt == rkv.CACHE_MX4:  # blocks that are not finite, tiny ones, huge ones
        c.x[4, 2:, 40] = float("inf")
        c.x[9, 4:] = 1e-30
        c.x[11, 4:] *= 1e6
        c.xn = c.x.cpu().numpy()
    k, v = c.turned(1).astype(np.float32), c.xn[:, 4:]
    g, before, after = c.pages(rkv, rko, fmt, k, v)
    got = c.run(rkv, ctx, g, fmt, before, c.rope(rkv))
    assert np.array_equal(got, after)
    pages, bt, sid, pos = c.dev
    for dtype in (torch.float32, torch.bfloat16):
        ko, vo = (torch.full(k.shape, 5.0, dtype=dtype, device="cuda") for _ in range(2))
        rkv.read_rows(ctx, g, fmt, pages, bt, sid, pos, ko, vo)
        one = torch.full(k.shape, 5.0, dtype=dtype, device="cuda")
        rkv.read_rows(ctx, g, fmt, pages, bt, sid, pos, None, one)
        assert torch.equal(torch.nan_to_num(one), torch.nan_to_num(vo))
        for o, x, kind in ((ko, k, "k"), (vo, v, "v")):
            if fmt == rkv.CACHE_MX4:
                want = torch.from_numpy(mx4_ref.quantize(x, kind)[2].astype(np.float32))
            else:
                rows = np.stack([rko.q8_encode(np.ascontiguousarray(x[:, h]).reshape(-1)) for h in range(2)])
                b = rows.reshape(2, len(c.pos), D // 32, 34)
                sc = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float32)
                val = sc * b[..., 2:].view(np.int8).astype(np.float32)
                want = torch.from_numpy(val.reshape(2, len(c.pos), D).transpose(1, 0, 2).copy())
            torch.testing.assert_close(o.cpu(), want.to(dtype), rtol=0, atol=0, equal_nan=True)


def test_read_rows_reports_bad_rows(rkv, rko, ctx):
    import torch
    c = Call(1, 1, 128, [(0, 9)], 11, torch.float32, 0, False)
    g, before, after = c.pages(rkv, rko, rkv.CACHE_MX4, c.xn[:, 1:2], c.xn[:, 2:])
    c.run(rkv, ctx, g, rkv.CACHE_MX4, before, None)
    pages, bt, sid, pos = c.dev
    pos[3] = 10 ** 6
    out = torch.full((9, 1, 128), 5.0, device="cuda")
    rkv.read_rows(ctx, g, rkv.CACHE_MX4, pages, bt, sid, pos, out, None)
    with pytest.raises(rkv.RkvError) as e:
        ctx.sync()
    assert "0x2" in e.value.message and (out[3] == 0).all() and (out[4] != 5).any()


def test_together_and_captured(rkv, ctx):
    """Tokens decoded one by one: append, then attention over what it wrote, in
    a graph replayed with the next rows, against the 64-bit formula."""
    import torch
    Hq, Hkv, D, PT, L, steps = 8, 2, 128, 32, 90, 5
    rng = np.random.default_rng(12)
    g = rkv.geometry(Hkv, D, PT, 8)
    alloc = rkv.Allocator(8, PT, 2, 4, seed=3)
    x = torch.from_numpy(rng.standard_normal((2, L + steps, Hq + 2 * Hkv, D)).astype(np.float32)).cuda().bfloat16()
    freqs = torch.from_numpy((100.0 ** (-np.arange(64) / 64)).astype(np.float32)).cuda()
    w = torch.from_numpy((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)).cuda()
    rope = rkv.rope_args(D, freqs, q_norm=w, k_norm=w, eps=1e-6)
    pages = torch.from_numpy(rng.integers(0, 256, 8 * rkv.mx4_page_bytes(g)).astype(np.uint8)).cuda()
    for s in range(2):
        alloc.reserve(s, L + steps)
    bt = torch.from_numpy(alloc.export()[0]).cuda()

    def rows(t, p0, n):
        v = t[:, p0:p0 + n].reshape(2 * n, Hq + 2 * Hkv, D)
        return v[:, :Hq], v[:, Hq:Hq + Hkv], v[:, Hq + Hkv:]
    sid = torch.tensor([0] * L + [1] * L, dtype=torch.int32, device="cuda")
    pos = torch.arange(L, dtype=torch.int32, device="cuda").repeat(2)
    q, k, v = rows(x, 0, L)
    rkv.append_rope(ctx, g, rkv.CACHE_MX4, pages, bt, sid, pos, k, v, rope)
    # the step's buffers
    now = x[:, L:L + 1].clone()
    step_pos = torch.full((2,), L, dtype=torch.int32, device="cuda")
    lens = step_pos + 1
    ids = torch.arange(2, dtype=torch.int32, device="cuda")
    q_out = torch.empty(2, 1, Hq, D, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(2, 1, Hq, D, device="cuda")
    a = rkv.decode_args(q_out, out, ids, D ** -0.5, L + steps)
    assert rkv.decode_mx4_workspace_bytes(g, a) == 0

    def step():
        q, k, v = rows(now, 0, 1)
        rkv.append_rope(ctx, g, rkv.CACHE_MX4, pages, bt, ids, step_pos, k, v, rope, q=q, q_out=q_out[:, 0])
        rkv.decode_mx4(ctx, g, pages, bt, lens, a)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    wn, fn = w.cpu().numpy(), freqs.cpu().numpy()
    axis = np.zeros(64, int)
    for i in range(steps):
        now.copy_(x[:, L + i:L + i + 1])
        step_pos.fill_(L + i)
        lens.fill_(L + i + 1)
        graph.replay()
        ctx.sync()
        got = out.cpu().numpy()
        for s in range(2):
            h = x[s, :L + i + 1].float().cpu().numpy()
            p = np.arange(L + i + 1)[None]
            kn = mx4_ref.quantize(mx4_ref.rope(h[:, Hq:Hq + Hkv], fn, p, axis, False, wn, 1e-6).astype(np.float32), "k")[2]
            vn = mx4_ref.quantize(h[:, Hq + Hkv:], "v")[2]
            qn = q_out[s].float().cpu().numpy()
            want = mx4_ref.attend(qn, kn, vn, D ** -0.5, [L + i + 1])
            assert np.abs(got[s] - want).max() < 2e-5
            turned = mx4_ref.rope(h[-1:, :Hq], fn, p[:, -1:], axis, False, wn, 1e-6)
            assert np.abs(qn - turned).max() <= 2.0 ** -8 * np.abs(turned).max()


@pytest.mark.parametrize("n", [3, 33003])
@pytest.mark.parametrize("src,out", [("float32", "bfloat16"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")])
def test_queries_are_rope_rows(rkv, ctx, n, src, out):
    """The append's queries bit for bit rkv_rope_rows', in one launch with the
    rows or by themselves; a large call's cached rows those of its parts."""
    import torch
    Hq, Hkv, D, PT, S = 5, 2, 128, 64, 7
    src, out = getattr(torch, src), getattr(torch, out)
    torch.manual_seed(n)
    x = torch.randn(n, Hq + 2 * Hkv, D, device="cuda").to(src)
    ids = (torch.arange(n, device="cuda") % S).sort().values.to(torch.int32)
    pos = torch.cat([torch.arange(int((ids == s).sum()), device="cuda") for s in range(S)]).to(torch.int32)
    f = torch.from_numpy((100.0 ** (-np.arange(32) / 32)).astype(np.float32)).cuda()
    w = torch.rand(D, device="cuda") + 0.5
    W = -(-(n // S + 1) // PT)
    g = rkv.geometry(Hkv, D, PT, S * W)
    bt = torch.randperm(S * W, device="cuda").to(torch.int32).view(S, W)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    got = []
    for parts in (1, 3):
        pages = torch.zeros(S * W * rkv.mx4_page_bytes(g), dtype=torch.uint8, device="cuda")
        q_out = torch.empty(n, Hq, D, dtype=out, device="cuda")
        cut = [n * i // parts for i in range(parts + 1)]
        for a, b in zip(cut, cut[1:]):
            rope = rkv.rope_args(64, f, pos[a:b], q_norm=w, k_norm=w, eps=1e-6)
            rkv.append_rope(ctx, g, rkv.CACHE_MX4, pages, bt, ids[a:b], pos[a:b], k[a:b], v[a:b], rope, q[a:b],
                            q_out[a:b])
        got.append((pages, q_out))
    want = torch.empty(n, Hq, D, dtype=out, device="cuda")
    rkv.rope_rows(ctx, rkv.rope_args(64, f, pos, q_norm=w, k_norm=w, eps=1e-6), q, None, want, None)
    ctx.sync()
    assert (got[0][1] == want).all() and (got[1][1] == want).all()
    assert (got[0][0] == got[1][0]).all()

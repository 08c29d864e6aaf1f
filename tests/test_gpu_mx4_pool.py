"""A pool of 4-bit pages: prompts in chunks, forks that share pages, rows
appended and attended, the copies of shared pages, streams in turn; every
result against the 64-bit statement over the sequence's own rows."""
import ctypes as C

import numpy as np
import pytest

import mx4_ref

pytestmark = pytest.mark.gpu

HQ, HKV, D, PT, LAYERS, W = 8, 2, 128, 32, 2, 8
# cached values are exact; a score is a sum of products of scale * |q||k| <= 16
# in all, over 9 f32 additions: off by at most 9 * 2^-24 * 16 = 8.6e-6, and so is
# a weight, with its 22 bits, relative to itself; an output by that times twice
# the weighted mean of |v - out|, which is below 1 here
TOL = 2e-5


class Model:
    """One sequence's rows, as a plain program would keep them."""

    def __init__(self, rope_of):
        self.rope_of, self.rows = rope_of, np.zeros((0, HQ + 2 * HKV, D), np.float32)

    def values(self, layer):
        k, v = self.rows[:, HQ:HQ + HKV], self.rows[:, HQ + HKV:] * np.float32(layer + 1)
        k = self.rope_of(k, np.arange(len(k))).astype(np.float32)
        return mx4_ref.quantize(k, "k")[2], mx4_ref.quantize(v, "v")[2]


@pytest.fixture
def setup(rkv, ctx):
    import torch
    pool = rkv.Pool(ctx, LAYERS, HKV, D, PT, 40, 6, W, seed=4, page_format=rkv.CACHE_MX4)
    freqs = (1000.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
    rope = rkv.rope_args(D, torch.from_numpy(freqs).cuda())

    def rope_of(x, pos):
        return mx4_ref.rope(x, freqs, np.asarray(pos)[None], np.zeros(D // 2, int), False)
    return pool, rope, rope_of


def _rows(rng, n):
    """bf16 values (as f32)."""
    import torch
    return torch.from_numpy(rng.standard_normal((n, HQ + 2 * HKV, D)).astype(np.float32)).bfloat16().float().numpy()


def _append(pool, rope, seq, start, x, q_out=None, layers=range(LAYERS), stream=None):
    import torch
    n = len(x)
    t = torch.from_numpy(x).cuda().bfloat16()
    ids = torch.full((n,), seq, dtype=torch.int32, device="cuda")
    pos = torch.arange(start, start + n, dtype=torch.int32, device="cuda")
    for layer in layers:
        v = (t[:, HQ + HKV:].float() * (layer + 1)).bfloat16()
        pool.append_rope(layer, ids, pos, t[:, HQ:HQ + HKV], v, rope, t[:, :HQ] if q_out is not None else None,
                         q_out, stream=stream)


def _check_rows(rkv, ctx, pool, seq, model):
    import torch
    n = len(model.rows)
    ids = torch.full((n,), seq, dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    for layer in range(LAYERS):
        k, v = torch.empty(n, HKV, D, device="cuda"), torch.empty(n, HKV, D, device="cuda")
        pool.read_rows(layer, ids, pos, k, v)
        ctx.sync()
        wk, wv = model.values(layer)
        assert (k.cpu().numpy() == wk).all() and (v.cpu().numpy() == wv).all()


def _check_decode(rkv, ctx, pool, models, q):
    import torch
    ids = torch.tensor(list(models), dtype=torch.int32, device="cuda")
    qt = torch.from_numpy(q).cuda().bfloat16()
    out = torch.empty(len(models), 1, HQ, D, device="cuda")
    a = rkv.decode_args(qt[:, None], out, ids, D ** -0.5, W * PT)
    for layer in range(LAYERS):
        pool.decode(layer, a)
        ctx.sync()
        for i, m in enumerate(models.values()):
            want = mx4_ref.attend(qt[i:i + 1].float().cpu().numpy(), *m.values(layer), D ** -0.5, [len(m.rows)])
            assert np.abs(out[i].cpu().numpy() - want).max() < TOL * (layer + 1)


def test_forks_copies_and_attention(rkv, ctx, setup):
    """A prompt of 70 rows, three forks (inside the last page, at a page's end,
    inside an earlier page), all grown in one window: copies of shared pages
    are whole 4-bit pages on both layers."""
    pool, rope, rope_of = setup
    rng = np.random.default_rng(8)
    models = {0: Model(rope_of)}
    pool.alloc.reserve(0, 70)
    pool.sync_tables()
    models[0].rows = _rows(rng, 70)
    _append(pool, rope, 0, 0, models[0].rows)
    for seq, n in ((1, 70), (2, 64), (3, 50)):
        pool.alloc.fork(0, seq, n)
        models[seq] = Model(rope_of)
        models[seq].rows = models[0].rows[:n]
    for seq, n in ((0, 5), (1, 9), (2, 20), (3, 3)):
        new = _rows(rng, n)
        at = len(models[seq].rows)
        pool.alloc.reserve(seq, at + n)
        models[seq].rows = np.concatenate([models[seq].rows, new])
    pool.sync_tables()
    for seq, n in ((0, 5), (1, 9), (2, 20), (3, 3)):
        at = len(models[seq].rows) - n
        _append(pool, rope, seq, at, models[seq].rows[at:])
    for seq, m in models.items():
        _check_rows(rkv, ctx, pool, seq, m)
    _check_decode(rkv, ctx, pool, models, rng.standard_normal((4, HQ, D)).astype(np.float32))


def test_chunks_then_steps_on_two_streams(rkv, ctx, setup):
    """A prompt in chunks (append, then attention over the rows before and in
    the chunk), then single tokens, the calls on two streams in turn: the pool
    orders them."""
    import torch
    pool, rope, rope_of = setup
    rng = np.random.default_rng(21)
    m = Model(rope_of)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    x = _rows(rng, 150)
    at = 0
    for i, n in enumerate((1, 60, 33, 40, 1, 1, 1)):
        s = streams[i % 2]
        pool.alloc.reserve(0, at + n)
        pool.sync_tables(stream=s)
        m.rows = x[:at + n]
        with torch.cuda.stream(s):
            q_out = torch.empty(n, HQ, D, dtype=torch.bfloat16, device="cuda")
            out = torch.empty(n, HQ, D, device="cuda")
            for layer in range(LAYERS):
                _append(pool, rope, 0, at, x[at:at + n], q_out, [layer], s)
                if n == 1:
                    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
                    a = rkv.decode_args(q_out[:, None], out[:, None], ids, D ** -0.5, W * PT)
                    pool.decode(layer, a, stream=s)
                else:
                    a = rkv.prefill_args([0], [at], [n], q_out, out, D ** -0.5)
                    assert pool.prefill_workspace_bytes(a) == rkv.prefill_mx4_workspace_bytes(pool.geometry, a)
                    pool.prefill(layer, a, stream=s)
                s.synchronize()
                want = mx4_ref.attend(q_out.float().cpu().numpy(), *m.values(layer), D ** -0.5,
                                      at + 1 + np.arange(n))
                assert np.abs(out.cpu().numpy() - want).max() < TOL * (layer + 1)
        at += n
    _check_rows(rkv, ctx, pool, 0, m)
    with pytest.raises(rkv.RkvError, match="length"):
        q = torch.zeros(2, HQ, D, dtype=torch.bfloat16, device="cuda")
        pool.prefill(0, rkv.prefill_args([0], [at], [2], q, torch.empty(2, HQ, D, device="cuda"), D ** -0.5))


def test_q8_pool_takes_rotated_rows(rkv, ctx):
    """The same calls on a pool of Q8_0 pages: the rotated keys' bytes are those
    of an append of the rotated rows."""
    import torch
    rng = np.random.default_rng(5)
    freqs = (1000.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
    rope = rkv.rope_args(D, torch.from_numpy(freqs).cuda())
    n = 45
    x = _rows(rng, n)
    turned = mx4_ref.rope(x[:, HQ:HQ + HKV], freqs, np.arange(n)[None], np.zeros(D // 2, int), False)
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    raw = []
    for rotate in (True, False):
        pool = rkv.Pool(ctx, 1, HKV, D, PT, 8, 1, 4, seed=4)
        pool.alloc.reserve(0, n)
        pool.sync_tables()
        v = torch.from_numpy(x[:, HQ + HKV:]).cuda()
        k = torch.from_numpy(x[:, HQ:HQ + HKV] if rotate else turned.astype(np.float32)).cuda()
        if rotate:
            pool.append_rope(0, ids, pos, k, v, rope)
        else:
            pool.append(0, ids, pos, k, v.contiguous())
        out = torch.empty(2, HKV * n * rkv.row_bytes(D), dtype=torch.uint8, device="cuda")
        for kind in (0, 1):
            pool.gather(0, 0, kind, out[kind])
        vals = torch.empty(2, n, HKV, D, device="cuda")
        pool.read_rows(0, ids, pos, vals[0], vals[1])
        ctx.sync()
        raw.append((out.cpu().numpy(), vals.cpu().numpy()))
    assert (raw[0][0] == raw[1][0]).all() and (raw[0][1] == raw[1][1]).all()
    # an 8-bit value is off by at most half a step of 1/127 of its block's largest, plus the f16 scale's rounding
    big = np.abs(turned.reshape(n, HKV, D // 32, 32)).max(-1).repeat(32, -1).reshape(n, HKV, D)
    assert (np.abs(raw[0][1][0] - turned) <= big * (0.5 / 127 + 2.0 ** -10)).all()


def test_refusals(rkv, ctx, setup):
    import torch
    pool, rope, _ = setup
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    k = torch.zeros(1, HKV, D, device="cuda")
    u8 = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    for call in (lambda: pool.append(0, ids, ids, k, k), lambda: pool.gather(0, 0, 0, u8)):
        with pytest.raises(rkv.RkvError, match="4-bit"):
            call()
    assert pool.r4kv_page_bytes(0, 0, 0) == 0
    lib = rkv.lib()
    head, expect, ref = rkv.R4kvHeader(), rkv.R4kvExpect(), C.c_int32()
    assert lib.rkv_pool_spill(pool.h, 0, 0, 0, 0, 0, C.byref(head), u8.data_ptr(), 4096, u8.data_ptr(), 4096,
                              None) == -4
    assert lib.rkv_pool_restore(pool.h, 0, u8.data_ptr(), 4096, C.byref(expect), u8.data_ptr(), 4096,
                                C.byref(ref), None) == -4
    a = rkv.AppendRopeArgs()
    a.format = rkv.CACHE_Q8
    assert lib.rkv_pool_append_rope(pool.h, 0, C.byref(a), None) == -1
    for layer in (-1, LAYERS):
        with pytest.raises(rkv.RkvError, match="layer"):
            pool.append_rope(layer, ids, ids, k, k)
        with pytest.raises(rkv.RkvError, match="layer"):
            pool.read_rows(layer, ids, ids, k, k)
    for kw in ({"page_memory": rkv.PAGES_HOST, "page_format": rkv.CACHE_MX4}, {"page_format": 2}):
        with pytest.raises(rkv.RkvError):
            rkv.Pool(ctx, 1, HKV, D, PT, 8, 1, 4, **kw)
    with pytest.raises(rkv.RkvError, match="page_tokens"):
        rkv.Pool(ctx, 1, HKV, D, 16, 8, 1, 4, page_format=rkv.CACHE_MX4)


def test_copy_pages(rkv, ctx):
    """Whole 4-bit pages on every layer, the others as they were."""
    import torch
    g = rkv.geometry(HKV, D, PT, 5)
    n = rkv.mx4_page_bytes(g)
    pages = torch.randint(0, 256, (2, 5, n), dtype=torch.uint8, device="cuda")
    want = pages.clone()
    want[:, 4], want[:, 0] = pages[:, 1], pages[:, 3]
    pairs = torch.tensor([[1, 4], [3, 0], [7, 2], [2, -1]], dtype=torch.int32, device="cuda")
    rkv.mx4_copy_pages(ctx, g, pages, 5 * n, 2, pairs, 4)
    ctx.sync()
    assert (pages == want).all()
    with pytest.raises(rkv.RkvError, match="stride"):
        rkv.mx4_copy_pages(ctx, g, pages, 5 * n - 16, 2, pairs, 4)


def test_host_pool_takes_rotated_rows(rkv, ctx):
    """Q8_0 pages in host memory: the bytes of the device pool's."""
    import torch
    rng = np.random.default_rng(6)
    rope = rkv.rope_args(D, torch.from_numpy((0.5 ** np.arange(D // 2)).astype(np.float32)).cuda())
    n = 37
    x = torch.from_numpy(_rows(rng, n)).cuda()
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    got = []
    for memory in (rkv.PAGES_DEVICE, rkv.PAGES_HOST):
        pool = rkv.Pool(ctx, 1, HKV, D, PT, 8, 1, 4, seed=4, page_memory=memory)
        pool.alloc.reserve(0, n)
        pool.sync_tables()
        pool.append_rope(0, ids, pos, x[:, HQ:HQ + HKV], x[:, HQ + HKV:], rope)
        k, v = torch.empty(n, HKV, D, device="cuda"), torch.empty(n, HKV, D, device="cuda")
        pool.read_rows(0, ids, pos, k, v)
        ctx.sync()
        got.append((k, v))
        pool.close()
    assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all() and (got[0][0] != 0).any()

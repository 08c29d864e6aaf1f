"""Performance cases of the position rotation, the rotating append and the attention over 4-bit pages.

A case is a dict of plain values; `kind` names the operator it stands for:

  rope     per-head norm of queries and keys and their position rotation (rope_rows)
  append   the same on the way into the paged cache, Q8_0 or 4-bit pages, V
           rows beside, the step's queries in the same call (append_rope);
           the cached rows are read back as values (read_rows)
  decode   attention of a step's rows over 4-bit pages, q_len > 1: causal
           verify (decode_mx4)
  prefill  attention of prompt chunks over 4-bit pages (prefill_mx4)

Projections and queries are N(0, 1), K and V with 1% of each head's channels
eight times larger; rotation frequencies base^(-2i/rot_dim).

The 4-bit pages: 32 values of a row share a power of two 2^e, e the smallest
with max|v| <= 7 * 2^e (K: -24..15, V: -22..7), and are held as E2M1 codes
(0, .5, 1, 1.5, 2, 3, 4, 6 and a sign bit), rounded to nearest, ties to the
even code.  A page holds, for every kv head, its K and then its V tiles of 32
tokens, a tile 16*D bytes of codes and D scale bytes:
  K codes  [j][h][b][m] 16 bytes: token 8*(m/4) + 4*j + m%4, dims
           128*h + 32*b .. +31, the even dim of a pair in the low nibble
  K scales [b][m][j][h] bytes e + 127
  V codes  [c][g][n][t] 4 bytes: dim 64*c + 32*(t/2) + 2*n + t%2, tokens
           8*g .. 8*g+7, the even token of a pair in the low nibble
  V scales [g][block][8 tokens] bytes 4*(e + 23)
"""
from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import torch

own = False
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
RANGE = {"k": (-24, 15), "v": (-22, 7)}  # exponents of the scales
TILE = 32
EPS = 1e-6


def listed():
    return [
        # one token of one request, deep in its context: launch and latency only
        dict(name="rope_one_token", kind="rope", rows=1, q_heads=24, kv_heads=4, head_dim=256,
             rot_dim=256, adjacent=False, axes=1, norm=True, src="bf16", out="bf16", far=262143),
        # the tokens of an image and its prompt: three axes over half of the dims
        dict(name="rope_image_4099", kind="rope", rows=4099, q_heads=16, kv_heads=2, head_dim=128,
             rot_dim=64, adjacent=True, axes=3, norm=True, src="bf16", out="bf16", far=9000),
        # the rows of a decode step of 64 requests, into the 8-bit cache
        dict(name="append_q8_step_64", kind="append", fmt="q8", rows=64, seqs=64, ctx=8000, q_heads=16,
             kv_heads=2, head_dim=256, rot_dim=256, adjacent=False, axes=1, norm=True, page=64, src="bf16",
             far=0),
        # eight prompt chunks of 512 tokens, into the 8-bit cache
        dict(name="append_q8_8x512", kind="append", fmt="q8", rows=4096, seqs=8, ctx=8192, q_heads=16,
             kv_heads=2, head_dim=256, rot_dim=64, adjacent=False, axes=1, norm=False, page=64, src="bf16",
             far=0),
        # long prompts of odd lengths, into the 4-bit cache
        dict(name="append_mx4_64k", kind="append", fmt="mx4", rows=65619, seqs=16, ctx=0, q_heads=16,
             kv_heads=2, head_dim=256, rot_dim=256, adjacent=False, axes=1, norm=True, page=64, src="bf16",
             far=0),
        # one short request alone on the GPU: launches and latency only
        dict(name="decode_one_short", kind="decode", batch=1, ctx_lo=300, ctx_hi=300, spread=0, q_len=1,
             q_heads=8, kv_heads=2, head_dim=128, page=32, q="f32", out="f32"),
        # a batch of chat requests of mixed lengths
        dict(name="decode_16_mixed", kind="decode", batch=16, ctx_lo=4096, ctx_hi=16384, spread=1, q_len=1,
             q_heads=16, kv_heads=2, head_dim=256, page=64, q="bf16", out="f32"),
        # one request over a very long document
        dict(name="decode_one_262k", kind="decode", batch=1, ctx_lo=262145, ctx_hi=262145, spread=0, q_len=1,
             q_heads=16, kv_heads=2, head_dim=256, page=64, q="bf16", out="f32"),
        # a full GPU of long requests
        dict(name="decode_64x32k", kind="decode", batch=64, ctx_lo=32768, ctx_hi=32768, spread=0, q_len=1,
             q_heads=16, kv_heads=2, head_dim=256, page=64, q="bf16", out="f32"),
        # speculative decoding: four draft rows per request, verified at once
        dict(name="verify_32x32k", kind="decode", batch=32, ctx_lo=32768, ctx_hi=32768, spread=0, q_len=4,
             q_heads=16, kv_heads=2, head_dim=256, page=64, q="bf16", out="bf16"),
        # chunked prefill of eight requests deep in their prompts
        dict(name="prefill_8x512", kind="prefill", batch=8, ctx_lo=8192, ctx_hi=8192, rows_lo=512,
             rows_hi=512, spread=0, q_heads=16, kv_heads=2, head_dim=256, page=64, q="bf16", out="f32"),
        # prompts of odd lengths arriving together, some just starting
        dict(name="prefill_6_mixed", kind="prefill", batch=6, ctx_lo=0, ctx_hi=3000, rows_lo=17, rows_hi=701,
             spread=2, q_heads=24, kv_heads=4, head_dim=256, page=32, q="bf16", out="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "decode", "decode", "decode", "prefill"])
    kv = rng.choice([1, 2, 2, 4, 4, 8])
    qh = kv * rng.choice([1, 2, 3, 4, 6, 8, 8])
    d = rng.choice([128, 256, 256])
    page = rng.choice([32, 64, 64, 128, 256])
    c = dict(kind=kind, q_heads=qh, kv_heads=kv, head_dim=d)
    rope = dict(rot_dim=rng.choice([d, d, d // 2, d // 4, 32, 80]), adjacent=rng.choice([False, False, True]),
                axes=rng.choice([1, 1, 2, 3, 4]), norm=rng.choice([True, False]),
                src=rng.choice(["bf16", "bf16", "f32"]))
    row = (qh + 2 * kv) * d
    if kind == "rope":
        c.update(rope, rows=_log(rng, 1, min(32768, (1 << 26) // row)), out=rng.choice(["bf16", "f32"]),
                 far=_log(rng, 10, 1000000))
    elif kind == "append":
        rows = _log(rng, 1, min(65536, (1 << 27) // row))
        c.update(rope, fmt=rng.choice(["q8", "mx4", "mx4"]), rows=rows, seqs=min(rows, rng.choice([1, 3, 8, 32, 64])),
                 ctx=rng.choice([0, 0, 1, 37, 1000, 8192]), page=page, far=rng.choice([0, 0, 100000]))
        if c["fmt"] == "q8":
            c["page"] = rng.choice([16, 32, 64, 64, 128])
    elif kind == "decode":
        q_len = rng.choice([1, 1, 1, 2, 3, 4])
        while q_len * (qh // kv) > 32:
            q_len -= 1
        batch = _log(rng, 1, 128)
        hi = _log(rng, 64, max(64, min(262144, (1 << 30) // (kv * d * batch))))
        c.update(batch=batch, ctx_lo=_log(rng, max(1, hi // 8), hi), ctx_hi=hi, spread=rng.randrange(1 << 20),
                 q_len=q_len, page=page, q=rng.choice(["bf16", "bf16", "f32"]), out=rng.choice(["f32", "bf16"]))
        c["ctx_lo"] = max(q_len, c["ctx_lo"])
        c["ctx_hi"] = max(c["ctx_lo"], c["ctx_hi"])
    else:
        batch = rng.choice([1, 1, 2, 3, 5, 8])
        rows = _log(rng, 8, 2048 if batch < 3 else 600)
        # rows * (context + rows) * heads * dim bounds the pass by the largest listed one
        room = (1 << 37) // (batch * rows * qh * d) - rows
        ctx = rng.choice([0, 1]) * _log(rng, 16, max(16, min(32768, room)))
        c.update(batch=batch, ctx_lo=ctx // 3, ctx_hi=ctx, rows_lo=max(1, rows // 3), rows_hi=rows,
                 spread=rng.randrange(1 << 20), page=page, q="bf16", out=rng.choice(["f32", "bf16"]))
    return c


# ---- sizes ----------------------------------------------------------------------------

def _spread(case, lo, hi, salt=0):
    """A length for each entry of the batch between lo and hi, spread over their logarithm."""
    rng = random.Random(case["spread"] * 2 + salt)
    return [_log(rng, lo, hi) if lo > 0 else (rng.randrange(0, hi + 1) if hi > 0 else 0)
            for _ in range(case["batch"])]


def _entries(case):
    """(tokens before the rows, rows) of each entry."""
    ctx = _spread(case, case["ctx_lo"], case["ctx_hi"])
    if case["kind"] == "decode":  # the rows are the last of the context's tokens
        return [(n - case["q_len"], case["q_len"]) for n in ctx]
    return list(zip(ctx, _spread(case, case["rows_lo"], case["rows_hi"], 1)))


def _append_rows(case):
    """(first position, rows) of each sequence of an append."""
    each, extra = divmod(case["rows"], case["seqs"])
    return [(case["ctx"] and case["ctx"] + 3 * s, each + (s < extra)) for s in range(case["seqs"])]


def _block_bytes(case):
    return 34 if case.get("fmt") == "q8" else 17


def work(case):
    qh, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    size = {"f32": 4, "bf16": 2}
    if case["kind"] == "rope":
        n = case["rows"] * (qh + kv) * d
        return {"bytes": n * (size[case["src"]] + size[case["out"]]), "flops": 7 * n}
    if case["kind"] == "append":
        rows, s = case["rows"], size[case["src"]]
        cached = 2 * kv * d // 32 * _block_bytes(case)
        # rows in, queries out, pages written, then read back as bf16 values
        return {"bytes": rows * ((qh + 2 * kv) * d * s + qh * d * 2 + 2 * cached + 2 * kv * d * 2),
                "flops": rows * (7 * (qh + kv) + 6 * kv) * d}
    io = size[case["q"]] + size[case["out"]]
    pairs = sum(n * ctx + n * (n + 1) // 2 for ctx, n in _entries(case))
    tokens = sum(ctx + n for ctx, n in _entries(case))
    rows = sum(n for _, n in _entries(case))
    return {"bytes": tokens * kv * 2 * (d // 32) * 17 + rows * qh * d * io, "flops": 4 * d * qh * pairs}


# ---- inputs ---------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) % (1 << 60))
    return g


def _i32(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def _loud(seed, heads, d):
    """Factors of a head's channels: 1% are eight times larger."""
    f = torch.ones((heads, d), device=DEV)
    f[torch.rand((heads, d), generator=_gen(seed, 7), device=DEV) < 0.01] = 8.0
    return f


def _kv(case, seed, s, n):
    """K and V rows [n][kv_heads][head_dim] of sequence s."""
    g, f = _gen(seed, 100 + s), _loud(seed, case["kv_heads"], case["head_dim"])
    k, v = (torch.randn((n, *f.shape), generator=g, device=DEV) * f for _ in range(2))
    return k, v


def _rope_inputs(case, seed):
    """Projections [rows][q | k | v], rotation and norm of a call."""
    qh, kv, d, rows = case["q_heads"], case["kv_heads"], case["head_dim"], case["rows"]
    x = torch.randn((rows, qh + 2 * kv, d), generator=_gen(seed, 1), device=DEV)
    x[:, qh:] *= _loud(seed, 2 * kv, d)
    half = case["rot_dim"] // 2
    freqs = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    g = _gen(seed, 2)
    weights = [1 + 0.1 * torch.randn(d, generator=g, device=DEV) for _ in range(2)] if case["norm"] else [None, None]
    axis = torch.arange(half, dtype=torch.int32, device=DEV) * case["axes"] // half if case["axes"] > 1 else None
    if case["far"]:
        positions = torch.randint(max(0, case["far"] - 4096), case["far"] + 1, (case["axes"], rows), generator=g,
                                  device=DEV, dtype=torch.int32)
    else:  # the rows' places in their sequences, on every axis
        at = _i32(p + i for p, n in _append_rows(case) for i in range(n))
        positions = at.expand(case["axes"], rows).contiguous()
    return dict(x=x.to(DTYPES[case["src"]]).reshape(rows, -1), freqs=freqs.float(), axis=axis, positions=positions,
                q_norm=weights[0], k_norm=weights[1])


def _tables(case, lens, seed):
    """Block tables of `lens` tokens per sequence over shuffled pages, and their number."""
    need = [-(-n // case["page"]) for n in lens]
    total = max(1, math.ceil(sum(need) * 1.1))
    order = torch.randperm(total, generator=_gen(seed, 3), device=DEV).to(torch.int32)
    bt, at = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32, device=DEV), 0
    for s, n in enumerate(need):
        bt[s, :n] = order[at:at + n]
        at += n
    return bt, total


def _exponent(amax, kind):
    m, x = torch.frexp(amax)  # amax = m * 2^x, m in [0.5, 1); 7 = 0.875 * 2^3
    return torch.where(m <= 0.875, x - 3, x - 2).where(amax > 0, -99).clamp(*RANGE[kind])


def _codes(y):
    """E2M1 codes of scaled values."""
    a = y.abs()
    c = sum((a > t).byte() for t in (0.25, 1.25, 2.5, 5.0)) + sum((a >= t).byte() for t in (0.75, 1.75, 3.5))
    return c + 8 * torch.signbit(y).byte()


def _tile_bytes(x, kind):
    """Page tiles [n/32][kv_heads][17*D] of rows x [n][kv_heads][D], n a multiple of 32."""
    n, kv, d = x.shape
    b = x.reshape(n, kv, d // 32, 32)
    e = _exponent(b.abs().amax(-1), kind)
    code = _codes(torch.ldexp(b, -e.unsqueeze(-1)))
    if kind == "k":  # tokens (m/4, j, m%4), blocks (h, b) -> [j][h][b][m][16 bytes]
        pair = code[..., 0::2] | code[..., 1::2] << 4
        c = pair.reshape(n // 32, 4, 2, 4, kv, d // 128, 4, 16).permute(0, 4, 2, 5, 6, 1, 3, 7)
        s = (e + 127).byte().reshape(n // 32, 4, 2, 4, kv, d // 128, 4).permute(0, 4, 6, 1, 3, 2, 5)
    else:  # token pairs; dims (c, t/2, n, t%2) -> [c][g][n][t][4 bytes]
        code = code.reshape(n // 32, 4, 4, 2, kv, d // 64, 2, 16, 2)
        pair = code[:, :, :, 0] | code[:, :, :, 1] << 4
        c = pair.permute(0, 3, 4, 1, 6, 5, 7, 2)
        s = (4 * (e + 23)).byte().reshape(n // 32, 4, 8, kv, d // 32).permute(0, 3, 1, 4, 2)
    return torch.cat([c.reshape(n // 32, kv, 16 * d), s.reshape(n // 32, kv, d)], -1)


def _prepare_attention(case, seed):
    page, kv, d = case["page"], case["kv_heads"], case["head_dim"]
    entries = _entries(case)
    lens = [c + n for c, n in entries]
    bt, total = _tables(case, lens, seed)
    pages = torch.zeros((total, kv, 2, page // TILE, 17 * d), dtype=torch.uint8, device=DEV)
    for s, n in enumerate(lens):
        used = -(-n // page)
        for i, (name, x) in enumerate(zip("kv", _kv(case, seed, s, n))):
            rows = torch.zeros((used * page, kv, d), device=DEV)
            rows[:n] = x
            tiles = _tile_bytes(rows, name).reshape(used, page // TILE, kv, 17 * d)
            pages[bt[s, :used].long(), :, i] = tiles.permute(0, 2, 1, 3)
    q = torch.randn((sum(n for _, n in entries), case["q_heads"], d), generator=_gen(seed, 11), device=DEV)
    return dict(case=case, pages=pages, bt=bt, lens=_i32(lens), seqs=_i32(range(len(lens))),
                q=q.to(DTYPES[case["q"]]), entries=entries)


def prepare(case, seed):
    if case["kind"] in ("decode", "prefill"):
        return _prepare_attention(case, seed)
    s = dict(_rope_inputs(case, seed), case=case)
    if case["kind"] == "append":
        placed = _append_rows(case)
        bt, total = _tables(case, [p + n for p, n in placed], seed)
        page = total * case["kv_heads"] * 2 * case["page"] * case["head_dim"] // 32 * _block_bytes(case)
        s.update(bt=bt, num_pages=total, pages=torch.zeros(page, dtype=torch.uint8, device=DEV),
                 seqs=_i32(i for i, (_, n) in enumerate(placed) for _ in range(n)),
                 at=_i32(p + i for p, n in placed for i in range(n)))
    return s


# ---- plain forms ----------------------------------------------------------------------

def _rotated(s, x, weight, t):
    """Rows x [rows][heads][D] normed and rotated, in type t."""
    case, x = s["case"], x.to(t)
    if weight is not None:
        eps = torch.tensor(EPS, dtype=torch.float32, device=DEV).to(t)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(t)
    rot, half = case["rot_dim"], case["rot_dim"] // 2
    at = s["positions"].double()
    at = at[0, :, None] if s["axis"] is None else at[s["axis"].long()].T
    angle = (at * s["freqs"].double())[:, None]
    cos, sin = torch.cos(angle).to(t), torch.sin(angle).to(t)
    if case["adjacent"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _heads(s):
    """The q, k and v rows of the projections."""
    case = s["case"]
    qh, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    return s["x"].reshape(-1, qh + 2 * kv, d).split([qh, kv, kv], 1)


def _plain_rope(s):
    t = DTYPES[s["case"]["out"]]
    q, k, _ = _heads(s)
    return {"q": _rotated(s, q, s["q_norm"], torch.float32).to(t),
            "k": _rotated(s, k, s["k_norm"], torch.float32).to(t)}


def _through_q8(x):
    """The values that Q8_0 blocks of f32 rows x stand for."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = b.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d > 0, 1.0 / d, 0.0)
    y = (b * inv).double()
    code = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-127, 127).float()
    return (d.half().float() * code).reshape(x.shape).bfloat16()


def _through_mx4(x, kind):
    """The values that 4-bit blocks of f32 rows x stand for."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    e = _exponent(b.abs().amax(-1), kind).unsqueeze(-1)
    code = _codes(torch.ldexp(b, -e))
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
    return torch.ldexp(table[code.long()], e).reshape(x.shape).bfloat16()


def _plain_append(s):
    q, k, v = _heads(s)
    k, v = _rotated(s, k, s["k_norm"], torch.float64).float(), v.float()
    if s["case"]["fmt"] == "q8":
        k, v = _through_q8(k), _through_q8(v)
    else:
        k, v = _through_mx4(k, "k"), _through_mx4(v, "v")
    return {"q": _rotated(s, q, s["q_norm"], torch.float32).bfloat16(), "k": k, "v": v}


def _unpacked(s):
    """K and V [entries][kv_heads][tokens][D] of the pages, f32."""
    case = s["case"]
    kv, d = case["kv_heads"], case["head_dim"]
    e = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
    pairs = torch.stack([e.repeat(16), e.repeat_interleave(16)], -1)  # byte -> its two values
    tiles = s["pages"][s["bt"].clamp(min=0).long()].permute(3, 0, 2, 1, 4, 5)  # K|V, entry, head, page, tile
    n = tiles.shape[1]
    tiles = tiles.reshape(2, n, kv, -1, 17 * d)
    t = tiles.shape[3]
    c, sc = tiles[..., :16 * d], tiles[..., 16 * d:]
    k = pairs[c[0].long()].reshape(n, kv, t, 2, d // 128, 4, 4, 4, 32)  # j h b m/4 m%4 dims
    ks = torch.exp2(sc[0].float() - 127).reshape(n, kv, t, 4, 4, 4, 2, d // 128)  # b m/4 m%4 j h
    k = k * ks.permute(0, 1, 2, 6, 7, 3, 4, 5).unsqueeze(-1)
    k = k.permute(0, 1, 2, 6, 3, 7, 4, 5, 8).reshape(n, kv, t * TILE, d)
    v = pairs[c[1].long()].reshape(n, kv, t, d // 64, 4, 16, 2, 2, 8)  # c g n t/2 t%2 tokens
    v = v.permute(0, 1, 2, 4, 8, 3, 6, 5, 7).reshape(n, kv, t, 4, 8, d // 32, 32)
    vs = torch.exp2(sc[1].float() / 4 - 23).reshape(n, kv, t, 4, d // 32, 8)
    v = v * vs.transpose(-1, -2).unsqueeze(-1)
    return k, v.reshape(n, kv, t * TILE, d)


def _plain_attention(s):
    case = s["case"]
    kv, d = case["kv_heads"], case["head_dim"]
    g = case["q_heads"] // kv
    counts = [n for _, n in s["entries"]]
    most, n = max(counts), len(counts)
    live = torch.arange(most, device=DEV) < _i32(counts)[:, None]
    q = torch.zeros((n, most, case["q_heads"], d), device=DEV)
    q[live] = s["q"].float()
    q = q.reshape(n, most, kv, g, d).transpose(1, 2).reshape(n, kv, most * g, d)
    k, v = _unpacked(s)
    seen = _i32([c for c, _ in s["entries"]])[:, None] + torch.arange(1, most + 1, device=DEV)
    hidden = torch.arange(k.shape[2], device=DEV) >= seen.repeat_interleave(g, 1)[:, None, :, None]
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1 / math.sqrt(d))
    p = p.masked_fill_(hidden, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.reshape(n, kv, most, g, d).transpose(1, 2).reshape(n, most, -1, d)
    return {"out": o[live].to(DTYPES[case["out"]])}


# ---- the framework's calls --------------------------------------------------------------

_held = {}


def _rkv():
    """The package and a device context, as a program keeps them."""
    if not _held:
        name = "remora_lab_amd"
        if name not in sys.modules:
            spec = importlib.util.spec_from_file_location(
                name, os.path.join(ROOT, "remora-lab_amd", "__init__.py"))
            mod = importlib.util.module_from_spec(spec)
            sys.modules[name] = mod
            spec.loader.exec_module(mod)
        _held.update(rkv=sys.modules[name], ctx=sys.modules[name].Ctx(0))
    return _held["rkv"], _held["ctx"]


def _plan(s):
    """Arguments, outputs and workspace of a program that makes the call again and again."""
    rkv, ctx = _rkv()
    case = s["case"]
    p = dict(rkv=rkv, ctx=ctx)
    if case["kind"] in ("rope", "append"):
        q, k, v = _heads(s)
        p["rope"] = rkv.rope_args(case["rot_dim"], s["freqs"], s["positions"], pair_axis=s["axis"],
                                  adjacent=case["adjacent"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        p.update(q=q, k=k, v=v)
        t = DTYPES[case.get("out", "bf16")]
        p["q_out"] = torch.empty(q.shape, dtype=t, device=DEV)
        p["k_out"] = torch.empty(k.shape, dtype=t, device=DEV)
        if case["kind"] == "append":
            p["v_out"] = torch.empty(v.shape, dtype=t, device=DEV)
            p["fmt"] = rkv.CACHE_Q8 if case["fmt"] == "q8" else rkv.CACHE_MX4
            p["g"] = rkv.geometry(case["kv_heads"], case["head_dim"], case["page"], s["num_pages"])
        return p
    p["g"] = rkv.geometry(case["kv_heads"], case["head_dim"], case["page"], s["pages"].shape[0])
    p["out"] = torch.empty(s["q"].shape, dtype=DTYPES[case["out"]], device=DEV)
    scale = 1 / math.sqrt(case["head_dim"])
    if case["kind"] == "decode":
        shape = (case["batch"], case["q_len"], case["q_heads"], case["head_dim"])
        most = max(c + n for c, n in s["entries"])

        def args(ws=None):
            return rkv.decode_args(s["q"].reshape(shape), p["out"].reshape(shape), s["seqs"], scale, most,
                                   q_len=case["q_len"], workspace=ws)
        need = rkv.decode_mx4_workspace_bytes(p["g"], args())
    else:
        def args(ws=None):
            ctx_lens, rows = zip(*s["entries"])
            return rkv.prefill_args(list(range(case["batch"])), ctx_lens, rows, s["q"], p["out"], scale, workspace=ws)
        need = rkv.prefill_mx4_workspace_bytes(p["g"], args())
    p["args"] = args(torch.empty(max(4, need), dtype=torch.uint8, device=DEV))
    return p


def _own(s):
    if "plan" not in s:
        s["plan"] = _plan(s)
    p, case = s["plan"], s["case"]
    rkv, ctx = p["rkv"], p["ctx"]
    if case["kind"] == "rope":
        rkv.rope_rows(ctx, p["rope"], p["q"], p["k"], p["q_out"], p["k_out"])
        return {"q": p["q_out"], "k": p["k_out"]}
    if case["kind"] == "append":
        rkv.append_rope(ctx, p["g"], p["fmt"], s["pages"], s["bt"], s["seqs"], s["at"], p["k"], p["v"], p["rope"],
                        q=p["q"], q_out=p["q_out"])
        rkv.read_rows(ctx, p["g"], p["fmt"], s["pages"], s["bt"], s["seqs"], s["at"], p["k_out"], p["v_out"])
        return {"q": p["q_out"], "k": p["k_out"], "v": p["v_out"]}
    if case["kind"] == "decode":
        rkv.decode_mx4(ctx, p["g"], s["pages"], s["bt"], s["lens"], p["args"])
    else:
        rkv.prefill_mx4(ctx, p["g"], s["pages"], s["bt"], s["bt"].shape[0], p["args"])
    return {"out": p["out"]}


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    return _plain_rope(s) if kind == "rope" else _plain_append(s) if kind == "append" else _plain_attention(s)


# ---- the definitions in 64 bits -----------------------------------------------------------

def _exact_rope(s, x, weight):
    """Normed rows as complex numbers, turned by e^(i*angle)."""
    x = x.double().clone()
    rot = s["case"]["rot_dim"]
    if weight is not None:
        x *= weight.double() / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    pairs = torch.arange(rot // 2, device=DEV)
    first, second = (2 * pairs, 2 * pairs + 1) if s["case"]["adjacent"] else (pairs, pairs + rot // 2)
    axis = torch.zeros_like(pairs) if s["axis"] is None else s["axis"].long()
    angle = s["positions"].double()[axis].T * s["freqs"].double()
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_q8(x):
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = b.abs().amax(-1, keepdim=True) / 127
    code = torch.where(d > 0, b / d, 0.0)
    code = torch.where(code < 0, torch.ceil(code - 0.5), torch.floor(code + 0.5))
    return (code * d.float().half().double()).reshape(x.shape)


def _exact_mx4(x, kind):
    """The nearest of the block's 15 values, the even code's where two are as near."""
    lo, hi = RANGE[kind]
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    scales = 2.0 ** torch.arange(lo, hi + 1, dtype=torch.float64, device=DEV)
    at = torch.searchsorted(7 * scales, top.contiguous()).clamp(max=hi - lo)
    scale = scales[at]
    a = (b.abs() / scale).unsqueeze(-1)
    values = torch.tensor(E2M1[0::2] + E2M1[1::2], dtype=torch.float64, device=DEV)  # even codes first
    near = torch.empty_like(b)
    for i in range(0, b.shape[0], 4096):
        near[i:i + 4096] = values[(a[i:i + 4096] - values).abs().argmin(-1)]
    return (near * b.sign() * scale).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("rope", "append"):
        q, k, v = _heads(s)
        r = {"q": _exact_rope(s, q, s["q_norm"]), "k": _exact_rope(s, k, s["k_norm"])}
        if case["kind"] == "append":
            q8 = case["fmt"] == "q8"
            r["k"] = _exact_q8(r["k"]) if q8 else _exact_mx4(r["k"], "k")
            r["v"] = _exact_q8(v.double()) if q8 else _exact_mx4(v.double(), "v")
        return r
    kv, d = case["kv_heads"], case["head_dim"]
    g, outs, at = case["q_heads"] // kv, [], 0
    for e, (ctx, n) in enumerate(s["entries"]):
        k, v = _kv(case, seed, e, ctx + n)
        k, v = _exact_mx4(k.double(), "k"), _exact_mx4(v.double(), "v")
        q = s["q"][at:at + n].double().reshape(n, kv, g, d)
        at += n
        later = torch.arange(ctx, ctx + n, device=DEV)[:, None] < torch.arange(ctx + n, device=DEV)
        out = torch.empty_like(q)
        for h in range(kv):
            score = (q[:, h].reshape(n * g, d) @ k[:, h].T / math.sqrt(d)).reshape(n, g, -1)
            score[later[:, None].expand_as(score)] = -math.inf
            out[:, h] = (torch.softmax(score, -1).reshape(n * g, -1) @ v[:, h]).reshape(n, g, d)
        outs.append(out.reshape(n, -1, d))
    return {"out": torch.cat(outs)}

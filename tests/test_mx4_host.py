"""CPU checks of the 4-bit pages: sizes, refusals before any device work, and
the reference's own layout against itself."""
import ctypes as C

import numpy as np
import pytest

import mx4_ref


def test_page_bytes(rkv):
    g = rkv.geometry(2, 256, 64, 10)
    assert rkv.mx4_page_bytes(g) == 2 * 2 * 64 * 256 // 32 * 17 == mx4_ref.page_bytes(2, 256, 64)
    assert rkv.mx4_page_bytes(rkv.geometry(3, 128, 32, 1)) == mx4_ref.page_bytes(3, 128, 32)
    assert rkv.mx4_page_bytes(rkv.geometry(2, 128, 16, 4)) == 0  # 16-token pages hold no whole tile


@pytest.mark.parametrize("D", [128, 256])
def test_layout_is_a_permutation(D):
    seen = np.zeros((17 * D, 2), int)
    for kind in "kv":
        seen[:] = 0
        for slot in range(32):
            off, nib = mx4_ref.code_place(D, kind, slot, np.arange(D))
            np.add.at(seen, (off, np.broadcast_to(nib, off.shape)), 1)
            seen[mx4_ref.scale_place(D, kind, slot, np.arange(D // 32))] += 1
        assert (seen == 1).all()


@pytest.mark.parametrize("kind", ["k", "v"])
def test_quantizer_rule(kind):
    lo, hi = mx4_ref.RANGE[kind]
    x = np.zeros((6, 32))
    x[0, 0] = 7.0          # the largest that a scale of 1 takes, rounds to 6
    x[1, 0] = 7.0001       # scale 2
    x[2, :8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5]  # ties to the even code
    x[3, 0] = 2.0 ** (hi + 10)  # saturates
    x[4, 0] = 2.0 ** (lo - 10)  # below the smallest scale
    x[5, 0] = np.inf
    _, e, v = mx4_ref.quantize(x, kind)
    assert e[0, 0] == 0 and v[0, 0] == 6 and e[1, 0] == 1 and v[1, 0] == 8
    assert v[2, :8].tolist() == [6, 0, 1, 1, 2, 2, 4, 4]
    assert v[3, 0] == 6 * 2.0 ** hi and (v[4] == 0).all() and e[4, 0] == lo and np.isnan(v[5]).all()


def _decode(rkv, g, **over):
    """rkv_decode_mx4 with no context and pointers that are never followed."""
    a = rkv.DecodeArgs(2, 64, 64, rkv.BF16, 1, 8, 0.1, 64, rkv.F32, 0, 4096, 64, 0, None, None)
    for k, v in over.items():
        setattr(a, k, v)
    st = rkv.lib().rkv_decode_mx4(None, C.byref(g), 64, 64, 8, 64, 2, C.byref(a), None)
    return st, rkv.lib().rkv_last_error().decode()


@pytest.mark.parametrize("over,status,text", [
    ({}, -1, "ctx is NULL"),
    ({"q_heads": 7}, -1, "q_heads=7"),
    ({"q_len": 5}, -4, "q_len=5"),
    ({"q_len": 4, "q_heads": 64}, -4, "rows per kv head"),
    ({"q_dtype": 2}, -4, "q_dtype"),
    ({"scale": float("nan")}, -1, "scale"),
    ({"partition_tokens": 48}, -1, "partition_tokens"),
    ({"q": None}, -1, "NULL"),
])
def test_decode_refusals(rkv, over, status, text):
    st, msg = _decode(rkv, rkv.geometry(2, 256, 64, 10), **over)
    assert st == status and text in msg and msg.startswith("rkv_decode_mx4")


def test_decode_refuses_append_and_small_pages(rkv):
    ap = rkv.AppendArgs(2, 64, 64, 64, 64, rkv.BF16, 0)
    st, msg = _decode(rkv, rkv.geometry(2, 256, 64, 10), append=C.pointer(ap))
    assert st == -4 and "append" in msg
    st, msg = _decode(rkv, rkv.geometry(2, 256, 16, 10))
    assert st == -4 and "page_tokens=16" in msg


def test_decode_workspace(rkv):
    g = rkv.geometry(2, 256, 64, 1000)

    def need(batch, longest):
        a = rkv.DecodeArgs(batch, 64, 64, rkv.BF16, 1, 16, 0.1, 64, rkv.F32, 0, longest, None, 0, None, None)
        return rkv.decode_mx4_workspace_bytes(g, a)
    assert need(64, 512) == 0 and need(1, 1) == 0 and need(1, 513) > 0
    assert need(1, 600) <= need(1, 4096) <= need(4, 4096) <= need(64, 32768)


def _prefill(rkv, g, **over):
    one = [(C.c_int32 * 1)(v) for v in (0, 100, 7, 0)]
    a = rkv.PrefillArgs(1, *[C.cast(x, rkv.I32P) for x in one], 7, 64, rkv.BF16, 8, 0.1, 64, rkv.F32, 0, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    st = rkv.lib().rkv_prefill_mx4(None, C.byref(g), 64, 64, 8, 2, C.byref(a), None)
    return st, rkv.lib().rkv_last_error().decode()


@pytest.mark.parametrize("over,status,text", [
    ({}, -1, "ctx is NULL"),
    ({"q_dtype": 0}, -4, "bf16"),
    ({"q_heads": 3}, -1, "q_heads=3"),
    ({"total_rows": 3}, -1, "total_rows=3"),
    ({"n_seqs": 65}, -1, "n_seqs=65"),
    ({"segment_tokens": 64}, -1, "workspace"),
    ({"workspace": 100}, -1, "256-byte"),
    ({"out": None}, -1, "NULL q/out"),
])
def test_prefill_refusals(rkv, over, status, text):
    st, msg = _prefill(rkv, rkv.geometry(2, 256, 64, 10), **over)
    assert st == status and text in msg and msg.startswith("rkv_prefill_mx4"), msg


def test_prefill_refuses_small_pages(rkv):
    st, msg = _prefill(rkv, rkv.geometry(2, 256, 16, 10))
    assert st == -4 and "page_tokens=16" in msg


def test_prefill_plan(rkv):
    """The split that rkv_prefill_mx4 plans, by its workspace: (m, l) rows padded
    to 256 bytes and o rows, rows * q_heads * segments of the entries that split."""
    import torch

    def rows(entries, G, kv, PT, seg=0):
        g = rkv.geometry(kv, 256, PT, 1 << 20)
        q = torch.empty(sum(r for _, r in entries), G * kv, 256, dtype=torch.bfloat16)
        a = rkv.prefill_args(list(range(len(entries))), [c for c, _ in entries], [r for _, r in entries], q, q, 1.0,
                             segment_tokens=seg)
        return rkv.prefill_mx4_workspace_bytes(g, a)

    def need(p):
        return (p * 8 + 255) // 256 * 256 + p * 1024
    assert rows([(8192, 512)] * 8, 8, 2, 64) == 0           # two equal units a CU
    assert rows([(0, 4096)], 8, 2, 64) == 0
    assert rows([(32768, 512)], 8, 2, 64, seg=-1) == 0
    assert rows([(32768, 512)], 8, 2, 64) == need(512 * 16 * 8)  # 64 units: 8 segments each, two a CU
    # among shorter ranges only the longest are cut, in two
    mixed = [(966, 173), (1242, 269), (422, 328), (2954, 567), (1622, 267), (1961, 526)]
    assert rows(mixed, 6, 4, 32) == need(24 * 2 * (567 + 526 + 267))

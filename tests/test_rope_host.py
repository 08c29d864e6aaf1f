"""CPU checks of the rotation's entry points: every refusal comes before any
device work, so they run here with no context and pointers never followed."""
import ctypes as C

import pytest

import mx4_ref  # noqa: F401  (the oracle imports on its own)


def _rope(rkv, **over):
    r = rkv.RopeArgs(128, 0, 64, 1, None, 64, None, None, rkv.F32, 1e-6)
    for k, v in over.items():
        setattr(r, k, v)
    return r


def _rows(rkv, rope=None, **over):
    a = rkv.RopeRowsArgs(3, 128, 4, 2, 64, 64, 0, 0, rkv.BF16, 64, 64, 0, 0, rkv.BF16)
    for k, v in over.items():
        setattr(a, k, v)
    rope = rope or _rope(rkv)
    return rkv.lib().rkv_rope_rows(None, C.byref(rope), C.byref(a), None), rkv.lib().rkv_last_error().decode()


@pytest.mark.parametrize("rope,rows,status,text", [
    ({}, {}, -1, "ctx is NULL"),
    ({"rot_dim": 12}, {}, -1, "rot_dim=12"),
    ({"rot_dim": 136}, {}, -1, "rot_dim=136"),
    ({"adjacent": 2}, {}, -1, "adjacent=2"),
    ({"n_axes": 5}, {}, -1, "n_axes=5"),
    ({"n_axes": 3}, {}, -1, "pair_axis"),
    ({"freqs": None}, {}, -1, "freqs"),
    ({"positions": None}, {}, -1, "positions"),
    ({"q_norm": 64, "norm_dtype": 7}, {}, -4, "norm_dtype"),
    ({"eps": -1.0}, {}, -1, "eps"),
    ({"eps": float("nan")}, {}, -1, "eps"),
    ({}, {"head_dim": 64}, -4, "head_dim=64"),
    ({}, {"n_rows": -1}, -1, "n_rows=-1"),
    ({}, {"src_dtype": 5}, -4, "src_dtype=5"),
    ({}, {"q_src": None}, -1, "q_src is NULL"),
    ({}, {"q_src": 66}, -1, "16 bytes"),
    ({}, {"k_stride": 260}, -1, "16 bytes"),
    ({}, {"k_stride": 248}, -1, "stride 248"),
    ({}, {"q_out": 72}, -1, "q_out"),
])
def test_rope_rows_refusals(rkv, rope, rows, status, text):
    st, msg = _rows(rkv, _rope(rkv, **rope), **rows)
    assert st == status and text in msg and msg.startswith("rkv_rope_rows"), msg


def test_no_rotation_needs_no_positions(rkv):
    st, msg = _rows(rkv, _rope(rkv, rot_dim=0, freqs=None, positions=None, q_norm=64))
    assert "ctx is NULL" in msg


def _append(rkv, g, **over):
    rope = _rope(rkv)
    a = rkv.AppendRopeArgs(5, 64, 64, 64, 64, 0, 0, rkv.BF16, rkv.CACHE_MX4, 0, C.pointer(rope), 64, 0, 8, 64,
                           rkv.BF16)
    for k, v in over.items():
        setattr(a, k, v)
    st = rkv.lib().rkv_append_rope(None, C.byref(g), 64, 64, 4, 2, C.byref(a), None)
    return st, rkv.lib().rkv_last_error().decode()


@pytest.mark.parametrize("over,status,text", [
    ({}, -1, "ctx is NULL"),
    ({"format": 2}, -4, "format=2"),
    ({"rule": 1}, -1, "rule=1"),
    ({"n_rows": -2}, -1, "n_rows=-2"),
    ({"seq_ids": None}, -1, "seq_ids"),
    ({"v_src": None}, -1, "v_src"),
    ({"k_stride": 128}, -1, "stride 128"),
    ({"q_heads": 0}, -1, "q_heads=0"),
    ({"q_out_dtype": 9}, -1, "q_out_dtype=9"),
    ({"q_out": None}, -1, "q_out is NULL"),
    ({"src_dtype": 3}, -4, "src_dtype=3"),
])
def test_append_refusals(rkv, over, status, text):
    st, msg = _append(rkv, rkv.geometry(2, 128, 32, 10), **over)
    assert st == status and text in msg and msg.startswith("rkv_append_rope"), msg


def test_append_formats_and_pages(rkv):
    g16 = rkv.geometry(2, 128, 16, 10)
    st, msg = _append(rkv, g16)
    assert st == -4 and "page_tokens=16" in msg
    st, msg = _append(rkv, g16, format=rkv.CACHE_Q8, rule=rkv.Q8_HARSERVE)
    assert "ctx is NULL" in msg


def test_read_rows_refusals(rkv):
    g = rkv.geometry(2, 128, 32, 10)

    def read(g=g, fmt=rkv.CACHE_MX4, n=3, seqs=64, k=64, dtype=rkv.F32):
        st = rkv.lib().rkv_read_rows(None, C.byref(g), fmt, 64, 64, 4, 2, n, seqs, 64, k, 64, dtype, None)
        return st, rkv.lib().rkv_last_error().decode()
    assert "ctx is NULL" in read()[1]
    assert read(fmt=5)[0] == -4 and read(n=-1)[0] == -1 and read(seqs=None)[0] == -1
    assert read(k=72)[0] == -1 and read(dtype=2)[0] == -4
    assert read(g=rkv.geometry(2, 128, 16, 10))[0] == -4


def test_binding_refuses_what_it_would_misread(rkv):
    import torch
    f = torch.ones(64)
    pos = torch.zeros(3, dtype=torch.int32)
    rope = rkv.rope_args(128, f, pos)
    q = torch.zeros(3, 4, 128)
    with pytest.raises(TypeError):
        rkv.rope_args(128, f.double(), pos)
    with pytest.raises(TypeError):
        rkv.rope_args(128, f, pos.long())
    with pytest.raises(ValueError):
        rkv.rope_args(64, f, pos)

    class Ctx:
        h, device = None, -1  # (a CPU tensor's device number)
    for bad in (q.half(), ):
        with pytest.raises((TypeError, ValueError)):
            rkv.rope_rows(Ctx, rope, bad, None, bad, None)
    with pytest.raises(ValueError):  # heads apart
        rkv.rope_rows(Ctx, rope, torch.zeros(3, 8, 128)[:, ::2], None, q, None)
    with pytest.raises(ValueError):  # other rows than positions
        rkv.rope_rows(Ctx, rope, torch.zeros(4, 4, 128), None, torch.zeros(4, 4, 128), None)
    class Gpu(Ctx):
        device = 0
    with pytest.raises(ValueError, match="device"):
        rkv.rope_rows(Gpu, rope, q, None, q, None)
    g = rkv.geometry(4, 128, 32, 3)
    bt = torch.zeros(1, 1, dtype=torch.int32)
    for k, v, sid in ((q, q[:, :2], pos), (q.double(), q.double(), pos), (q, q, pos.long()), (q, q, pos[:2])):
        with pytest.raises((TypeError, ValueError, KeyError)):
            rkv.append_rope(Ctx, g, rkv.CACHE_MX4, bt, bt, sid, pos, k, v, rope, stream=0)
    with pytest.raises(ValueError):
        rkv.read_rows(Ctx, g, rkv.CACHE_MX4, bt, bt, pos, pos, q[:, :, :64], None, stream=0)


def test_pages_in_whole_words_and_row_limits(rkv):
    """Pages off 16 bytes and calls beyond the documented sizes are refused."""
    g = rkv.geometry(2, 128, 32, 10)
    rope = _rope(rkv)
    lib, err = rkv.lib(), lambda: rkv.lib().rkv_last_error().decode()
    a = rkv.AppendRopeArgs(5, 64, 64, 64, 64, 0, 0, rkv.BF16, rkv.CACHE_MX4, 0, C.pointer(rope), 64, 0, 8, 64, rkv.BF16)
    assert lib.rkv_append_rope(None, C.byref(g), 72, 64, 4, 2, C.byref(a), None) == -1 and "pages" in err()
    assert lib.rkv_read_rows(None, C.byref(g), 1, 72, 64, 4, 2, 3, 64, 64, 64, 64, 0, None) == -1 and "pages" in err()
    assert lib.rkv_read_rows(None, C.byref(g), 1, 64, 64, 4, 2, (1 << 23) + 1, 64, 64, 64, 64, 0, None) == -1
    assert "n_rows" in err()
    for over in ({"n_rows": (1 << 23) + 1}, {"q_heads": 1 << 15}):
        assert _append(rkv, g, **over)[0] == -1
        assert _rows(rkv, rope, **over)[0] == -1
    d = rkv.DecodeArgs(2, 64, 64, rkv.BF16, 1, 8, 0.1, 64, rkv.F32, 0, 4096, 64, 0, None, None)
    assert lib.rkv_decode_mx4(None, C.byref(g), 72, 64, 8, 64, 2, C.byref(d), None) == -1 and "pages" in err()
    p = rkv.PrefillArgs()
    assert lib.rkv_prefill_mx4(None, C.byref(g), 72, 64, 8, 2, C.byref(p), None) == -1 and "pages" in err()


def test_binding_refuses_other_memory(rkv):
    """Rows over each other, and tensors of another device than the context's."""
    import torch

    class Cpu:
        h, device = None, -1

    class Gpu:
        h, device = None, 0
    f, pos = torch.ones(64), torch.zeros(3, dtype=torch.int32)
    rope = rkv.rope_args(128, f, pos)
    x = torch.zeros(3, 4, 128)
    with pytest.raises(ValueError, match="follow each other"):
        rkv.rope_rows(Cpu, rope, torch.zeros(1, 4, 128).expand(3, 4, 128), None, x, None, stream=0)
    with pytest.raises(ValueError, match="rope"):
        rkv.rope_rows(Gpu, rope, x, None, x, None, stream=0)
    g = rkv.geometry(4, 128, 32, 3)
    bt, pages = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(64, dtype=torch.uint8)
    over = torch.zeros(516).as_strided((3, 4, 128), (2, 128, 1))
    with pytest.raises(ValueError, match="follow each other"):
        rkv.append_rope(Cpu, g, rkv.CACHE_MX4, pages, bt, pos, pos, x, over, stream=0)
    with pytest.raises(ValueError, match="device 0"):
        rkv.read_rows(Gpu, g, rkv.CACHE_MX4, pages, bt, pos, pos, None, None, stream=0)
    with pytest.raises(ValueError, match="device 0"):
        rkv.append_rope(Gpu, g, rkv.CACHE_MX4, pages, bt, pos, pos, x, x, stream=0)
    # what fits reaches the library, which refuses the missing context
    buf = torch.zeros(4096, dtype=torch.uint8)
    pages = buf[-buf.data_ptr() % 16:]
    for call in (lambda: rkv.rope_rows(Cpu, rope, x, None, x, None, stream=0),
                 lambda: rkv.append_rope(Cpu, g, rkv.CACHE_MX4, pages, bt, pos, pos, x, x, rope, stream=0),
                 lambda: rkv.read_rows(Cpu, g, rkv.CACHE_MX4, pages, bt, pos, pos, x, None, stream=0)):
        with pytest.raises(rkv.RkvError, match="ctx is NULL"):
            call()

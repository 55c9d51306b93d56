"""The rotating cache write, and attention over a cache in 8 bits with a scale for each block, without
a GPU: invalid arguments are rejected with the documented status codes before any device access (the
pointers below are never read), sizes, and the torch ops' checks, real and fake (meta) kernels alike."""
import ctypes as C

import pytest
import torch

import voltattn_amd as va
import voltattn_amd.torch_ops  # noqa: F401

VA_OK, VA_EINVAL, VA_EALIGN, VA_ENULL, VA_ERANGE = 0, 1, 2, 3, 4
B8 = va.B8
FMTS = {f.label: int(f) for f in va.Fmt} | {"b8+": B8}
ops = torch.ops.voltattn


def _message():
    return va.lib.va_last_error().decode()


def test_sizes_of_the_block_format():
    assert va.lib.va_fmt_name(B8).decode() == "b8+"
    assert va.lib.va_page_bytes(B8, 8, 256, 128) == 8 * 256 * 128
    assert va.lib.va_page_scale_bytes(B8, 8, 256, 128, 64) == 8 * 256 // 64 * 2
    assert va.lib.va_page_scale_bytes(B8, 8, 256, 64, 32) == 8 * 256 // 32 * 2


def test_what_has_rows_with_scales_of_their_own_refuses_the_block_format():
    shape = va._PagedShape(4, 32, 8, 128, 32, 64, 64, 256, 4096)
    n = C.c_int()
    assert va.lib.va_pick_splits_paged(B8, C.byref(shape), C.byref(n)) == VA_EINVAL
    p = [C.c_void_p(0x1000 * i) for i in range(1, 6)]
    assert va.lib.va_append_kv(B8, p[0], 1, p[1], p[2], C.byref(shape), p[3], p[4], None) == VA_EINVAL
    b = va._TreeBufs(*(0x1000 * i for i in range(1, 12)))
    assert va.lib.va_decode_tree(B8, C.byref(b), C.byref(shape), 4, None) == VA_EINVAL


# -------------------------------------------------------------------- append --
def _rope(fmt="b8+", bufs=None, **kw):
    s = dict(B=2, total=100, Hq=8, Hkv=2, D=128, G=32, page_rows=64, max_pages=8, num_pages=32, rot=128, interleaved=0, scaling=1.0,
             q_row=1024, q_head=128, k_row=256, k_head=128, v_row=256, v_head=128)
    s.update(kw)
    b = dict(q=0x1000, k=0x2000, v=0x3000, cu=0x4000, start=0x5000, positions=0, block_table=0x6000, inv_freq=0x7000, q_out=0x8000,
             k_out=0x9000, kp=0x10000, vp=0x20000, ks=0x30000, vs=0x40000)
    b.update(bufs or {})
    return va.lib.va_append_rope(FMTS.get(fmt, fmt), C.byref(va._RopeBufs(*b.values())), C.byref(va._RopeShape(*s.values())), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(fmt=7), VA_EINVAL, "invalid format"), (dict(fmt=-1), VA_EINVAL, "invalid format"), (dict(fmt=17), VA_EINVAL, "invalid format"),
    (dict(B=0), VA_EINVAL, "B, Hq and Hkv"), (dict(Hq=0), VA_EINVAL, "B, Hq and Hkv"), (dict(Hkv=0), VA_EINVAL, "B, Hq and Hkv"),
    (dict(total=-1), VA_EINVAL, "total"), (dict(D=96), VA_EINVAL, "D must be"), (dict(G=16), VA_EINVAL, "G must be"),
    (dict(G=48, fmt="q4+"), VA_EINVAL, "G must be"), (dict(page_rows=96, G=64), VA_EINVAL, "multiple of G"), (dict(page_rows=0), VA_EINVAL, "page_rows"),
    (dict(max_pages=0), VA_EINVAL, "max_pages"), (dict(num_pages=0), VA_EINVAL, "num_pages"),
    (dict(num_pages=1 << 30, page_rows=1 << 20), VA_ERANGE, "pool too large"),
    (dict(rot=8), VA_EINVAL, "rot must"), (dict(rot=144), VA_EINVAL, "rot must"), (dict(rot=24), VA_EINVAL, "rot must"),
    (dict(interleaved=2), VA_EINVAL, "interleaved"), (dict(q_row=1028), VA_EINVAL, "strides"), (dict(v_head=-8), VA_EINVAL, "strides"),
    (dict(bufs=dict(cu=0)), VA_EINVAL, "without cu"),
    (dict(Hq=1 << 25), VA_ERANGE, "heads too large"), (dict(total=2 ** 31 - 1, Hq=1 << 10), VA_ERANGE, "too large"),
    (dict(total=0), VA_OK, ""),                              # nothing to write: no launch
])
def test_rope_shape(kw, code, msg):
    assert _rope(**kw) == code
    assert code == VA_OK or msg in _message()


@pytest.mark.parametrize("fmt,field,ptr,code", [
    *[("b8+", n, 0, VA_ENULL) for n in ("q", "k", "v", "start", "block_table", "inv_freq", "q_out", "kp", "vp", "ks", "vs")],
    ("q4+", "ks", 0, VA_ENULL), ("q8", "vs", 0, VA_ENULL),
    *[("b8+", n, 0x1008, VA_EALIGN) for n in ("q", "k", "v", "q_out", "k_out", "inv_freq", "kp", "vp")],
    ("q4+", "kp", 0x10002, VA_EALIGN), ("f16+", "vp", 0x10008, VA_EALIGN),
    *[("b8+", n, 0x5002, VA_EALIGN) for n in ("cu", "start", "positions", "block_table")],
    ("b8+", "ks", 0x30001, VA_EALIGN), ("q8+", "vs", 0x40001, VA_EALIGN),
])
def test_rope_buffers(fmt, field, ptr, code):
    assert _rope(fmt, {field: ptr}) == code


def test_rope_null_structs():
    b, s = va._RopeBufs(), va._RopeShape()
    assert va.lib.va_append_rope(B8, None, C.byref(s), None) == VA_ENULL
    assert va.lib.va_append_rope(B8, C.byref(b), None, None) == VA_ENULL


# -------------------------------------------------------------------- attend --
def _attend(fmt="b8+", total=40, bufs=None, ws=False, **kw):
    s = dict(B=4, Hq=32, Hkv=8, D=128, G=32, page_rows=64, max_pages=64, num_pages=256, max_seq_len=4096)
    s.update(kw)
    shape = va._PagedShape(*s.values())
    if ws:
        return va.lib.va_attend_ws_bytes(FMTS.get(fmt, fmt), C.byref(shape), total)
    b = dict(k=0x10000, v=0x20000, sk=0x30000, sv=0x40000, block_table=0x50000, cu=0x60000, seq_lens=0x70000, q=0x80000, out=0x90000, ws=0xA0000)
    b.update(bufs or {})
    return va.lib.va_attend_paged(FMTS.get(fmt, fmt), C.byref(va._AttendBufs(*b.values())), C.byref(shape), total, None)


SHAPES = [
    (dict(fmt=9), VA_EINVAL, "invalid format"), (dict(fmt="q8+"), VA_EINVAL, "b8+ only"), (dict(fmt="f16"), VA_EINVAL, "b8+ only"),
    (dict(total=-1), VA_EINVAL, "total"), (dict(B=0), VA_EINVAL, "B and Hkv"), (dict(Hkv=0), VA_EINVAL, "B and Hkv"),
    (dict(Hq=30), VA_EINVAL, "multiple of Hkv"), (dict(Hq=0), VA_EINVAL, "multiple of Hkv"), (dict(D=96), VA_EINVAL, "D must be"),
    (dict(G=16), VA_EINVAL, "G must be"), (dict(G=128), VA_EINVAL, "G must be"), (dict(page_rows=96), VA_EINVAL, "power of two"),
    (dict(page_rows=32), VA_EINVAL, "power of two"), (dict(max_seq_len=4097), VA_EINVAL, "max_seq_len"), (dict(max_seq_len=-1), VA_EINVAL, "max_seq_len"),
    (dict(max_pages=1 << 26), VA_ERANGE, "below 2^31"), (dict(num_pages=1 << 28, page_rows=1 << 20, max_pages=1), VA_ERANGE, "pool too large"),
    (dict(total=2 ** 31 - 1), VA_ERANGE, "total*Hq"),
    (dict(B=1 << 14, total=1 << 14, Hkv=1 << 5, Hq=1 << 5, max_pages=1 << 20, max_seq_len=1 << 26), VA_ERANGE, "batch too large"),
]


@pytest.mark.parametrize("kw,code,msg", SHAPES + [(dict(bufs=dict(cu=0)), VA_EINVAL, "without cu"), (dict(total=0), VA_OK, "")])
def test_attend_shape(kw, code, msg):
    assert _attend(**kw) == code
    assert code == VA_OK or msg in _message()
    if "bufs" not in kw:
        assert _attend(ws=True, **kw) == 0


@pytest.mark.parametrize("field,ptr,code", [
    *[(n, 0, VA_ENULL) for n in ("k", "v", "sk", "sv", "block_table", "seq_lens", "q", "out", "ws")],
    *[(n, 0x10008, VA_EALIGN) for n in ("k", "v", "q", "out", "ws")],
    *[(n, 0x10002, VA_EALIGN) for n in ("sk", "sv", "block_table", "cu", "seq_lens")],
])
def test_attend_buffers(field, ptr, code):
    assert _attend(bufs={field: ptr}) == code


def test_attend_null_structs():
    b, s = va._AttendBufs(), va._PagedShape(4, 32, 8, 128, 32, 64, 64, 256, 4096)
    assert va.lib.va_attend_paged(B8, None, C.byref(s), 4, None) == VA_ENULL
    assert va.lib.va_attend_paged(B8, C.byref(b), None, 4, None) == VA_ENULL
    assert va.lib.va_attend_ws_bytes(B8, None, 4) == 0


def test_attend_workspace_does_not_grow_with_the_batch():
    a = _attend(ws=True, total=4096)
    assert a > 0 and a % 16 == 0
    assert _attend(ws=True, total=1 << 14, B=16, num_pages=1024) == a
    assert _attend(ws=True, total=1 << 24, B=64, num_pages=4096) <= 1 << 28


# --------------------------------------------------------------------- torch --
def _t(shape, dtype=torch.float16, device="cpu"):
    return torch.zeros(shape, dtype=dtype, device=device)


E4 = torch.float8_e4m3fn


def _rope_args(device, fmt="b8+", group=32, **kw):
    a = dict(q=_t((10, 8, 128), device=device), k=_t((10, 2, 128), device=device), v=_t((10, 2, 128), device=device),
             freq=_t((64,), torch.float32, device), cu=_t((4,), torch.int32, device), start=_t((3,), torch.int32, device), positions=None,
             table=_t((3, 5), torch.int32, device), kp=_t((9, 2, 64, 128), E4, device), vp=_t((9, 2, 64, 128), E4, device),
             ks=_t((9, 2, 2), device=device), vs=_t((9, 2, 2), device=device))
    a.update(kw)
    return list(a.values()) + [fmt, group]


def _attend_args(device, fmt="b8+", cap=300, group=32, **kw):
    a = dict(q=_t((10, 8, 128), device=device), kp=_t((9, 2, 64, 128), E4, device), vp=_t((9, 2, 64, 128), E4, device),
             ks=_t((9, 2, 2), device=device), vs=_t((9, 2, 2), device=device), table=_t((3, 5), torch.int32, device),
             cu=_t((4,), torch.int32, device), lens=_t((3,), torch.int32, device))
    a.update(kw)
    return list(a.values()) + [fmt, cap, group]


BAD = [
    ("append_rope", _rope_args, dict(q=((10, 128),)), "q must be"), ("append_rope", _rope_args, dict(q=((10, 8, 96),)), "D must be"),
    ("append_rope", _rope_args, dict(q=((10, 8, 128), torch.float32)), "q has dtype"), ("append_rope", _rope_args, dict(k=((11, 2, 128),)), "k has shape"),
    ("append_rope", _rope_args, dict(k=((10, 0, 128),)), "at least one head"), ("append_rope", _rope_args, dict(v=((10, 3, 128),)), "v has shape"),
    ("append_rope", _rope_args, dict(freq=((4,), torch.float32)), "multiple of 8"), ("append_rope", _rope_args, dict(freq=((72,), torch.float32)), "multiple of 8"),
    ("append_rope", _rope_args, dict(freq=((64,), torch.float64)), "inv_freq has dtype"), ("append_rope", _rope_args, dict(cu=((3,), torch.int32)), "cu_seqlens"),
    ("append_rope", _rope_args, dict(cu=None), "a row to each sequence"), ("append_rope", _rope_args, dict(start=((3, 1), torch.int32)), "start"),
    ("append_rope", _rope_args, dict(positions=((9,), torch.int32)), "positions"), ("append_rope", _rope_args, dict(positions=((10,), torch.int64)), "positions has dtype"),
    ("append_rope", _rope_args, dict(table=((2, 5), torch.int32)), "block_table"), ("append_rope", _rope_args, dict(kp=((9, 2, 64, 128), torch.uint8)), "k_pages has dtype"),
    ("append_rope", _rope_args, dict(kp=((9, 2, 48, 128), E4)), "multiple of group"), ("append_rope", _rope_args, dict(vp=((9, 2, 64, 64), E4)), "v_pages"),
    ("append_rope", _rope_args, dict(ks=((9, 2, 64, 4),)), "k_scale_pages"), ("append_rope", _rope_args, dict(vs=None), "v_scale_pages is required"),
    ("append_rope", _rope_args, dict(group=16), "group must be"), ("append_rope", _rope_args, dict(fmt="q8+"), "k has"),
    ("attend_paged", _attend_args, dict(fmt="q8+"), "b8\\+ only"), ("attend_paged", _attend_args, dict(q=((10, 128),)), "q must be"),
    ("attend_paged", _attend_args, dict(q=((10, 7, 128),)), "multiple of K/V heads"), ("attend_paged", _attend_args, dict(q=((10, 8, 96),)), "D must be"),
    ("attend_paged", _attend_args, dict(kp=((9, 2, 64, 128),)), "k_pages has dtype"), ("attend_paged", _attend_args, dict(kp=((9, 2, 128), E4)), "k_pages must be"),
    ("attend_paged", _attend_args, dict(vp=((9, 2, 64, 64), E4)), "v_pages"), ("attend_paged", _attend_args, dict(ks=((9, 2, 1),)), "k_scale_pages"),
    ("attend_paged", _attend_args, dict(vs=((9, 2, 2), torch.float32)), "v_scale_pages has dtype"), ("attend_paged", _attend_args, dict(vs=None), "v_scale_pages"),
    ("attend_paged", _attend_args, dict(table=((15,), torch.int32)), "block_table"), ("attend_paged", _attend_args, dict(lens=((4,), torch.int32)), "seq_lens"),
    ("attend_paged", _attend_args, dict(cu=((3,), torch.int32)), "cu_seqlens"), ("attend_paged", _attend_args, dict(cu=None), "a row to each sequence"),
    ("attend_paged", _attend_args, dict(group=128), "group must be"),
]


@pytest.mark.parametrize("device", ["cpu", "meta"])
@pytest.mark.parametrize("name,args,kw,msg", BAD)
def test_torch_checks(device, name, args, kw, msg):
    kw = {k: _t(v[0], v[1] if len(v) > 1 else torch.float16, device) if isinstance(v, tuple) else v for k, v in kw.items()}
    with pytest.raises((RuntimeError, TypeError), match=msg):
        getattr(ops, name)(*args(device, **kw))


@pytest.mark.parametrize("name,args", [("append_rope", _rope_args), ("attend_paged", _attend_args)])
def test_no_cpu_fallback_and_fake_shapes(name, args):
    with pytest.raises(RuntimeError, match="gfx950"):
        getattr(ops, name)(*args("cpu"))
    out = getattr(ops, name)(*args("meta"))
    if name == "append_rope":
        assert [tuple(t.shape) for t in out] == [(10, 8, 128), (0, 2, 128)]
        out = getattr(ops, name)(*args("meta"), False, True)
        assert [tuple(t.shape) for t in out] == [(10, 8, 128), (10, 2, 128)] and all(t.dtype == torch.float16 for t in out)
    else:
        assert tuple(out.shape) == (10, 8, 128) and out.dtype == torch.float16


@pytest.mark.parametrize("name,args", [("append_rope", _rope_args), ("attend_paged", _attend_args)])
def test_backward_raises(name, args):
    a = args("meta", q=_t((10, 8, 128), device="meta").requires_grad_())
    out = getattr(ops, name)(*a)
    out = out[0] if isinstance(out, tuple) else out
    with pytest.raises(RuntimeError, match=name):
        out.sum().backward()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name,args", [("append_rope", _rope_args), ("attend_paged", _attend_args)])
def test_fake_gpu_tensors(name, args, grad):
    """What torch.compile runs: fake tensors of a GPU, through the keys that the calls without Python have."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        a = args("cuda")
        a[0].requires_grad_(grad)
        out = getattr(ops, name)(*a)
        out = out[0] if isinstance(out, tuple) else out
        assert tuple(out.shape) == (10, 8, 128) and out.device.type == "cuda" and out.requires_grad == grad
        a[0] = _t((10, 8, 96), device="cuda")
        with pytest.raises(RuntimeError, match="D must be"):
            getattr(ops, name)(*a)


def test_trees_are_as_large_as_they_were():
    """The limit of this format's batches is none of the other cache formats'."""
    shape = va._PagedShape(1 << 8, 32, 32, 128, 32, 64, 1 << 15, 256, 1 << 21)
    assert va.lib.va_tree_ws_bytes(int(va.Fmt.parse("q8+")), C.byref(shape), 4) > 0

"""The prompt, tree and page entry points without a GPU: invalid arguments are rejected with
the documented status codes before any device access (the pointers below are never read),
sizes, and the torch ops' checks, real and fake (meta) kernels alike."""
import ctypes as C

import pytest
import torch

import voltattn_amd as va
import voltattn_amd.torch_ops  # noqa: F401

VA_OK, VA_EINVAL, VA_EALIGN, VA_ENULL, VA_ERANGE = 0, 1, 2, 3, 4
ops = torch.ops.voltattn


def _message():
    return va.lib.va_last_error().decode()


# ---------------------------------------------------------------- prefill --
def _prefill(bufs=None, **kw):
    s = dict(B=2, total=100, Hq=8, Hkv=2, D=128, q_row=1024, q_head=128, k_row=256, k_head=128, v_row=256, v_head=128)
    s.update(kw)
    b = dict(q=0x1000, k=0x2000, v=0x3000, cu=0x4000, out=0x5000)
    b.update(bufs or {})
    cb, cs = va._PrefillBufs(*(b[n] for n in ("q", "k", "v", "cu", "out"))), va._PrefillShape(*s.values())
    return va.lib.va_prefill(C.byref(cb), C.byref(cs), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(B=0), VA_EINVAL, "B and Hkv"), (dict(Hkv=0), VA_EINVAL, "B and Hkv"), (dict(total=-1), VA_EINVAL, "total"),
    (dict(D=96), VA_EINVAL, "D must be"), (dict(Hq=7), VA_EINVAL, "multiple of Hkv"), (dict(Hq=0), VA_EINVAL, "multiple of Hkv"),
    (dict(q_row=1028), VA_EINVAL, "multiples of 8"), (dict(v_head=-8), VA_EINVAL, "multiples of 8"),
    (dict(k_row=120), VA_EINVAL, "k_row and v_row"), (dict(v_row=1 << 24), VA_EINVAL, "k_row and v_row"),
    (dict(total=2 ** 31 - 1, Hq=1 << 10), VA_ERANGE, "too large"),
    (dict(total=0), VA_OK, ""),                             # nothing to compute: no launch
])
def test_prefill_shape(kw, code, msg):
    assert _prefill(**kw) == code
    assert code == VA_OK or msg in _message()


@pytest.mark.parametrize("field,ptr,code", [("q", 0, VA_ENULL), ("k", 0, VA_ENULL), ("v", 0, VA_ENULL), ("cu", 0, VA_ENULL), ("out", 0, VA_ENULL),
                                            ("q", 0x1008, VA_EALIGN), ("k", 0x2002, VA_EALIGN), ("v", 0x3004, VA_EALIGN),
                                            ("cu", 0x4002, VA_EALIGN), ("out", 0x5008, VA_EALIGN)])
def test_prefill_buffers(field, ptr, code):
    assert _prefill({field: ptr}) == code


def test_prefill_null_structs():
    s, b = va._PrefillShape(), va._PrefillBufs()
    assert va.lib.va_prefill(None, C.byref(s), None) == VA_ENULL
    assert va.lib.va_prefill(C.byref(b), None, None) == VA_ENULL


# ------------------------------------------------------------------- tree --
def _shape(**kw):
    s = dict(B=4, Hq=32, Hkv=8, D=128, G=32, page_rows=64, max_pages=64, num_pages=256, max_seq_len=4096)
    s.update(kw)
    return va._PagedShape(*s.values())


def _tree(fmt="q8+", T=16, bufs=None, **kw):
    b = dict(k=0x10000, v=0x20000, sk=0x30000, sv=0x40000, block_table=0x50000, ctx_lens=0x60000, tree_sizes=0x70000,
             tree_mask=0x80000, q=0x90000, out=0xA0000, ws=0xB0000)
    b.update(bufs or {})
    s = _shape(**kw)
    return va.lib.va_decode_tree(int(va.Fmt.parse(fmt)), C.byref(va._TreeBufs(*b.values())), C.byref(s), T, None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(fmt="q8"), VA_EINVAL, "tiled format"), (dict(T=0), VA_EINVAL, "T must be"), (dict(T=65), VA_EINVAL, "T must be"),
    (dict(page_rows=32), VA_EINVAL, "power of two"), (dict(Hq=30), VA_EINVAL, "multiple of Hkv"), (dict(D=80), VA_EINVAL, "D must be"),
    (dict(G=48), VA_EINVAL, "G must be"), (dict(max_seq_len=4097), VA_EINVAL, "max_seq_len"), (dict(B=0), VA_EINVAL, "B and Hkv"),
    (dict(B=1 << 20, Hq=1 << 12), VA_ERANGE, "too large"),
    (dict(B=1 << 12, Hkv=1 << 5, Hq=1 << 5, max_pages=1 << 20, max_seq_len=1 << 26), VA_ERANGE, "too large"),
])
def test_tree_shape(kw, code, msg):
    assert _tree(**kw) == code
    assert msg in _message()
    s = _shape(**{k: v for k, v in kw.items() if k not in ("fmt", "T")})
    assert va.lib.va_tree_ws_bytes(int(va.Fmt.parse(kw.get("fmt", "q8+"))), C.byref(s), kw.get("T", 16)) == 0


@pytest.mark.parametrize("field,ptr,code", [(n, 0, VA_ENULL) for n in ("k", "v", "sk", "sv", "block_table", "ctx_lens", "tree_mask", "q", "out", "ws")] + [
    ("k", 0x10008, VA_EALIGN), ("sk", 0x30002, VA_EALIGN), ("block_table", 0x50001, VA_EALIGN), ("ctx_lens", 0x60002, VA_EALIGN),
    ("tree_sizes", 0x70002, VA_EALIGN), ("tree_mask", 0x80004, VA_EALIGN), ("q", 0x90008, VA_EALIGN), ("out", 0xA0004, VA_EALIGN), ("ws", 0xB0008, VA_EALIGN)])
def test_tree_buffers(field, ptr, code):
    assert _tree(bufs={field: ptr}) == code


def test_tree_null_structs():
    s, b = _shape(), va._TreeBufs()
    assert va.lib.va_decode_tree(int(va.Fmt.Q8M), None, C.byref(s), 4, None) == VA_ENULL
    assert va.lib.va_decode_tree(int(va.Fmt.Q8M), C.byref(b), None, 4, None) == VA_ENULL


def test_tree_workspace_does_not_grow_with_the_batch():
    """Two pieces per work-group, whatever the batch: 128 query rows of (D + 2) floats each at most."""
    def ws(**kw):
        s = _shape(**kw)
        return va.lib.va_tree_ws_bytes(int(va.Fmt.Q8M), C.byref(s), 64)

    assert 0 < ws(B=1) <= ws(B=64) == ws(B=512) <= 2 * 4 * 256 * 128 * 130 * 4


# ------------------------------------------------------------------ pages --
def _pools(**kw):
    p = dict(k=0x10000, v=0x20000, sk=0x30000, sv=0x40000)
    p.update(kw)
    return va._Pools(*p.values())


def _compact(fmt="q8+", pools=None, n=8, ptrs=None, **kw):
    a = dict(table=0x50000, base=0x60000, keep=0x70000, counts=0x80000)
    a.update(ptrs or {})
    s, p = _shape(**kw), _pools(**(pools or {}))
    return va.lib.va_compact_kv(int(va.Fmt.parse(fmt)), C.byref(p), C.byref(s), *(x or None for x in a.values()), n, None)


def _fork(fmt="q8+", pools=None, children=4, ptrs=None, **kw):
    a = dict(table=0x50000, lens=0x60000, parents=0x70000, refs=0x80000, new_table=0x90000, new_lens=0xA0000, missing=0xB0000)
    a.update(ptrs or {})
    s, p = _shape(**kw), _pools(**(pools or {}))
    t = [x or None for x in a.values()]
    return va.lib.va_fork_pages(int(va.Fmt.parse(fmt)), C.byref(p), C.byref(s), *t[:3], children, *t[3:], None)


def _resize(ptrs=None, **kw):
    s = dict(B=4, page_rows=64, max_pages=64, num_pages=256)
    s.update(kw)
    a = dict(table=0x50000, refs=0x60000, old=0x70000, new=0x80000, missing=0x90000)
    a.update(ptrs or {})
    return va.lib.va_resize_pages(*s.values(), *(x or None for x in a.values()), None)


@pytest.mark.parametrize("call,kw,code,msg", [
    (_compact, dict(n=-1), VA_EINVAL, "n must be"), (_compact, dict(n=65), VA_EINVAL, "n must be"), (_compact, dict(n=0), VA_OK, ""),
    (_compact, dict(D=80), VA_EINVAL, "D must be"), (_compact, dict(B=0), VA_EINVAL, "B and Hkv"),
    (_compact, dict(max_pages=1 << 20, page_rows=1 << 12), VA_ERANGE, "2^31"), (_compact, dict(num_pages=(1 << 30) + 1, page_rows=1, max_pages=1, Hkv=1), VA_ERANGE, "2^30"),
    (_fork, dict(children=0), VA_EINVAL, "children"), (_fork, dict(G=16), VA_EINVAL, "G must be"), (_fork, dict(children=1 << 29), VA_ERANGE, "too many"),
    (_fork, dict(ptrs=dict(new_table=0x50000)), VA_EINVAL, "must not be"), (_fork, dict(ptrs=dict(new_lens=0x60000)), VA_EINVAL, "must not be"),
    (_resize, dict(B=0), VA_EINVAL, ">= 1"), (_resize, dict(page_rows=0), VA_EINVAL, ">= 1"), (_resize, dict(max_pages=0), VA_EINVAL, ">= 1"),
    (_resize, dict(num_pages=0), VA_EINVAL, ">= 1"), (_resize, dict(max_pages=1 << 26), VA_ERANGE, "2^31"), (_resize, dict(num_pages=(1 << 30) + 1), VA_ERANGE, "2^30"),
])
def test_page_shapes(call, kw, code, msg):
    assert call(**kw) == code
    assert code == VA_OK or msg in _message()


@pytest.mark.parametrize("call,names", [(_compact, ("table", "base", "keep", "counts")),
                                        (_fork, ("table", "lens", "parents", "refs", "new_table", "new_lens", "missing")),
                                        (_resize, ("table", "refs", "old", "new", "missing"))])
def test_page_buffers(call, names):
    for n in names:
        assert call(ptrs={n: 0x100002}) == VA_EALIGN, n
        if n != "missing":
            assert call(ptrs={n: 0}) == VA_ENULL, n


@pytest.mark.parametrize("call", [_compact, _fork])
def test_page_pools(call):
    for n in ("k", "v", "sk", "sv"):
        assert call(pools={n: 0}) == VA_ENULL, n
    assert call(pools=dict(k=0x10002)) == VA_EALIGN
    assert call(pools=dict(sv=0x40001)) == VA_EALIGN
    assert call(fmt="f16+", pools=dict(v=0x20008, sk=0, sv=0)) == VA_EALIGN   # f16 rows are 16-byte words


# -------------------------------------------------------------- torch ops --
def _t(shape, dtype=torch.float16, device="cpu"):
    return torch.zeros(shape, dtype=dtype, device=device)


def _prefill_args(device, **kw):
    a = dict(q=_t((10, 8, 128), device=device), k=_t((10, 2, 128), device=device), v=_t((10, 2, 128), device=device),
             cu=_t((3,), torch.int32, device))
    a.update(kw)
    return list(a.values())


def _tree_args(device, fmt="q8+", **kw):
    a = dict(q=_t((2, 5, 8, 128), device=device), k=_t((9, 2, 64, 128), torch.uint8, device), v=_t((9, 2, 64, 128), torch.uint8, device),
             ks=_t((9, 2, 64, 4), device=device), vs=_t((9, 2, 64, 4), device=device), table=_t((2, 4), torch.int32, device),
             ctx=_t((2,), torch.int32, device), sizes=None, mask=_t((2, 5), torch.int64, device))
    a.update(kw)
    return list(a.values()) + [fmt, 256, 32]


def _compact_args(device, **kw):
    a = dict(k=_t((9, 2, 64, 128), torch.uint8, device), v=_t((9, 2, 64, 128), torch.uint8, device),
             ks=_t((9, 2, 64, 4), device=device), vs=_t((9, 2, 64, 4), device=device), table=_t((2, 4), torch.int32, device),
             base=_t((2,), torch.int32, device), keep=_t((2, 5), torch.int32, device), counts=_t((2,), torch.int32, device))
    a.update(kw)
    return list(a.values()) + ["q8+", 32]


def _fork_args(device, **kw):
    a = dict(table=_t((2, 4), torch.int32, device), lens=_t((2,), torch.int32, device), parents=_t((5,), torch.int32, device),
             refs=_t((9,), torch.int32, device), k=_t((9, 2, 64, 128), torch.uint8, device), v=_t((9, 2, 64, 128), torch.uint8, device),
             ks=_t((9, 2, 64, 4), device=device), vs=_t((9, 2, 64, 4), device=device))
    a.update(kw)
    return list(a.values()) + ["q8+", 32]


def _resize_args(device, **kw):
    a = dict(table=_t((2, 4), torch.int32, device), refs=_t((9,), torch.int32, device), old=_t((2,), torch.int32, device),
             new=_t((2,), torch.int32, device), page_rows=64)
    a.update(kw)
    return list(a.values())


BAD = [
    ("prefill", _prefill_args, dict(q=((10, 8, 128), torch.float32)), "q has dtype"),
    ("prefill", _prefill_args, dict(q=((10, 128), torch.float16)), "q must be"),
    ("prefill", _prefill_args, dict(k=((10, 3, 128), torch.float16)), "multiple of K/V heads"),
    ("prefill", _prefill_args, dict(v=((11, 2, 128), torch.float16)), "v has shape"),
    ("prefill", _prefill_args, dict(cu=((1,), torch.int32)), "cu_seqlens"),
    ("prefill", _prefill_args, dict(cu=((3,), torch.int64)), "cu_seqlens has dtype"),
    ("decode_tree", _tree_args, dict(q=((2, 65, 8, 128), torch.float16), mask=((2, 65), torch.int64)), "T must be"),
    ("decode_tree", _tree_args, dict(q=((2, 0, 8, 128), torch.float16), mask=((2, 0), torch.int64)), "T must be"),
    ("decode_tree", _tree_args, dict(mask=((2, 4), torch.int64)), "tree_mask"),
    ("decode_tree", _tree_args, dict(mask=((2, 5), torch.int32)), "tree_mask has dtype"),
    ("decode_tree", _tree_args, dict(sizes=((3,), torch.int32)), "tree_sizes"),
    ("decode_tree", _tree_args, dict(ks=((9, 2, 64, 2), torch.float16)), "k_scale"),
    ("compact_kv", _compact_args, dict(keep=((2, 65), torch.int32)), "keep"),
    ("compact_kv", _compact_args, dict(keep=((10,), torch.int32)), "keep"),
    ("compact_kv", _compact_args, dict(counts=((3,), torch.int32)), "counts"),
    ("compact_kv", _compact_args, dict(vs=None), "v_scale is required"),
    ("fork_pages", _fork_args, dict(refs=((8,), torch.int32)), "refs"),
    ("fork_pages", _fork_args, dict(parents=((5, 1), torch.int32)), "parents"),
    ("fork_pages", _fork_args, dict(lens=((3,), torch.int32)), "seq_lens"),
    ("resize_pages", _resize_args, dict(old=((3,), torch.int32)), "old_lens"),
    ("resize_pages", _resize_args, dict(refs=((9,), torch.int64)), "refs has dtype"),
    ("resize_pages", _resize_args, dict(page_rows=0), "page_rows"),
]


@pytest.mark.parametrize("device", ["cpu", "meta"])
@pytest.mark.parametrize("name,args,kw,msg", BAD)
def test_torch_checks(device, name, args, kw, msg):
    kw = {k: _t(*v, device=device) if isinstance(v, tuple) else v for k, v in kw.items()}
    with pytest.raises(RuntimeError, match=msg):
        getattr(ops, name)(*args(device, **kw))


@pytest.mark.parametrize("name,args", [("prefill", _prefill_args), ("decode_tree", _tree_args), ("compact_kv", _compact_args),
                                       ("fork_pages", _fork_args), ("resize_pages", _resize_args)])
def test_no_cpu_fallback_and_fake_shapes(name, args):
    with pytest.raises(RuntimeError, match="gfx950"):
        getattr(ops, name)(*args("cpu"))
    out = getattr(ops, name)(*args("meta"))
    want = {"prefill": [((10, 8, 128), torch.float16)], "decode_tree": [((2, 5, 8, 128), torch.float16)], "compact_kv": [],
            "fork_pages": [((5, 4), torch.int32), ((5,), torch.int32), ((1,), torch.int32)], "resize_pages": [((1,), torch.int32)]}[name]
    got = [] if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    assert [(tuple(t.shape), t.dtype) for t in got] == want

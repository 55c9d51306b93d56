"""PyTorch-ROCm binding: ``torch.ops.voltattn.*`` custom ops over the C ABI.

Importing this module registers

* ``voltattn::decode(q, k, v, k_scale, v_scale, fmt, group, splits) -> out``
  — one decode step (va_decode; the reference's launch(), src/voltattn.cu:803-835);
* ``voltattn::decode_gqa(...)`` — Hq query heads over Hkv KV heads (va_decode_gqa);
* ``voltattn::decode_paged(...)`` — a batch over a page pool (va_decode_paged);
* ``voltattn::append_kv(...)`` — quantize-and-append new rows (va_append_kv; mutates the pools);
* ``voltattn::prefill(q, k, v, cu_seqlens) -> out`` — causal attention of packed prompts
  (va_prefill);
* ``voltattn::decode_tree(...)`` — drafted tokens over a page pool (va_decode_tree);
* ``voltattn::compact_kv(...)`` — accepted drafts' rows moved together (va_compact_kv; mutates
  the pools);
* ``voltattn::fork_pages(...) -> (block_table, seq_lens, missing)`` — the next step's sequences
  (va_fork_pages; mutates refs and the pools);
* ``voltattn::resize_pages(...) -> missing`` — pages given up and handed out (va_resize_pages;
  mutates block_table and refs);
* ``voltattn::append_rope(...) -> (q, k)`` — a projection's rows rotated by their positions, k and v
  written into a paged cache (va_append_rope; mutates the pools);
* ``voltattn::attend_paged(...) -> out`` — the newest tokens of every sequence over a cache in 8 bits
  with a scale for each block of positions and head (va_attend_paged);
* ``voltattn::quantize(x, bits, group) -> (packed, scales)`` (va_quantize; the reference's
  quantize(), src/voltattn.cu:705-745);
* ``voltattn::dequantize(packed, scales, bits, group) -> x`` (va_dequantize; the reference's
  dq(), src/voltattn.cu:747-767, over whole rows: fp32 [..., D]).

Tensors keep the C ABI's layouts (include/voltattn.h): q/out fp16 [.., H, D];
quantized K/V payload uint8 [.., L, row bytes]; f16 K/V fp16 [.., L, D]; scales
fp16 [.., L, D/G]. Every op runs asynchronously on torch's current HIP stream
and fails loudly on invalid input: the shapes and dtypes of every tensor are
checked against (fmt, D, G) before the C ABI is called, in the real and the
fake (meta) implementation alike (RuntimeError), and the library's own checks
raise with its message. There is no CPU fallback: the tensors must live on a
gfx950 device. Each op has a fake implementation, so shapes propagate under
torch.compile.
"""
from __future__ import annotations

import ctypes as C
import re
import warnings
from pathlib import Path
from typing import Optional

import torch
from torch.autograd import forward_ad as _forward

from . import (B8, TREE_MAX, Fmt, _AttendBufs, _Bufs, _PagedBufs, _PagedShape, _Pools, _PrefillBufs, _PrefillShape,
               _RopeBufs, _RopeShape, _TreeBufs, check, fmt_bits, lib, ws_bytes)

__all__ = ["decode", "decode_gqa", "decode_paged", "append_kv", "quantize", "dequantize",
           "prefill", "decode_tree", "compact_kv", "fork_pages", "resize_pages", "append_rope", "attend_paged"]


# What an op does on the host per call is most of a small call's time: the names are
# looked up once, plain sizes are compared without torch._check, and the stream handle
# is read directly (decode_paged 45 -> 25 us per call, append_kv 35 -> 20).
_FMTS = {f.label: f for f in Fmt}
_BITS = [fmt_bits(f) for f in Fmt]


def _fmt(name: str) -> Fmt:
    f = _FMTS.get(name)
    return Fmt.parse(name) if f is None else f


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor):
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _need_gpu(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("voltattn ops need tensors on a gfx950 device (no CPU fallback)")
        if t is not None and not t.is_contiguous():
            raise RuntimeError("voltattn ops need contiguous tensors")


def _D_of(q: torch.Tensor) -> int:
    return int(q.shape[-1])


def _fail(msg: str):
    raise RuntimeError(f"voltattn: {msg}")


# The validators run in the real and the fake (meta) implementations alike.
# Sizes may be symbolic (torch.compile with dynamic shapes): they are compared
# with torch._check, which records a runtime assertion instead of fixing a
# size to its traced value, and are never converted with int() here, so a
# decode loop whose L grows does not recompile on every step. Only the head
# dimension D (64 or 128) and the group size decide which kernel runs.

def _check(cond, msg) -> None:           # callers may skip it where cond is True: nothing to record
    if cond is True:
        return
    torch._check(cond, lambda: f"voltattn: {msg()}")


def _expect(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype) -> None:
    if type(t) is torch.Tensor and t.shape == shape and t.dtype == dtype:
        return                               # plain sizes only: a traced tensor has another type
    if t is None:
        _fail(f"{name} is required")
    if t.dim() != len(shape):
        _fail(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    for got, want in zip(t.shape, shape):
        _check(got == want, lambda: f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        _fail(f"{name} has dtype {t.dtype}, expected {dtype}")


def _check_dg(f: Fmt, D, group: int) -> None:
    if (ok := (D == 64) | (D == 128)) is not True:
        _check(ok, lambda: f"D must be 64 or 128 (got {D})")
    if _BITS[f] != 16:
        if group not in (32, 64):
            _fail(f"group must be 32 or 64 (got {group})")
        if (ok := D >= group) is not True:
            _check(ok, lambda: f"group must be <= D (got {group}, D={D})")


def _row_shape(f: Fmt, D) -> tuple[tuple, torch.dtype]:
    """Trailing shape and dtype of one K/V row of format f: fp16 [D] for the f16
    formats, uint8 [row bytes] for the quantized ones."""
    if _BITS[f] == 16:
        return (D,), torch.float16
    return (D * _BITS[f] // 8,), torch.uint8


def _check_kv(f: Fmt, k, v, ks, vs, lead: tuple, D, group: int) -> None:
    """k, v [*lead, row]; scales fp16 [*lead, D/G] for quantized formats."""
    tail, dt = _row_shape(f, D)
    _expect(k, "k", lead + tail, dt)
    _expect(v, "v", lead + tail, dt)
    if _BITS[f] != 16:
        _expect(ks, "k_scale", lead + (D // group,), torch.float16)
        _expect(vs, "v_scale", lead + (D // group,), torch.float16)


def _validate_decode(q, k, v, ks, vs, f: Fmt, group: int, grouped: bool) -> None:
    if q.dim() != 2:
        _fail(f"q must be [H, D] (got {tuple(q.shape)})")
    H, D = q.shape
    _expect(q, "q", (H, D), torch.float16)
    _check_dg(f, D, group)
    if k.dim() != 3:
        _fail(f"k must be [heads, L, row] (got {tuple(k.shape)})")
    Hk, L = k.shape[0], k.shape[1]
    if grouped:
        _check(Hk >= 1, lambda: f"k must have at least one head (got {Hk})")
        _check(H % Hk == 0, lambda: f"query heads ({H}) must be a multiple of K/V heads ({Hk})")
    else:
        _check(Hk == H, lambda: f"k has {Hk} heads, q has {H}")
    _check_kv(f, k, v, ks, vs, (Hk, L), D, group)


def _validate_paged(q, kp, vp, ksp, vsp, block_table, seq_lens, f: Fmt, group: int) -> None:
    if q.dim() != 3:
        _fail(f"q must be [B, Hq, D] (got {tuple(q.shape)})")
    B, Hq, D = q.shape
    _expect(q, "q", (B, Hq, D), torch.float16)
    _check_dg(f, D, group)
    if kp.dim() != 4:
        _fail(f"k_pages must be [num_pages, Hkv, page_rows, row] (got {tuple(kp.shape)})")
    num_pages, Hkv, page_rows = kp.shape[:3]
    _check(Hkv >= 1, lambda: f"k_pages must have at least one head (got {Hkv})")
    _check(Hq % Hkv == 0, lambda: f"query heads ({Hq}) must be a multiple of K/V heads ({Hkv})")
    _check_kv(f, kp, vp, ksp, vsp, (num_pages, Hkv, page_rows), D, group)
    if block_table.dim() != 2:
        _fail(f"block_table must be [B={B}, max_pages] (got {tuple(block_table.shape)})")
    _check(block_table.shape[0] == B, lambda: f"block_table must be [B={B}, max_pages] (got {tuple(block_table.shape)})")
    _expect(block_table, "block_table", (B, block_table.shape[1]), torch.int32)
    _expect(seq_lens, "seq_lens", (B,), torch.int32)


def _validate_append(x, start, block_table, pages, scale_pages, f: Fmt, group: int) -> None:
    if x.dim() != 4:
        _fail(f"x must be [B, Hkv, n, D] (got {tuple(x.shape)})")
    B, Hkv, n, D = x.shape
    _expect(x, "x", (B, Hkv, n, D), torch.float16)
    _check_dg(f, D, group)
    if pages.dim() != 4:
        _fail(f"pages must be [num_pages, Hkv, page_rows, row] (got {tuple(pages.shape)})")
    num_pages, Hp, page_rows = pages.shape[:3]
    _check(Hp == Hkv, lambda: f"pages hold {Hp} K/V heads, x has {Hkv}")
    tail, dt = _row_shape(f, D)
    _expect(pages, "pages", (num_pages, Hkv, page_rows) + tail, dt)
    if _BITS[f] != 16:
        _expect(scale_pages, "scale_pages", (num_pages, Hkv, page_rows, D // group), torch.float16)
    _expect(start, "start", (B,), torch.int32)
    if block_table.dim() != 2:
        _fail(f"block_table must be [B={B}, max_pages] (got {tuple(block_table.shape)})")
    _check(block_table.shape[0] == B, lambda: f"block_table must be [B={B}, max_pages] (got {tuple(block_table.shape)})")
    _expect(block_table, "block_table", (B, block_table.shape[1]), torch.int32)


def _validate_quantize(x, bits: int, group: int) -> None:
    if bits not in (8, 4, 3):
        _fail(f"bits must be 8, 4 or 3 (got {bits})")
    if x.dtype != torch.float32:
        _fail(f"x must be fp32 (got {x.dtype})")
    if group not in (32, 64):
        _fail(f"group must be 32 or 64 (got {group})")
    if x.dim() == 0:
        _fail("x must have a last dimension D")
    D = x.shape[-1]
    _check((D >= group) & (D % group == 0) & (D % 8 == 0),
           lambda: f"group must be 32 or 64 and divide D (got group={group}, D={D})")


def _validate_dequantize(packed, scales, bits: int, group: int):
    """Checks packed uint8 [..., D*bits/8] and scales fp16 [..., D/G]; returns D."""
    if bits not in (8, 4, 3):
        _fail(f"bits must be 8, 4 or 3 (got {bits})")
    if packed.dtype != torch.uint8:
        _fail(f"packed must be uint8 (got {packed.dtype})")
    if group not in (32, 64):
        _fail(f"group must be 32 or 64 (got {group})")
    if packed.dim() == 0:
        _fail("packed must have a last dimension (row bytes)")
    nb = packed.shape[-1]
    _check(nb * 8 % bits == 0, lambda: f"packed rows of {nb} bytes do not hold whole {bits}-bit codes")
    D = nb * 8 // bits
    _check((D >= group) & (D % group == 0) & (D % 8 == 0),
           lambda: f"group must be 32 or 64 and divide D (got group={group}, D={D})")
    _expect(scales, "scales", tuple(packed.shape[:-1]) + (D // group,), torch.float16)
    return D


@torch.library.custom_op("voltattn::decode", mutates_args=())
def decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor],
           v_scale: Optional[torch.Tensor], fmt: str, group: int = 32, splits: int = 0) -> torch.Tensor:
    """q fp16 [H, D]; k, v [H, L, row] (uint8) or [H, L, D] (fp16 formats); scales fp16 [H, L, D/G]."""
    f = _fmt(fmt)
    _validate_decode(q, k, v, k_scale, v_scale, f, group, grouped=False)
    _need_gpu(q, k, v, k_scale, v_scale)
    H, D, L = int(q.shape[0]), _D_of(q), int(k.shape[1])
    S = splits
    if S <= 0:
        s = C.c_int(0)
        check(lib.va_pick_splits(int(f), H, L, D, C.byref(s)))
        S = s.value
    out = torch.empty((H, D), dtype=torch.float16, device=q.device)
    ws = torch.empty(ws_bytes(H, D, S) // 4, dtype=torch.float32, device=q.device)
    b = _Bufs(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), _ptr(q), _ptr(out), _ptr(ws))
    check(lib.va_decode(int(f), C.byref(b), H, L, D, group, S, _stream(q)))
    return out


@decode.register_fake
def _(q, k, v, k_scale, v_scale, fmt, group=32, splits=0):
    _validate_decode(q, k, v, k_scale, v_scale, _fmt(fmt), group, grouped=False)
    return q.new_empty((q.shape[0], q.shape[-1]), dtype=torch.float16)


@torch.library.custom_op("voltattn::decode_gqa", mutates_args=())
def decode_gqa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor],
               v_scale: Optional[torch.Tensor], fmt: str, group: int = 32, splits: int = 0) -> torch.Tensor:
    """q fp16 [Hq, D]; k, v [Hkv, L, ...]; query head h attends KV head h // (Hq / Hkv)."""
    f = _fmt(fmt)
    _validate_decode(q, k, v, k_scale, v_scale, f, group, grouped=True)
    _need_gpu(q, k, v, k_scale, v_scale)
    Hq, Hkv, D, L = int(q.shape[0]), int(k.shape[0]), _D_of(q), int(k.shape[1])
    S = splits
    if S <= 0:
        s = C.c_int(0)
        check(lib.va_pick_splits_gqa(int(f), Hq, Hkv, L, D, C.byref(s)))
        S = s.value
    out = torch.empty((Hq, D), dtype=torch.float16, device=q.device)
    ws = torch.empty(ws_bytes(Hq, D, S) // 4, dtype=torch.float32, device=q.device)
    b = _Bufs(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), _ptr(q), _ptr(out), _ptr(ws))
    check(lib.va_decode_gqa(int(f), C.byref(b), Hq, Hkv, L, D, group, S, _stream(q)))
    return out


@decode_gqa.register_fake
def _(q, k, v, k_scale, v_scale, fmt, group=32, splits=0):
    _validate_decode(q, k, v, k_scale, v_scale, _fmt(fmt), group, grouped=True)
    return q.new_empty((q.shape[0], q.shape[-1]), dtype=torch.float16)


def _paged_shape(q, k_pages, block_table, group, max_seq_len):
    B, Hq, D = (int(x) for x in q.shape)
    num_pages, Hkv, page_rows = (int(x) for x in k_pages.shape[:3])
    return _PagedShape(B, Hq, Hkv, D, group, page_rows, int(block_table.shape[1]), num_pages,
                       max_seq_len)


@torch.library.custom_op("voltattn::decode_paged", mutates_args=())
def decode_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 k_scale_pages: Optional[torch.Tensor], v_scale_pages: Optional[torch.Tensor],
                 block_table: torch.Tensor, seq_lens: torch.Tensor, fmt: str, max_seq_len: int,
                 group: int = 32, splits: int = 0) -> torch.Tensor:
    """q fp16 [B, Hq, D]; pages [num_pages, Hkv, page_rows, ...]; block_table int32
    [B, max_pages]; seq_lens int32 [B] (each <= max_seq_len)."""
    f = _fmt(fmt)
    _validate_paged(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, seq_lens, f, group)
    _need_gpu(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, seq_lens)
    shape = _paged_shape(q, k_pages, block_table, group, max_seq_len)
    S = splits
    if S <= 0:
        s = C.c_int(0)
        check(lib.va_pick_splits_paged(int(f), C.byref(shape), C.byref(s)))
        S = s.value
    B, Hq, D = (int(x) for x in q.shape)
    out = torch.empty((B, Hq, D), dtype=torch.float16, device=q.device)
    ws = torch.empty(ws_bytes(B * Hq, D, S) // 4, dtype=torch.float32, device=q.device)
    b = _PagedBufs(_ptr(k_pages), _ptr(v_pages), _ptr(k_scale_pages), _ptr(v_scale_pages),
                   _ptr(block_table), _ptr(seq_lens), _ptr(q), _ptr(out), _ptr(ws))
    check(lib.va_decode_paged(int(f), C.byref(b), C.byref(shape), S, _stream(q)))
    return out


@decode_paged.register_fake
def _(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, seq_lens, fmt, max_seq_len,
      group=32, splits=0):
    _validate_paged(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, seq_lens, _fmt(fmt), group)
    return q.new_empty(q.shape, dtype=torch.float16)


@torch.library.custom_op("voltattn::append_kv", mutates_args=("pages", "scale_pages"))
def append_kv(x: torch.Tensor, start: torch.Tensor, block_table: torch.Tensor, pages: torch.Tensor,
              scale_pages: Optional[torch.Tensor], fmt: str, group: int = 32) -> None:
    """x fp16 [B, Hkv, n, D] new rows written at positions start[b] + r of the paged cache
    pages [num_pages, Hkv, page_rows, ...] (+ scale_pages for quantized formats)."""
    f = _fmt(fmt)
    _validate_append(x, start, block_table, pages, scale_pages, f, group)
    _need_gpu(x, start, block_table, pages, scale_pages)
    B, Hkv, n, D = (int(s) for s in x.shape)
    num_pages, _, page_rows = (int(s) for s in pages.shape[:3])
    shape = _PagedShape(B, Hkv, Hkv, D, group, page_rows, int(block_table.shape[1]), num_pages, 0)
    check(lib.va_append_kv(int(f), _ptr(x), n, _ptr(start), _ptr(block_table), C.byref(shape),
                           _ptr(pages), _ptr(scale_pages), _stream(x)))


@append_kv.register_fake
def _(x, start, block_table, pages, scale_pages, fmt, group=32):
    _validate_append(x, start, block_table, pages, scale_pages, _fmt(fmt), group)
    return None


@torch.library.custom_op("voltattn::quantize", mutates_args=())
def quantize(x: torch.Tensor, bits: int, group: int = 32) -> tuple[torch.Tensor, torch.Tensor]:
    """x fp32 [..., D] -> (packed uint8 [..., D*bits/8], fp16 scales [..., D/G])."""
    _validate_quantize(x, bits, group)
    _need_gpu(x)
    D = int(x.shape[-1])
    rows = x.numel() // D
    packed = torch.empty(x.shape[:-1] + (D * bits // 8,), dtype=torch.uint8, device=x.device)
    scales = torch.empty(x.shape[:-1] + (D // group,), dtype=torch.float16, device=x.device)
    check(lib.va_quantize(bits, group, _ptr(x), rows, D, _ptr(packed), _ptr(scales), _stream(x)))
    return packed, scales


@quantize.register_fake
def _(x, bits, group=32):
    _validate_quantize(x, bits, group)
    D = x.shape[-1]
    return (x.new_empty(x.shape[:-1] + (D * bits // 8,), dtype=torch.uint8),
            x.new_empty(x.shape[:-1] + (D // group,), dtype=torch.float16))


@torch.library.custom_op("voltattn::dequantize", mutates_args=())
def dequantize(packed: torch.Tensor, scales: torch.Tensor, bits: int, group: int = 32) -> torch.Tensor:
    """(packed uint8 [..., D*bits/8], fp16 scales [..., D/G]) -> fp32 [..., D], bit-exact dq()."""
    D = int(_validate_dequantize(packed, scales, bits, group))
    _need_gpu(packed, scales)
    rows = packed.numel() // max(1, int(packed.shape[-1]))
    out = torch.empty(packed.shape[:-1] + (D,), dtype=torch.float32, device=packed.device)
    check(lib.va_dequantize(bits, group, _ptr(packed), _ptr(scales), rows, D, _ptr(out), _stream(packed)))
    return out


@dequantize.register_fake
def _(packed, scales, bits, group=32):
    D = _validate_dequantize(packed, scales, bits, group)
    return packed.new_empty(packed.shape[:-1] + (D,), dtype=torch.float32)


# ------------------------------------- prompts, drafted tokens, page pool --

# Registered through the dispatcher directly: per call torch.library.custom_op takes 15 us on
# the host, more than most of these kernels run for, this 4. One implementation for every
# device, so that CPU tensors meet the ops' own error.
_LIBRARY = torch.library.Library("voltattn", "FRAGMENT")


_KEY = torch._C.DispatchKey
_PLAIN = (torch._C.DispatchKeySet(_KEY.CUDA) | torch._C.DispatchKeySet(_KEY.AutogradCUDA)).raw_repr()


class _NoGradient(torch.autograd.Function):
    """An op's output for inputs that require grad: backward() raises, as that of custom_op's ops does."""

    @staticmethod
    def forward(ctx, name, call, *args):
        ctx.name = name
        return call(*args)

    @staticmethod
    def backward(ctx, *grads):
        _fail(f"backward through voltattn::{ctx.name}, which has no gradient formula")


def _no_tangents(name: str, args) -> None:
    """Forward mode: an output without a tangent would be a wrong one."""
    if torch._C._is_fwd_grad_enabled() and any(
            isinstance(a, torch.Tensor) and a.is_floating_point() and _forward.unpack_dual(a).tangent is not None for a in args):
        _fail(f"forward-mode gradient through voltattn::{name}, which has no gradient formula")


def _op(schema: str, fake, computes: Optional[bool] = None, native: bool = False):
    """Registers the decorated function and its fake implementation; what it returns is the op.
    computes: whether its outputs are computed from its inputs (None: if it changes none in place).
    native: its plain calls on a GPU are host/torch_calls.cpp's, which hands the others to <name>_checked."""
    name = schema.split("(")[0]
    if native:
        checked = _op(f"{name}_checked{schema[len(name):]}", fake, computes)

    def register(fn):
        if native:
            checked(fn)
        _LIBRARY.define(schema)
        _LIBRARY.impl(name, fn, "CompositeExplicitAutograd")
        torch.library.register_fake(f"voltattn::{name}", fake, lib=_LIBRARY)
        op = getattr(torch.ops.voltattn, name)
        op.__doc__ = fn.__doc__
        if "!" not in schema if computes is None else computes:

            def autograd(keys, *args):
                if _forward._current_level >= 0:                # in a dual_level()
                    _no_tangents(name, args)
                grads = torch._C.is_grad_enabled() and torch._C._any_requires_grad(*args)
                if not grads and keys.raw_repr() == _PLAIN:     # on a GPU: the dispatcher's second turn takes 3 us
                    return fn(*args)
                below = keys & torch._C._after_autograd_keyset
                if grads:
                    return _NoGradient.apply(name, lambda *a: op.default.redispatch(below, *a), *args)
                with torch._C._AutoDispatchBelowAutograd():
                    return op.default.redispatch(below, *args)

            _LIBRARY.impl(name, autograd, "Autograd", with_keyset=True)
        return op

    return register


def _on_device(t: torch.Tensor, *others) -> int:
    """The stream to launch on: every tensor is on t's device, which must be the current one."""
    at = t.get_device()                                     # -1: not on a GPU
    for x in others:
        if x is not None and x.get_device() != at:
            _fail(f"tensors on {t.device} and {x.device}")
    if at < 0 or not t.is_cuda:
        _fail("ops need tensors on a gfx950 device (no CPU fallback)")
    if at != torch._C._cuda_getDevice():
        _fail(f"tensors on {t.device}, but the current device is cuda:{torch._C._cuda_getDevice()} (torch.cuda.device)")
    return torch._C._cuda_getCurrentRawStream(at)


def _contiguous(*ts) -> None:
    for t in ts:
        if t is not None and not t.is_contiguous():
            _fail(f"a tensor of shape {tuple(t.shape)} must be contiguous")


# Notes that tensors have changed in place, so that backward() does not take them for what was saved;
# those made in inference mode keep no such count and are passed over.
_changed = torch._C._increment_version


def _ready(t: torch.Tensor, *others) -> int:
    """_on_device and _contiguous in one pass."""
    at = t.get_device()
    ok = t.is_contiguous()
    for x in others:
        if x is not None and (x.get_device() != at or not x.is_contiguous()):
            ok = False
    if not ok or at < 0 or not t.is_cuda or at != torch._C._cuda_getDevice():
        _on_device(t, *others)
        _contiguous(t, *others)
    return torch._C._cuda_getCurrentRawStream(at)


def _validate_prefill(q, k, v, cu) -> None:
    if q.dim() != 3:
        _fail(f"q must be [T, Hq, D] (got {tuple(q.shape)})")
    T, Hq, D = q.shape
    _expect(q, "q", (T, Hq, D), torch.float16)
    if (ok := (D == 64) | (D == 128)) is not True:
        _check(ok, lambda: f"D must be 64 or 128 (got {D})")
    if k.dim() != 3:
        _fail(f"k must be [T, Hkv, D] (got {tuple(k.shape)})")
    Hkv = k.shape[1]
    if (ok := Hkv >= 1) is not True:
        _check(ok, lambda: f"k must have at least one head (got {Hkv})")
    if (ok := Hq >= 1) is not True:
        _check(ok, lambda: f"q must have at least one head (got {Hq})")
    if (ok := Hq % Hkv == 0) is not True:
        _check(ok, lambda: f"query heads ({Hq}) must be a multiple of K/V heads ({Hkv})")
    _expect(k, "k", (T, Hkv, D), torch.float16)
    _expect(v, "v", (T, Hkv, D), torch.float16)
    if cu.dim() != 1:
        _fail(f"cu_seqlens must be [B + 1] (got {tuple(cu.shape)})")
    _expect(cu, "cu_seqlens", (cu.shape[0],), torch.int32)
    if (ok := cu.shape[0] >= 2) is not True:
        _check(ok, lambda: f"cu_seqlens must be [B + 1] with B >= 1 (got {tuple(cu.shape)})")


def _strides(name: str, t: torch.Tensor):
    """(row, head) strides; the last dimension must be dense. The stride of a dimension of one is never
    stepped: any that the library takes."""
    T, H, D = t.shape
    row, head, last = t.stride()
    if last != 1:
        _fail(f"{name} must be dense in its last dimension (stride {last})")
    if H == 1:
        head = 0
    if T <= 1:
        row = D
    return row, head


def _prefill_fake(q, k, v, cu_seqlens):
    _validate_prefill(q, k, v, cu_seqlens)
    return q.new_empty(q.shape, dtype=torch.float16)


@_op("prefill(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens) -> Tensor", _prefill_fake)
def prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor) -> torch.Tensor:
    """q fp16 [T, Hq, D]; k, v fp16 [T, Hkv, D], dense in D only (slices of a fused projection);
    cu_seqlens int32 [B + 1]: rows cu[b] .. cu[b+1] - 1 are prompt b. out [T, Hq, D], zeros in rows of no prompt."""
    _validate_prefill(q, k, v, cu_seqlens)
    stream = _on_device(q, k, v, cu_seqlens)
    _contiguous(cu_seqlens)
    T, Hq, D = q.shape
    out = torch.empty((T, Hq, D), dtype=torch.float16, device=q.device)
    if T == 0:
        return out
    shape = _PrefillShape(cu_seqlens.shape[0] - 1, T, Hq, k.shape[1], D, *_strides("q", q), *_strides("k", k),
                          *_strides("v", v))
    b = _PrefillBufs(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens.data_ptr(), out.data_ptr())
    check(lib.va_prefill(C.byref(b), C.byref(shape), stream))
    return out


def _validate_tree(q, kp, vp, ksp, vsp, block_table, ctx_lens, sizes, mask, f: Fmt, group: int) -> None:
    if q.dim() != 4:
        _fail(f"q must be [B, T, Hq, D] (got {tuple(q.shape)})")
    B, T, Hq, D = q.shape
    _expect(q, "q", (B, T, Hq, D), torch.float16)
    if (ok := (T >= 1) & (T <= TREE_MAX)) is not True:
        _check(ok, lambda: f"T must be 1 .. {TREE_MAX} (got {T})")
    _check_dg(f, D, group)
    if kp.dim() != 4:
        _fail(f"k_pages must be [num_pages, Hkv, page_rows, row] (got {tuple(kp.shape)})")
    num_pages, Hkv, page_rows, _ = kp.shape
    if (ok := Hkv >= 1) is not True:
        _check(ok, lambda: f"k_pages must have at least one head (got {Hkv})")
    if (ok := Hq % Hkv == 0) is not True:
        _check(ok, lambda: f"query heads ({Hq}) must be a multiple of K/V heads ({Hkv})")
    _check_kv(f, kp, vp, ksp, vsp, (num_pages, Hkv, page_rows), D, group)
    if block_table.dim() != 2:
        _fail(f"block_table must be [B={B}, max_pages] (got {tuple(block_table.shape)})")
    _expect(block_table, "block_table", (B, block_table.shape[1]), torch.int32)
    _expect(ctx_lens, "ctx_lens", (B,), torch.int32)
    if sizes is not None:
        _expect(sizes, "tree_sizes", (B,), torch.int32)
    _expect(mask, "tree_mask", (B, T), torch.int64)


def _decode_tree_fake(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, ctx_lens, tree_sizes, tree_mask, fmt,
      max_seq_len, group=32):
    _validate_tree(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, ctx_lens, tree_sizes, tree_mask,
                   _fmt(fmt), group)
    return q.new_empty(q.shape, dtype=torch.float16)


@_op("decode_tree(Tensor q, Tensor k_pages, Tensor v_pages, Tensor? k_scale_pages, Tensor? v_scale_pages, Tensor block_table, "
     "Tensor ctx_lens, Tensor? tree_sizes, Tensor tree_mask, str fmt, SymInt max_seq_len, int group=32) -> Tensor", _decode_tree_fake)
def decode_tree(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale_pages: Optional[torch.Tensor],
                v_scale_pages: Optional[torch.Tensor], block_table: torch.Tensor, ctx_lens: torch.Tensor,
                tree_sizes: Optional[torch.Tensor], tree_mask: torch.Tensor, fmt: str, max_seq_len: int,
                group: int = 32) -> torch.Tensor:
    """q fp16 [B, T, Hq, D]; pages [num_pages, Hkv, page_rows, ...]; ctx_lens int32 [B]; tree_sizes int32 [B] or
    None (T each); tree_mask int64 [B, T]: bit j of entry i: draft i attends draft j, whose rows are position
    ctx_lens[b] + j. max_seq_len >= every context and its drafts."""
    f = _fmt(fmt)
    _validate_tree(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, ctx_lens, tree_sizes, tree_mask, f,
                   group)
    stream = _ready(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, ctx_lens, tree_sizes, tree_mask)
    B, T, Hq, D = q.shape
    num_pages, Hkv, page_rows = k_pages.shape[:3]
    shape = _PagedShape(B, Hq, Hkv, D, group, page_rows, block_table.shape[1], num_pages, max_seq_len)
    nbytes = lib.va_tree_ws_bytes(int(f), C.byref(shape), T)
    out = torch.empty_like(q)
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=q.device)
    b = _TreeBufs(k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scale_pages), _ptr(v_scale_pages), block_table.data_ptr(),
                  ctx_lens.data_ptr(), _ptr(tree_sizes), tree_mask.data_ptr(), q.data_ptr(), out.data_ptr(), ws.data_ptr())
    check(lib.va_decode_tree(int(f), C.byref(b), C.byref(shape), T, stream))
    return out


def _validate_pools(kp, vp, ksp, vsp, block_table, f: Fmt, group: int) -> None:
    """Pools [num_pages, Hkv, page_rows, row] and block_table [B, max_pages]."""
    if kp.dim() != 4:
        _fail(f"k_pages must be [num_pages, Hkv, page_rows, row] (got {tuple(kp.shape)})")
    row = kp.shape[-1]
    D = row if _BITS[f] == 16 else row * 8 // _BITS[f]
    _check_dg(f, D, group)
    _check_kv(f, kp, vp, ksp, vsp, tuple(kp.shape[:3]), D, group)
    if block_table.dim() != 2:
        _fail(f"block_table must be [B, max_pages] (got {tuple(block_table.shape)})")
    _expect(block_table, "block_table", tuple(block_table.shape), torch.int32)


def _pools(kp, vp, ksp, vsp, block_table, f: Fmt, group: int):
    """(va_pools, va_paged_shape) of checked tensors."""
    num_pages, Hkv, page_rows, row = kp.shape
    D = row if _BITS[f] == 16 else row * 8 // _BITS[f]
    return (_Pools(_ptr(kp), _ptr(vp), _ptr(ksp), _ptr(vsp)),
            _PagedShape(block_table.shape[0], Hkv, Hkv, D, group, page_rows, block_table.shape[1], num_pages, 0))


def _validate_compact(kp, vp, ksp, vsp, block_table, base, keep, counts, f: Fmt, group: int) -> None:
    _validate_pools(kp, vp, ksp, vsp, block_table, f, group)
    B = block_table.shape[0]
    _expect(base, "base", (B,), torch.int32)
    if keep.dim() != 2:
        _fail(f"keep must be [B={B}, n] (got {tuple(keep.shape)})")
    _expect(keep, "keep", (B, keep.shape[1]), torch.int32)
    _check(keep.shape[1] <= TREE_MAX, lambda: f"keep holds at most {TREE_MAX} rows a sequence (got {keep.shape[1]})")
    _expect(counts, "counts", (B,), torch.int32)


def _compact_kv_fake(k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, base, keep, counts, fmt, group=32):
    _validate_compact(k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, base, keep, counts, _fmt(fmt), group)
    return None


@_op("compact_kv(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!)? k_scale_pages, Tensor(d!)? v_scale_pages, "
     "Tensor block_table, Tensor base, Tensor keep, Tensor counts, str fmt, int group=32) -> ()", _compact_kv_fake)
def compact_kv(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale_pages: Optional[torch.Tensor],
               v_scale_pages: Optional[torch.Tensor], block_table: torch.Tensor, base: torch.Tensor,
               keep: torch.Tensor, counts: torch.Tensor, fmt: str, group: int = 32) -> None:
    """For i < counts[b], row base[b] + i of sequence b becomes what row base[b] + keep[b, i] was (K, V, scales)."""
    f = _fmt(fmt)
    _validate_compact(k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, base, keep, counts, f, group)
    stream = _ready(k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, base, keep, counts)
    p, shape = _pools(k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, f, group)
    check(lib.va_compact_kv(int(f), C.byref(p), C.byref(shape), _ptr(block_table), _ptr(base), _ptr(keep),
                            _ptr(counts), keep.shape[1], stream))
    _changed((k_pages, v_pages) if k_scale_pages is None else (k_pages, v_pages, k_scale_pages, v_scale_pages))


def _validate_fork(block_table, seq_lens, parents, refs, kp, vp, ksp, vsp, f: Fmt, group: int) -> None:
    _validate_pools(kp, vp, ksp, vsp, block_table, f, group)
    _expect(seq_lens, "seq_lens", (block_table.shape[0],), torch.int32)
    if parents.dim() != 1:
        _fail(f"parents must be [children] (got {tuple(parents.shape)})")
    _expect(parents, "parents", tuple(parents.shape), torch.int32)
    _expect(refs, "refs", (kp.shape[0],), torch.int32)


def _fork_pages_fake(block_table, seq_lens, parents, refs, k_pages, v_pages, k_scale_pages, v_scale_pages, fmt, group=32):
    _validate_fork(block_table, seq_lens, parents, refs, k_pages, v_pages, k_scale_pages, v_scale_pages, _fmt(fmt), group)
    n = parents.shape[0]
    return block_table.new_empty((n, block_table.shape[1])), block_table.new_empty((n,)), block_table.new_empty((1,))


@_op("fork_pages(Tensor block_table, Tensor seq_lens, Tensor parents, Tensor(a!) refs, Tensor(b!) k_pages, Tensor(c!) v_pages, "
     "Tensor(d!)? k_scale_pages, Tensor(e!)? v_scale_pages, str fmt, int group=32) -> (Tensor, Tensor, Tensor)", _fork_pages_fake)
def fork_pages(block_table: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor, refs: torch.Tensor,
               k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale_pages: Optional[torch.Tensor],
               v_scale_pages: Optional[torch.Tensor], fmt: str,
               group: int = 32) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The next step's sequences: child c continues sequence parents[c] (int32 [children]), sharing its full pages
    (refs int32 [num_pages] counts the holders) and with a last page of its own. Returns (block_table
    [children, max_pages], seq_lens [children], missing [1]: pages that the pool did not have)."""
    f = _fmt(fmt)
    _validate_fork(block_table, seq_lens, parents, refs, k_pages, v_pages, k_scale_pages, v_scale_pages, f, group)
    stream = _ready(block_table, seq_lens, parents, refs, k_pages, v_pages, k_scale_pages, v_scale_pages)
    p, shape = _pools(k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, f, group)
    n = parents.shape[0]
    table = block_table.new_empty((n, block_table.shape[1]))
    lens, missing = block_table.new_empty((n,)), block_table.new_empty((1,))
    check(lib.va_fork_pages(int(f), C.byref(p), C.byref(shape), _ptr(block_table), _ptr(seq_lens), _ptr(parents), n,
                            _ptr(refs), _ptr(table), _ptr(lens), _ptr(missing), stream))
    _changed((refs, k_pages, v_pages) if k_scale_pages is None else (refs, k_pages, v_pages, k_scale_pages, v_scale_pages))
    return table, lens, missing


def _validate_resize(block_table, refs, old_lens, new_lens, page_rows) -> None:
    if block_table.dim() != 2:
        _fail(f"block_table must be [B, max_pages] (got {tuple(block_table.shape)})")
    _expect(block_table, "block_table", tuple(block_table.shape), torch.int32)
    if refs.dim() != 1:
        _fail(f"refs must be [num_pages] (got {tuple(refs.shape)})")
    _expect(refs, "refs", tuple(refs.shape), torch.int32)
    _expect(old_lens, "old_lens", (block_table.shape[0],), torch.int32)
    _expect(new_lens, "new_lens", (block_table.shape[0],), torch.int32)
    _check(page_rows >= 1, lambda: f"page_rows must be >= 1 (got {page_rows})")


def _resize_pages_fake(block_table, refs, old_lens, new_lens, page_rows):
    _validate_resize(block_table, refs, old_lens, new_lens, page_rows)
    return block_table.new_empty((1,))


@_op("resize_pages(Tensor(a!) block_table, Tensor(b!) refs, Tensor old_lens, Tensor new_lens, SymInt page_rows) -> Tensor", _resize_pages_fake)
def resize_pages(block_table: torch.Tensor, refs: torch.Tensor, old_lens: torch.Tensor, new_lens: torch.Tensor,
                 page_rows: int) -> torch.Tensor:
    """Every sequence from old_lens[b] to new_lens[b] positions: pages no longer held are given up (0 frees the
    sequence), missing ones handed out, lowest free id (refs 0) first. Returns how many the pool did not have, [1]."""
    _validate_resize(block_table, refs, old_lens, new_lens, page_rows)
    stream = _ready(block_table, refs, old_lens, new_lens)
    missing = block_table.new_empty((1,))
    check(lib.va_resize_pages(block_table.shape[0], page_rows, block_table.shape[1], refs.shape[0], _ptr(block_table),
                              _ptr(refs), _ptr(old_lens), _ptr(new_lens), _ptr(missing), stream))
    _changed((block_table, refs))
    return missing


# ------------------------------------- rotating cache write, block-scaled cache --

def _block_pools(kp, vp, ksp, vsp, num_pages, Hkv, page_rows, D, group: int) -> None:
    """Checks of pools of the format b8+: e4m3 codes, a scale for `group` positions of a head."""
    if group not in (32, 64):
        _fail(f"group must be 32 or 64 (got {group})")
    if (ok := page_rows % group == 0) is not True:
        _check(ok, lambda: f"page_rows must be a multiple of group (got {page_rows}, group={group})")
    _expect(kp, "k_pages", (num_pages, Hkv, page_rows, D), torch.float8_e4m3fn)
    _expect(vp, "v_pages", (num_pages, Hkv, page_rows, D), torch.float8_e4m3fn)
    _expect(ksp, "k_scale_pages", (num_pages, Hkv, page_rows // group), torch.float16)
    _expect(vsp, "v_scale_pages", (num_pages, Hkv, page_rows // group), torch.float16)


def _validate_bounds(cu, T, B) -> None:
    if cu is None:
        if (ok := T == B) is not True:
            _check(ok, lambda: f"without cu_seqlens there is a row to each sequence (got {T} rows, {B} sequences)")
    else:
        _expect(cu, "cu_seqlens", (B + 1,), torch.int32)


def _validate_rope(q, k, v, inv_freq, cu, start, positions, block_table, kp, vp, ksp, vsp, fmt: str, group: int) -> None:
    if q.dim() != 3:
        _fail(f"q must be [T, Hq, D] (got {tuple(q.shape)})")
    T, Hq, D = q.shape
    _expect(q, "q", (T, Hq, D), torch.float16)
    if (ok := (D == 64) | (D == 128)) is not True:
        _check(ok, lambda: f"D must be 64 or 128 (got {D})")
    if k.dim() != 3:
        _fail(f"k must be [T, Hkv, D] (got {tuple(k.shape)})")
    Hkv = k.shape[1]
    if (ok := (Hkv >= 1) & (Hq >= 1)) is not True:
        _check(ok, lambda: f"q and k must have at least one head (got {Hq} and {Hkv})")
    _expect(k, "k", (T, Hkv, D), torch.float16)
    _expect(v, "v", (T, Hkv, D), torch.float16)
    if inv_freq.dim() != 1:
        _fail(f"inv_freq must be [rot / 2] (got {tuple(inv_freq.shape)})")
    half = inv_freq.shape[0]
    _expect(inv_freq, "inv_freq", (half,), torch.float32)
    if (ok := (half >= 8) & (half % 8 == 0) & (2 * half <= D)) is not True:
        _check(ok, lambda: f"inv_freq must have a multiple of 8 entries, D / 2 at most (got {half})")
    if start.dim() != 1:
        _fail(f"start must be [B] (got {tuple(start.shape)})")
    B = start.shape[0]
    _expect(start, "start", (B,), torch.int32)
    if (ok := B >= 1) is not True:
        _check(ok, lambda: "start must have at least one sequence")
    _validate_bounds(cu, T, B)
    if positions is not None:
        _expect(positions, "positions", (T,), torch.int32)
    if block_table.dim() != 2:
        _fail(f"block_table must be [B={B}, max_pages] (got {tuple(block_table.shape)})")
    _expect(block_table, "block_table", (B, block_table.shape[1]), torch.int32)
    if kp.dim() != 4:
        _fail(f"k_pages must be [num_pages, Hkv, page_rows, row] (got {tuple(kp.shape)})")
    num_pages, _, page_rows, _ = kp.shape
    if fmt == "b8+":
        _block_pools(kp, vp, ksp, vsp, num_pages, Hkv, page_rows, D, group)
    else:
        f = _fmt(fmt)
        _check_dg(f, D, group)
        _check_kv(f, kp, vp, ksp, vsp, (num_pages, Hkv, page_rows), D, group)


def _append_rope_fake(q, k, v, inv_freq, cu_seqlens, start, positions, block_table, k_pages, v_pages, k_scale_pages, v_scale_pages, fmt,
                      group=32, interleaved=False, rotated_k=False, scaling=1.0):
    _validate_rope(q, k, v, inv_freq, cu_seqlens, start, positions, block_table, k_pages, v_pages, k_scale_pages, v_scale_pages, fmt, group)
    return q.new_empty(q.shape), k.new_empty(k.shape if rotated_k else (0,) + k.shape[1:])


@_op("append_rope(Tensor q, Tensor k, Tensor v, Tensor inv_freq, Tensor? cu_seqlens, Tensor start, Tensor? positions, Tensor block_table, "
     "Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!)? k_scale_pages, Tensor(d!)? v_scale_pages, str fmt, int group=32, "
     "bool interleaved=False, bool rotated_k=False, float scaling=1.0) -> (Tensor, Tensor)", _append_rope_fake, computes=True, native=True)
def append_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, inv_freq: torch.Tensor, cu_seqlens: Optional[torch.Tensor],
                start: torch.Tensor, positions: Optional[torch.Tensor], block_table: torch.Tensor, k_pages: torch.Tensor,
                v_pages: torch.Tensor, k_scale_pages: Optional[torch.Tensor], v_scale_pages: Optional[torch.Tensor], fmt: str,
                group: int = 32, interleaved: bool = False, rotated_k: bool = False,
                scaling: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """q fp16 [T, Hq, D], k and v [T, Hkv, D], dense in D only (slices of a fused projection); rows cu_seqlens[b] ..
    cu_seqlens[b+1] - 1 (None: row b) are sequence b's, written at positions start[b] on. q and k are rotated by
    inv_freq fp32 [rot / 2] times their cache position, or positions int32 [T]; dimensions i and i + rot/2 are a pair
    (interleaved: 2i and 2i + 1). fmt: any; "b8+": pages float8_e4m3fn [num_pages, Hkv, page_rows, D], scales fp16
    [num_pages, Hkv, page_rows / group]. Returns q [T, Hq, D] and, if rotated_k, k [T, Hkv, D] (else [0, Hkv, D])."""
    _validate_rope(q, k, v, inv_freq, cu_seqlens, start, positions, block_table, k_pages, v_pages, k_scale_pages, v_scale_pages, fmt, group)
    stream = _on_device(q, k, v, inv_freq, cu_seqlens, start, positions, block_table, k_pages, v_pages, k_scale_pages, v_scale_pages)
    _contiguous(inv_freq, cu_seqlens, start, positions, block_table, k_pages, v_pages, k_scale_pages, v_scale_pages)
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    q_out = torch.empty((T, Hq, D), dtype=torch.float16, device=q.device)
    k_out = torch.empty((T if rotated_k else 0, Hkv, D), dtype=torch.float16, device=q.device)
    if T == 0:
        return q_out, k_out
    num_pages, _, page_rows, _ = k_pages.shape
    shape = _RopeShape(start.shape[0], T, Hq, Hkv, D, group, page_rows, block_table.shape[1], num_pages, 2 * inv_freq.shape[0],
                       interleaved, scaling, *_strides("q", q), *_strides("k", k), *_strides("v", v))
    b = _RopeBufs(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(cu_seqlens), start.data_ptr(), _ptr(positions), block_table.data_ptr(),
                  inv_freq.data_ptr(), q_out.data_ptr(), k_out.data_ptr() if rotated_k else None, k_pages.data_ptr(), v_pages.data_ptr(),
                  _ptr(k_scale_pages), _ptr(v_scale_pages))
    check(lib.va_append_rope(B8 if fmt == "b8+" else int(_fmt(fmt)), C.byref(b), C.byref(shape), stream))
    _changed((k_pages, v_pages) if k_scale_pages is None else (k_pages, v_pages, k_scale_pages, v_scale_pages))
    return q_out, k_out


def _validate_attend(q, kp, vp, ksp, vsp, block_table, cu, seq_lens, fmt: str, group: int) -> None:
    if fmt != "b8+":
        _fail(f"attend_paged takes the format b8+ only (got {fmt!r})")
    if q.dim() != 3:
        _fail(f"q must be [T, Hq, D] (got {tuple(q.shape)})")
    T, Hq, D = q.shape
    _expect(q, "q", (T, Hq, D), torch.float16)
    if (ok := (D == 64) | (D == 128)) is not True:
        _check(ok, lambda: f"D must be 64 or 128 (got {D})")
    if kp.dim() != 4:
        _fail(f"k_pages must be [num_pages, Hkv, page_rows, D] (got {tuple(kp.shape)})")
    num_pages, Hkv, page_rows, _ = kp.shape
    if (ok := (Hkv >= 1) & (Hq >= 1)) is not True:
        _check(ok, lambda: f"q and k_pages must have at least one head (got {Hq} and {Hkv})")
    if (ok := Hq % Hkv == 0) is not True:
        _check(ok, lambda: f"query heads ({Hq}) must be a multiple of K/V heads ({Hkv})")
    _block_pools(kp, vp, ksp, vsp, num_pages, Hkv, page_rows, D, group)
    if block_table.dim() != 2:
        _fail(f"block_table must be [B, max_pages] (got {tuple(block_table.shape)})")
    B = block_table.shape[0]
    _expect(block_table, "block_table", (B, block_table.shape[1]), torch.int32)
    _expect(seq_lens, "seq_lens", (B,), torch.int32)
    _validate_bounds(cu, T, B)


def _attend_paged_fake(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, cu_seqlens, seq_lens, fmt, max_seq_len, group=32):
    _validate_attend(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, cu_seqlens, seq_lens, fmt, group)
    return q.new_empty(q.shape)


@_op("attend_paged(Tensor q, Tensor k_pages, Tensor v_pages, Tensor k_scale_pages, Tensor v_scale_pages, Tensor block_table, "
     "Tensor? cu_seqlens, Tensor seq_lens, str fmt, SymInt max_seq_len, int group=32) -> Tensor", _attend_paged_fake, native=True)
def attend_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale_pages: torch.Tensor, v_scale_pages: torch.Tensor,
                 block_table: torch.Tensor, cu_seqlens: Optional[torch.Tensor], seq_lens: torch.Tensor, fmt: str, max_seq_len: int,
                 group: int = 32) -> torch.Tensor:
    """q fp16 [T, Hq, D], the newest tokens of every sequence, whose rows are in the cache already: rows cu_seqlens[b] ..
    cu_seqlens[b+1] - 1 (int32 [B + 1]; None: row b) are the last of sequence b's seq_lens[b] positions; each attends
    the positions up to its own. fmt "b8+": pages float8_e4m3fn [num_pages, Hkv, page_rows, D], scales fp16
    [num_pages, Hkv, page_rows / group]. max_seq_len >= every length."""
    _validate_attend(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, cu_seqlens, seq_lens, fmt, group)
    if max_seq_len > 2147483647:
        _fail(f"max_seq_len must be below 2^31 (got {max_seq_len})")
    stream = _ready(q, k_pages, v_pages, k_scale_pages, v_scale_pages, block_table, cu_seqlens, seq_lens)
    T, Hq, D = q.shape
    num_pages, Hkv, page_rows, _ = k_pages.shape
    shape = _PagedShape(block_table.shape[0], Hq, Hkv, D, group, page_rows, block_table.shape[1], num_pages, max_seq_len)
    out = torch.empty_like(q)
    ws = torch.empty(lib.va_attend_ws_bytes(B8, C.byref(shape), T) // 4, dtype=torch.float32, device=q.device)
    b = _AttendBufs(k_pages.data_ptr(), v_pages.data_ptr(), k_scale_pages.data_ptr(), v_scale_pages.data_ptr(), block_table.data_ptr(),
                    _ptr(cu_seqlens), seq_lens.data_ptr(), q.data_ptr(), out.data_ptr(), ws.data_ptr())
    check(lib.va_attend_paged(B8, C.byref(b), C.byref(shape), T, stream))
    return out


def row_format_bits(fmt: str) -> int:
    return _BITS[_fmt(fmt)]


def _load_calls(path: Path = Path(__file__).resolve().parent / "libvoltattn_torch.so") -> None:
    """host/torch_calls.cpp's plain calls: the C ABI's functions by their addresses in the library
    that is loaded. Where it was built without PyTorch, or for another one, these ops' plain calls go
    through Python too, to the same kernels: said once, and nothing else changes. Without a GPU nothing
    calls them."""
    why = "is not built"
    if path.exists():
        if b"voltattn calls for PyTorch " + re.match(r"\d+\.\d+\.\d+", torch.__version__)[0].encode() + b"\0" not in path.read_bytes():
            why = f"was built for another PyTorch than {torch.__version__}"
        else:
            try:
                torch.ops.load_library(str(path))
                torch.ops.voltattn._bind([C.cast(f, C.c_void_p).value for f in (lib.va_append_rope, lib.va_attend_paged, lib.va_attend_ws_bytes)])
                return
            except OSError as e:
                why = f"does not load ({e})"
    if torch.cuda.device_count() > 0:
        warnings.warn(f"{path} {why}: append_rope and attend_paged take about 10 us more of host time a call; "
                      "run `python voltattn_amd/build.py` (needs g++)", stacklevel=2)


_load_calls()

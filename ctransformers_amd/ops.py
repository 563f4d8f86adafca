"""Operators on device memory, called with torch tensors (include/ctransformers_amd_ops.h is the C interface): a KV cache held in 4 bits, in pages that
several sequences may share.

    pages = torch.zeros(n_pages, kv4_page_bytes(n_head_kv, head_dim, 64), dtype=torch.uint8, device="cuda")      # one layer's cache
    table, lens, refs, short = kv_reserve(pages, table, lens, refs, add, page_tokens=64)                          # room for `add` more tokens each
    kv4_append(k, v, pages, table, lens, cu, max_rows, page_tokens=64)                                            # rows -> 4.5 bits a value
    out = kv4_attention(q, pages, table, lens, cu, max_rows, n_head_kv=n_head_kv, page_tokens=64)                 # causal, grouped heads
    table, lens, refs = kv_fork(table, lens, refs, parents, page_tokens=64)                                       # beams; parent -1 frees a sequence
    table, refs, used = kv_compact(pages, table, refs)                                                            # pages in use to the front

Sequences are packed: rows ``cu[b] .. cu[b + 1] - 1`` of q, k and v are the LAST rows of sequence b, whose length with them is ``lens[b]``; no sequence may
have more than ``max_rows`` of them (rows beyond are not processed).  ``cu=None``: one sequence, all rows.  table, lens, cu, refs, parents and add are int32
tensors on the device; a table entry outside [0, n_pages) names no page (rows for it are not stored, its tokens are not attended to).

Every operator runs on the current stream of its tensors' device and returns without waiting for it; nothing is kept between calls.  Workspaces and results come from
torch's allocator, so calls can be captured into a graph and several graphs share nothing.  What a user may get wrong raises ValueError / TypeError before anything is
launched.  There is no CPU path: without the HIP library, or with tensors elsewhere than on a GPU, a call raises.  No operator has a gradient.
"""
import ctypes
import math
import os
from ctypes import POINTER, Structure, byref, c_float, c_int, c_longlong, c_void_p

import torch

from .llm import find_library

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class _Cache(Structure):
    _fields_ = [("pages", c_void_p), ("table", c_void_p), ("lens", c_void_p), ("cu", c_void_p), ("page_stride", c_longlong), ("n_pages", c_int),
                ("table_stride", c_int), ("table_width", c_int), ("n_seq", c_int), ("total", c_int), ("n_head_kv", c_int), ("head_dim", c_int),
                ("page_tokens", c_int), ("max_rows", c_int)]


class _Rows(Structure):
    _fields_ = [("p", c_void_p), ("row", c_longlong), ("head", c_longlong), ("dim", c_longlong), ("type", c_int)]


class _Tables(Structure):
    _fields_ = [("table", c_void_p), ("lens", c_void_p), ("refs", c_void_p), ("table_out", c_void_p), ("lens_out", c_void_p), ("refs_out", c_void_p),
                ("n_seq", c_int), ("width", c_int), ("n_pages", c_int), ("page_tokens", c_int)]


# name -> (restype, argtypes); the CPU test-suite checks include/ctransformers_amd_ops.h and the built library against this table
ABI = {
    "ctamd_ops_error": (ctypes.c_char_p, []),
    "ctamd_ops_host_memory": (c_int, []),
    "ctamd_kv4_page_bytes": (c_longlong, [c_int, c_int, c_int]),
    "ctamd_kv4_append": (c_int, [POINTER(_Cache), POINTER(_Rows), POINTER(_Rows), c_void_p]),
    "ctamd_kv4_read": (c_int, [POINTER(_Cache), POINTER(_Rows), POINTER(_Rows), c_void_p]),
    "ctamd_kv4_attention_ws": (c_longlong, [POINTER(_Cache), c_int]),
    "ctamd_kv4_attention": (c_int, [POINTER(_Cache), c_int, POINTER(_Rows), POINTER(_Rows), c_float, c_void_p, c_longlong, c_void_p]),
    "ctamd_kv_fork": (c_int, [POINTER(_Tables), c_void_p, c_int, c_void_p]),
    "ctamd_kv_reserve_ws": (c_longlong, [c_int, c_int]),
    "ctamd_kv_reserve": (c_int, [POINTER(_Tables), c_void_p, c_void_p, c_int, c_longlong, c_longlong, c_void_p, c_void_p, c_void_p]),
    "ctamd_kv_compact_ws": (c_longlong, [c_int]),
    "ctamd_kv_compact": (c_int, [POINTER(_Tables), c_void_p, c_int, c_longlong, c_longlong, c_void_p, c_void_p, c_void_p]),
}
_lib = None
_device = "cuda"


def load(path=None):
    """Binds the library (`path`: another one than the package's).  Called by the first operator; returns the ctypes library."""
    global _lib, _device
    lib = ctypes.CDLL(find_library(path))
    for name, (restype, argtypes) in ABI.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = restype, argtypes
    if not lib.ctamd_ops_host_memory() and os.path.exists("/proc/self/maps"):
        with open("/proc/self/maps") as f:
            runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
        if len(runtimes) > 1:   # a stream of one runtime means nothing to the other
            raise RuntimeError("two HIP runtimes in this process (%s): import torch before the first model is loaded" % ", ".join(sorted(runtimes)))
    _device = "cpu" if lib.ctamd_ops_host_memory() else "cuda"
    _lib = lib
    return lib


def _library():
    return _lib if _lib is not None else load()


def _call(code):
    if code:
        raise ValueError(_lib.ctamd_ops_error().decode())


class _On:
    """The tensors' device made current for a call, if it is not; `stream` is its current stream."""
    __slots__ = ("guard", "stream")

    def __init__(self, device):
        self.guard = None
        if device.type != "cuda":
            self.stream = None
            return
        if device.index is not None and device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(device)
            self.guard.__enter__()
        self.stream = torch.cuda.current_stream().cuda_stream

    def __enter__(self):
        return self.stream

    def __exit__(self, *what):
        if self.guard is not None:
            self.guard.__exit__(*what)


def _ints(name, x, device, *shape):
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32:
        raise TypeError("%s is an int32 tensor" % name)
    if x.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, x.device, device))
    if x.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, x.shape)):
        raise ValueError("%s has shape %s" % (name, tuple(x.shape)))
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError("the entries of %s are not adjacent" % name)


def _rows(name, x, device, shape=None):
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES:
        raise TypeError("%s is a float16, bfloat16 or float32 tensor" % name)
    if x.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, x.device, device))
    if x.dim() != 3 or (shape is not None and tuple(x.shape) != tuple(shape)):
        raise ValueError("%s has shape %s%s" % (name, tuple(x.shape), "" if shape is None else ", not %s" % (tuple(shape),)))
    s = x.stride()
    return _Rows(x.data_ptr(), s[0], s[1], s[2], _TYPES[x.dtype])


def _cache(pages, table, lens, cu, total, n_head_kv, head_dim, page_tokens, max_rows):
    _library()
    if not isinstance(pages, torch.Tensor) or pages.dtype != torch.uint8:
        raise TypeError("pages is a uint8 tensor")
    device = pages.device
    if device.type != _device:
        raise ValueError("pages is on %s: the operators run on GPU memory only" % device)
    width = _lib.ctamd_kv4_page_bytes(n_head_kv, head_dim, page_tokens)
    if not width:
        raise ValueError("sizes not supported: head_dim %s (a multiple of 8 up to 256), page_tokens %s (32, 64, 128 or 256), n_head_kv %s (1 .. 1024)"
                         % (head_dim, page_tokens, n_head_kv))
    if pages.dim() != 2 or pages.shape[1] != width or pages.stride(1) != 1:
        raise ValueError("pages has shape %s, not [n_pages, %d] with adjacent bytes" % (tuple(pages.shape), width))
    _ints("table", table, device, None, None)
    n_seq = table.shape[0]
    _ints("lens", lens, device, n_seq)
    if cu is not None:
        _ints("cu", cu, device, n_seq + 1)
    elif n_seq != 1:
        raise ValueError("cu is needed for more than one sequence")
    if n_seq > 1 and table.stride(0) < table.shape[1]:
        raise ValueError("the rows of table overlap")
    if max_rows < 0:
        raise ValueError("max_rows is negative")
    return _Cache(pages.data_ptr(), table.data_ptr(), lens.data_ptr(), cu.data_ptr() if cu is not None else None, pages.stride(0), pages.shape[0],
                  max(table.stride(0), table.shape[1]), table.shape[1], n_seq, total, n_head_kv, head_dim, page_tokens, min(max_rows, total))


def kv4_page_bytes(n_head_kv, head_dim, page_tokens):
    """Bytes of a page of `page_tokens` tokens (32, 64, 128 or 256): 4.5 bits for each of K's and V's values, head_dim rounded up to 32."""
    n = _library().ctamd_kv4_page_bytes(n_head_kv, head_dim, page_tokens)
    if not n:
        raise ValueError("sizes not supported: head_dim is a multiple of 8 up to 256, page_tokens 32, 64, 128 or 256, n_head_kv 1 .. 1024")
    return n


def kv4_append(k, v, pages, table, lens, cu, max_rows, *, page_tokens):
    """Quantizes the rows k, v [total, n_head_kv, head_dim] (any strides) into the pages; row i of a sequence with n of them goes to position lens - n + i.

    A group of 32 dims of a token becomes f16(d) * (code - 8), code 0 .. 15, d = the value of largest magnitude / -8 (the rounding of Q4_0 weights); values beyond
    +-65504 are stored as that.  A token whose K or V of a head holds a NaN makes every row that sees it NaN.  No two sequences of a call may write one page."""
    if not isinstance(pages, torch.Tensor):
        raise TypeError("pages is a uint8 tensor")
    device = pages.device
    kr, vr = _rows("k", k, device), _rows("v", v, device, k.shape)
    c = _cache(pages, table, lens, cu, k.shape[0], k.shape[1], k.shape[2], page_tokens, max_rows)
    with _On(device) as stream:
        _call(_lib.ctamd_kv4_append(byref(c), byref(kr), byref(vr), stream))


def kv4_read(pages, table, lens, cu, max_rows, total, *, n_head_kv, head_dim, page_tokens, dtype=torch.float16):
    """The last rows of every sequence as (k, v) [total, n_head_kv, head_dim]; 0 where there is no page or no position.  Rows of no sequence are undefined."""
    if dtype not in _TYPES:
        raise TypeError("dtype is float16, bfloat16 or float32")
    c = _cache(pages, table, lens, cu, total, n_head_kv, head_dim, page_tokens, max_rows)
    device = pages.device
    with _On(device) as stream:
        k = torch.empty((total, n_head_kv, head_dim), dtype=dtype, device=device)
        v = torch.empty((total, n_head_kv, head_dim), dtype=dtype, device=device)
        _call(_lib.ctamd_kv4_read(byref(c), byref(_rows("k", k, device)), byref(_rows("v", v, device)), stream))
    return k, v


def kv4_attention(q, pages, table, lens, cu, max_rows, *, n_head_kv, page_tokens, scale=None, out=None):
    """Causal attention of the rows q [total, n_head, head_dim] over the cache: row i of a sequence with n rows sees the positions 0 .. lens - n + i, query head h
    reads KV head h // (n_head / n_head_kv), scores are q.k * scale (default 1 / sqrt(head_dim)).  A row that sees nothing becomes 0.  q is float16, bfloat16 or
    float32; the result has q's type, or is written into `out` [total, n_head, head_dim] of any of the three, where rows that belong to no sequence are left as they
    are.  Products are taken in float16 (K's codes and V's values; q scaled by a power of two per row, and p), everything else in float32."""
    if not isinstance(pages, torch.Tensor):
        raise TypeError("pages is a uint8 tensor")
    device = pages.device
    qr = _rows("q", q, device)
    total, n_head, head_dim = q.shape
    if n_head_kv < 1 or n_head < 1 or n_head % n_head_kv:
        raise ValueError("%d query heads over %d KV heads" % (n_head, n_head_kv))
    if qr.dim != 1 and head_dim > 1:
        q = q.contiguous()
        qr = _rows("q", q, device)
    c = _cache(pages, table, lens, cu, total, n_head_kv, head_dim, page_tokens, max_rows)
    with _On(device) as stream:
        if out is None:
            out = torch.empty((total, n_head, head_dim), dtype=q.dtype, device=device)
        orow = _rows("out", out, device, q.shape)
        n = _lib.ctamd_kv4_attention_ws(byref(c), n_head)
        ws = torch.empty(n, dtype=torch.float32, device=device) if n else None
        _call(_lib.ctamd_kv4_attention(byref(c), n_head, byref(qr), byref(orow), 1.0 / math.sqrt(head_dim) if scale is None else scale,
                                       ws.data_ptr() if n else None, n, stream))
    return out


def _tables(table, lens, refs, page_tokens, rows):
    _library()
    if not isinstance(table, torch.Tensor) or table.device.type != _device:
        raise ValueError("table is a tensor in GPU memory")
    device = table.device
    _ints("table", table, device, None, None)
    _ints("refs", refs, device, None)
    if lens is not None:
        _ints("lens", lens, device, table.shape[0])
    if page_tokens < 1:
        raise ValueError("page_tokens is positive")
    if not table.is_contiguous():
        table = table.contiguous()
    n = table.shape[0] if rows is None else rows
    new = (torch.empty((n, table.shape[1]), dtype=torch.int32, device=device),
           torch.empty((n,), dtype=torch.int32, device=device) if lens is not None else None, torch.empty_like(refs))
    t = _Tables(table.data_ptr(), lens.data_ptr() if lens is not None else None, refs.data_ptr(), new[0].data_ptr(),
                new[1].data_ptr() if lens is not None else None, new[2].data_ptr(), table.shape[0], table.shape[1], refs.shape[0], page_tokens)
    return t, new, table


def _pool(pages, refs):
    if not isinstance(pages, torch.Tensor) or pages.device != refs.device:
        raise ValueError("pages is a tensor on the device of the tables")
    if pages.dim() not in (2, 3) or pages.shape[-2] != refs.shape[0]:
        raise ValueError("pages has shape %s: [n_pages, page] or [layers, n_pages, page] with %d pages" % (tuple(pages.shape), refs.shape[0]))
    if pages.stride(-1) != 1 or pages.stride(-2) != pages.shape[-1]:
        raise ValueError("the pages of a layer are not adjacent")
    e = pages.element_size()
    return (pages.data_ptr(), pages.shape[0], pages.stride(0) * e, pages.shape[-1] * e) if pages.dim() == 3 else (
        pages.data_ptr(), 1, pages.shape[0] * pages.shape[1] * e, pages.shape[1] * e)


def kv_fork(table, lens, refs, parents, *, page_tokens):
    """(table, lens, refs) of a batch whose sequence i continues sequence parents[i], sharing its pages: the batch may grow, shrink, permute and repeat, a parent
    outside [0, n_seq) makes an empty sequence (-1: freed).  A page whose last reference goes is free.  table [n_seq, width], refs [n_pages]."""
    _library()
    if not isinstance(parents, torch.Tensor) or parents.dim() != 1:
        raise TypeError("parents is an int32 tensor with one dimension")
    t, new, keep = _tables(table, lens, refs, page_tokens, parents.shape[0])
    _ints("parents", parents, table.device, None)
    with _On(table.device) as stream:
        _call(_lib.ctamd_kv_fork(byref(t), parents.data_ptr(), parents.shape[0], stream))
    return new


def kv_reserve(pages, table, lens, refs, add, *, page_tokens):
    """(table, lens, refs, short) with room for add[i] more tokens in sequence i: lens grows by it, pages are taken lowest free first in the order of the sequences,
    and a last page that others share is copied before its sequence writes it.  pages: [n_pages, ..] or [layers, n_pages, ..], any type.  short (int32, on the
    device): 0, or the pages that were missing, or -1 where a sequence outgrows its row of the table; then nothing has changed."""
    t, new, keep = _tables(table, lens, refs, page_tokens, None)
    device = table.device
    _ints("add", add, device, table.shape[0])
    p = _pool(pages, refs)
    with _On(device) as stream:
        short = torch.empty((), dtype=torch.int32, device=device)
        ws = torch.empty(_lib.ctamd_kv_reserve_ws(table.shape[0], refs.shape[0]), dtype=torch.int32, device=device)
        _call(_lib.ctamd_kv_reserve(byref(t), add.data_ptr(), p[0], p[1], p[2], p[3], short.data_ptr(), ws.data_ptr(), stream))
    return new + (short,)


def kv_compact(pages, table, refs):
    """(table, refs, used) after the pages in use have become pages 0 .. used - 1: those beyond move, in order, into the holes below.  used: int32, on the device."""
    t, new, keep = _tables(table, None, refs, 1, None)
    device = table.device
    p = _pool(pages, refs)
    with _On(device) as stream:
        used = torch.empty((), dtype=torch.int32, device=device)
        ws = torch.empty(_lib.ctamd_kv_compact_ws(refs.shape[0]), dtype=torch.int32, device=device)
        _call(_lib.ctamd_kv_compact(byref(t), p[0], p[1], p[2], p[3], used.data_ptr(), ws.data_ptr(), stream))
    return new[0], new[2], used

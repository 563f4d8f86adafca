"""Operators on device memory, called with torch tensors (include/ctransformers_amd_ops.h is the C interface): a KV cache held in 4 bits, in pages that
several sequences may share.

    pages = torch.zeros(n_pages, kv4_page_bytes(n_head_kv, head_dim, 64), dtype=torch.uint8, device="cuda")      # one layer's cache
    table, lens, refs, short = kv_reserve(pages, table, lens, refs, add, page_tokens=64)                          # room for `add` more tokens each
    kv4_append(k, v, pages, table, lens, cu, max_rows, page_tokens=64)                                            # rows -> 4.5 bits a value
    out = kv4_attention(q, pages, table, lens, cu, max_rows, n_head_kv=n_head_kv, page_tokens=64)                 # causal, grouped heads
    table, lens, refs = kv_fork(table, lens, refs, parents, page_tokens=64)                                       # beams; parent -1 frees a sequence
    table, refs, used = kv_compact(pages, table, refs)                                                            # pages in use to the front

Sequences are packed: rows ``cu[b] .. cu[b + 1] - 1`` of q, k and v are the LAST rows of sequence b, whose length with them is ``lens[b]``; ``cu`` ascends, and
no sequence may have more than ``max_rows`` rows (rows beyond are not processed).  ``cu=None``: one sequence, all rows.  table, lens, cu, refs, parents and add are int32
tensors on the device; a table entry outside [0, n_pages) names no page (rows for it are not stored, its tokens are not attended to).

Every operator runs on the current stream of its tensors' device and returns without waiting for it; nothing is kept between calls.  Workspaces and results come from
torch's allocator, so calls can be captured into a graph and several graphs share nothing.  What a user may get wrong raises ValueError / TypeError before anything is
launched.  There is no CPU path: without the HIP library, or with tensors elsewhere than on a GPU, a call raises.  No operator has a gradient:
q, k, v or out that require one are refused unless gradients are off.
"""
import ctypes
import math
import os
from ctypes import c_char_p, c_float, c_int, c_longlong, c_void_p
from struct import Struct

import torch

from .llm import find_library

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_INT = torch.int32

# The C structures as packed bytes (a token step calls an operator per layer: building ctypes structures field by field costs more than the GPU's work at small sizes)
CACHE = Struct("@4Pq9i4x")    # ctamd_kv4_cache
ROWS = Struct("@P3qi4x")      # ctamd_rows
TABLES = Struct("@6P4i")      # ctamd_kv_tables

# name -> (restype, argtypes); the CPU test-suite checks include/ctransformers_amd_ops.h and the built library against this table
ABI = {
    "ctamd_ops_error": (c_char_p, []),
    "ctamd_ops_host_memory": (c_int, []),
    "ctamd_kv4_page_bytes": (c_longlong, [c_int, c_int, c_int]),
    "ctamd_kv4_append": (c_int, [c_char_p, c_char_p, c_char_p, c_void_p]),
    "ctamd_kv4_read": (c_int, [c_char_p, c_char_p, c_char_p, c_void_p]),
    "ctamd_kv4_attention_ws": (c_longlong, [c_char_p, c_int]),
    "ctamd_kv4_attention": (c_int, [c_char_p, c_int, c_char_p, c_char_p, c_float, c_void_p, c_longlong, c_void_p]),
    "ctamd_kv_fork": (c_int, [c_char_p, c_void_p, c_void_p, c_int, c_void_p]),
    "ctamd_kv_reserve_ws": (c_longlong, [c_int, c_int]),
    "ctamd_kv_reserve": (c_int, [c_char_p, c_void_p, c_void_p, c_int, c_longlong, c_longlong, c_void_p, c_void_p, c_void_p]),
    "ctamd_kv_compact_ws": (c_longlong, [c_int]),
    "ctamd_kv_compact": (c_int, [c_char_p, c_void_p, c_int, c_longlong, c_longlong, c_void_p, c_void_p, c_void_p]),
}
_lib = None
_on_gpu = True
# the address of a device's current stream without making a Stream object of it, where torch has that
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def load(path=None):
    """Binds the library (`path`: another one than the package's).  Called by the first operator; returns the ctypes library."""
    global _lib, _on_gpu
    lib = ctypes.CDLL(find_library(path))
    for name, (restype, argtypes) in ABI.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = restype, argtypes
    on_gpu = not lib.ctamd_ops_host_memory()
    if on_gpu and os.path.exists("/proc/self/maps"):
        with open("/proc/self/maps") as f:
            runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
        if len(runtimes) > 1:   # a stream of one runtime means nothing to the other
            raise RuntimeError("two HIP runtimes in this process (%s): import torch before the first model is loaded" % ", ".join(sorted(runtimes)))
    _lib, _on_gpu = lib, on_gpu
    return lib


def _launch(device, fn):
    """fn(stream) with the tensors' device (its index) current, on that device's current stream."""
    if device < 0:
        code = fn(None)
    elif device == torch.cuda.current_device():
        code = fn(_stream(device))
    else:
        with torch.cuda.device(device):
            code = fn(_stream(device))
    if code:
        raise ValueError(_lib.ctamd_ops_error().decode())


def _ints(device, name, x, dims, rows=None):
    """x: int32, `dims`-dimensional, entries adjacent, `rows` of them; returns its address."""
    if not isinstance(x, torch.Tensor) or x.dtype is not _INT:
        raise TypeError("%s is an int32 tensor" % name)
    if x.get_device() != device:
        raise ValueError("%s is on %s, not on device %d" % (name, x.device, device))
    shape = x.shape
    if len(shape) != dims or (rows is not None and shape[0] != rows):
        raise ValueError("%s has shape %s" % (name, tuple(shape)))
    if x.stride()[-1] != 1 and shape[-1] > 1:
        raise ValueError("the entries of %s are not adjacent" % name)
    return x.data_ptr()


def _rows(device, name, x, shape=None):
    t = _TYPES.get(x.dtype) if isinstance(x, torch.Tensor) else None
    if t is None:
        raise TypeError("%s is a float16, bfloat16 or float32 tensor" % name)
    if x.get_device() != device:
        raise ValueError("%s is on %s, not on device %d" % (name, x.device, device))
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires a gradient, and no operator has one: detach it, or call under torch.no_grad()" % name)
    if len(x.shape) != 3 or (shape is not None and x.shape != shape):
        raise ValueError("%s has shape %s%s" % (name, tuple(x.shape), "" if shape is None else ", not %s" % (tuple(shape),)))
    return ROWS.pack(x.data_ptr(), *x.stride(), t)


def _device_of(name, x):
    if _lib is None:
        load()
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s is a tensor" % name)
    device = x.get_device()
    if (device < 0) is _on_gpu:
        raise ValueError("%s is on %s: the operators run on GPU memory only" % (name, x.device))
    return device


def _cache(device, pages, table, lens, cu, total, n_head_kv, head_dim, page_tokens, max_rows):
    if pages.dtype is not torch.uint8:
        raise TypeError("pages is a uint8 tensor")
    width = _lib.ctamd_kv4_page_bytes(n_head_kv, head_dim, page_tokens)
    if not width:
        raise ValueError("sizes not supported: head_dim %s (a multiple of 8 up to 256), page_tokens %s (32, 64, 128 or 256), n_head_kv %s (1 .. 1024)"
                         % (head_dim, page_tokens, n_head_kv))
    shape, step = pages.shape, pages.stride()
    if len(shape) != 2 or shape[1] != width or step[1] != 1:
        raise ValueError("pages has shape %s, not [n_pages, %d] with adjacent bytes" % (tuple(shape), width))
    tp = _ints(device, "table", table, 2)
    n_seq, entries = table.shape
    pitch = table.stride()[0]
    if pitch < entries:
        if n_seq > 1:
            raise ValueError("the rows of table overlap")
        pitch = entries
    lp = _ints(device, "lens", lens, 1, n_seq)
    if cu is not None:
        cp = _ints(device, "cu", cu, 1, n_seq + 1)
    elif n_seq == 1:
        cp = 0
    else:
        raise ValueError("cu is needed for more than one sequence")
    if max_rows < 0:
        raise ValueError("max_rows is negative")
    return CACHE.pack(pages.data_ptr(), tp, lp, cp, step[0], shape[0], pitch, entries, n_seq, total, n_head_kv, head_dim, page_tokens, min(max_rows, total))


def kv4_page_bytes(n_head_kv, head_dim, page_tokens):
    """Bytes of a page of `page_tokens` tokens (32, 64, 128 or 256): 4.5 bits for each of K's and V's values, head_dim rounded up to 32."""
    if _lib is None:
        load()
    n = _lib.ctamd_kv4_page_bytes(n_head_kv, head_dim, page_tokens)
    if not n:
        raise ValueError("sizes not supported: head_dim is a multiple of 8 up to 256, page_tokens 32, 64, 128 or 256, n_head_kv 1 .. 1024")
    return n


def kv4_append(k, v, pages, table, lens, cu, max_rows, *, page_tokens):
    """Quantizes the rows k, v [total, n_head_kv, head_dim] (any strides) into the pages; row i of a sequence with n of them goes to position lens - n + i.

    A group of 32 dims of a token becomes f16(d) * (code - 8), code 0 .. 15, d = the value of largest magnitude / -8 (the rounding of Q4_0 weights); values beyond
    +-65504 are stored as that.  A token whose K or V of a head holds a NaN makes every row that sees it NaN.  No two sequences of a call may write one page."""
    device = _device_of("pages", pages)
    kr = _rows(device, "k", k)
    total, n_head_kv, head_dim = k.shape
    vr = _rows(device, "v", v, k.shape)
    c = _cache(device, pages, table, lens, cu, total, n_head_kv, head_dim, page_tokens, max_rows)
    _launch(device, lambda stream: _lib.ctamd_kv4_append(c, kr, vr, stream))


def kv4_read(pages, table, lens, cu, max_rows, total, *, n_head_kv, head_dim, page_tokens, dtype=torch.float16):
    """The last rows of every sequence as (k, v) [total, n_head_kv, head_dim]; 0 where there is no page or no position.  Rows of no sequence are undefined."""
    if dtype not in _TYPES:
        raise TypeError("dtype is float16, bfloat16 or float32")
    device = _device_of("pages", pages)
    c = _cache(device, pages, table, lens, cu, total, n_head_kv, head_dim, page_tokens, max_rows)
    both = torch.empty((2, total, n_head_kv, head_dim), dtype=dtype, device=pages.device)
    k, v = both.unbind(0)
    kr, vr = _rows(device, "k", k), _rows(device, "v", v)
    _launch(device, lambda stream: _lib.ctamd_kv4_read(c, kr, vr, stream))
    return k, v


def kv4_attention(q, pages, table, lens, cu, max_rows, *, n_head_kv, page_tokens, scale=None, out=None):
    """Causal attention of the rows q [total, n_head, head_dim] over the cache: row i of a sequence with n rows sees the positions 0 .. lens - n + i, query head h
    reads KV head h // (n_head / n_head_kv), scores are q.k * scale (finite; default 1 / sqrt(head_dim)).  A row that sees nothing becomes 0.  q is float16, bfloat16 or
    float32; the result has q's type, or is written into `out` [total, n_head, head_dim] of any of the three, where rows that belong to no sequence are left as they
    are; `out` may be q itself, but shares no memory with any other tensor of the call, nor any two of its own elements.  Products are taken in float16 (K's codes and V's values; q scaled by a power of two per row, so that
    float32 queries keep 11 bits; and p), everything else in float32.  The same call gives the same bits; a row's last bits may depend on the other rows of the call."""
    device = _device_of("pages", pages)
    qr = _rows(device, "q", q)
    total, n_head, head_dim = q.shape
    if n_head_kv < 1 or n_head < 1 or n_head % n_head_kv:
        raise ValueError("%d query heads over %d KV heads" % (n_head, n_head_kv))
    if q.stride()[2] != 1 and head_dim > 1:
        q = q.contiguous()
        qr = _rows(device, "q", q)
    c = _cache(device, pages, table, lens, cu, total, n_head_kv, head_dim, page_tokens, max_rows)
    if out is None:
        out = torch.empty((total, n_head, head_dim), dtype=q.dtype, device=q.device)
    orow = _rows(device, "out", out, q.shape)
    n = _lib.ctamd_kv4_attention_ws(c, n_head)
    if n:
        ws = torch.empty(n, dtype=torch.float32, device=q.device)
        at = ws.data_ptr()
    else:
        at = None
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    _launch(device, lambda stream: _lib.ctamd_kv4_attention(c, n_head, qr, orow, scale, at, n, stream))
    return out


def _tables(device, table, lens, refs, page_tokens, rows=None, extra=0):
    """(the packed structure, outputs, the extra ints, their address, what has to outlive the call)"""
    tp = _ints(device, "table", table, 2)
    n_seq, width = table.shape
    rp = _ints(device, "refs", refs, 1)
    lp = _ints(device, "lens", lens, 1, n_seq) if lens is not None else 0
    if page_tokens < 1:
        raise ValueError("page_tokens is positive")
    if n_seq > 1 and table.stride()[0] != width:
        table = table.contiguous()
        tp = table.data_ptr()
    if rows is None:
        rows = n_seq
    # the results are parts of one allocation, behind them `extra` ints (a status word and a workspace)
    n_pages, cells = refs.shape[0], rows * width
    both = torch.empty(cells + rows + n_pages + extra, dtype=_INT, device=refs.device)
    t, n, r, more = both.split((cells, rows, n_pages, extra))
    at = both.data_ptr()
    ends = at + 4 * cells, at + 4 * (cells + rows), at + 4 * (cells + rows + n_pages)
    return TABLES.pack(tp, lp, rp, at, ends[0] if lens is not None else 0, ends[1], n_seq, width, n_pages, page_tokens), (t.view(rows, width), n, r), more, ends[2], table


def _pool(device, pages, refs):
    """(address, layers, bytes from layer to layer, bytes of a page)"""
    if not isinstance(pages, torch.Tensor) or pages.get_device() != device:
        raise ValueError("pages is a tensor on the device of the tables")
    shape, step, e = pages.shape, pages.stride(), pages.element_size()
    if len(shape) not in (2, 3) or shape[-2] != refs.shape[0]:
        raise ValueError("pages has shape %s: [n_pages, page] or [layers, n_pages, page] with %d pages" % (tuple(shape), refs.shape[0]))
    if step[-1] != 1 or step[-2] != shape[-1]:
        raise ValueError("the pages of a layer are not adjacent")
    return (pages.data_ptr(), shape[0], step[0] * e, shape[2] * e) if len(shape) == 3 else (pages.data_ptr(), 1, shape[0] * shape[1] * e, shape[1] * e)


def kv_fork(table, lens, refs, parents, *, page_tokens, keep=None):
    """(table, lens, refs) of a batch whose sequence i continues sequence parents[i], sharing its pages: the batch may grow, shrink, permute and repeat, a parent
    outside [0, n_seq) makes an empty sequence (-1: freed).  keep (int32, one per new sequence): only its first keep[i] tokens — to take drafted tokens back, for one.
    A page whose last reference goes is free.  table [n_seq, width], refs [n_pages]."""
    device = _device_of("table", table)
    at = _ints(device, "parents", parents, 1)
    n_new = parents.shape[0]
    kept = _ints(device, "keep", keep, 1, n_new) if keep is not None else None
    t, new, _, _, alive = _tables(device, table, lens, refs, page_tokens, n_new)
    _launch(device, lambda stream: _lib.ctamd_kv_fork(t, at, kept, n_new, stream))
    return new


def kv_reserve(pages, table, lens, refs, add, *, page_tokens):
    """(table, lens, refs, short) with room for add[i] more tokens in sequence i: lens grows by it, pages are taken lowest free first in the order of the sequences,
    and a last page that others share is copied before its sequence writes it.  pages: [n_pages, page] or [layers, n_pages, page], any type.  short (int32, on the
    device): 0, or the pages that were missing, or -1 where a sequence outgrows its row of the table, or 2^31 - 1 tokens; then nothing has changed."""
    device = _device_of("table", table)
    _ints(device, "refs", refs, 1)
    n_seq = table.shape[0]
    t, new, rest, sp, alive = _tables(device, table, lens, refs, page_tokens, None, 1 + _lib.ctamd_kv_reserve_ws(n_seq, refs.shape[0]))
    more = _ints(device, "add", add, 1, n_seq)
    at, layers, layer_bytes, page_bytes = _pool(device, pages, refs)
    _launch(device, lambda stream: _lib.ctamd_kv_reserve(t, more, at, layers, layer_bytes, page_bytes, sp, sp + 4, stream))
    return new + (rest[0],)


def kv_compact(pages, table, refs):
    """(table, refs, used) after the pages in use have become pages 0 .. used - 1: those beyond move, in order, into the holes below.  used: int32, on the device."""
    device = _device_of("table", table)
    _ints(device, "refs", refs, 1)
    t, new, rest, up, alive = _tables(device, table, None, refs, 1, None, 1 + _lib.ctamd_kv_compact_ws(refs.shape[0]))
    at, layers, layer_bytes, page_bytes = _pool(device, pages, refs)
    _launch(device, lambda stream: _lib.ctamd_kv_compact(t, at, layers, layer_bytes, page_bytes, up, up + 4, stream))
    return new[0], new[2], rest[0]

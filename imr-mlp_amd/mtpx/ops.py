"""Operators on device tensors (the last section of include/mtpx.h) for torch
tensors: rotary positions with several axes, differential attention over
ragged batches and over a cache, the norms around a block with its gate
and residual scale, norms of queries and keys with the rotation in the same
pass, and a cache in pages: rows appended to it, and differential attention
of a chunk of new rows over it.

Every function takes the Context first, queues its kernels on torch's current
stream of the tensors' device and returns without waiting; workspaces and
results come from torch's allocator, so a call can be captured into a graph.
Functions with gradients come twice: as a pair (f, f_backward) on plain
tensors, and as an autograd function (RotaryFn, DiffAttentionFn, NormBlockFn, HeadNormRotaryFn).
Gradients are first derivatives: differentiating one of them again (a loss of
forces that were taken through a block) raises.  A backward pass can be recorded
into a graph if no earlier graph of the same leaves lives that was made on the
default stream; the autograd functions raise where one does and the leaf is an
argument of theirs (a leaf behind other operations is torch's matter).
Tensors are float32, bfloat16 or float16; their last dimension has to be
contiguous, other strides are free.  There is no fallback: a missing library
or a refused argument raises.  torch and the library share one HIP runtime if
this module or torch is imported before the library is first used; the other
order is refused.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
import sys

import numpy as np

from . import capi
from .capi import MtpxError  # noqa: F401 -- what the calls raise

if capi._lib is not None and "torch" not in sys.modules:
    # the library has brought its own HIP runtime, and a process's second one
    # finds no device
    raise ImportError("import torch or mtpx.ops before the first call of mtpx.capi: "
                      "the library then uses torch's HIP runtime")

import torch  # noqa: E402

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
POSITION_DTYPES = {torch.float32: 0, torch.float64: 3, torch.int32: 4, torch.int64: 5}
NORMS = {"rms": 0, "layer": 1}
APPEND_NORMS = {"rms": 0, "layer": 1, "none": 2}
GATES = {"none": 0, "sigmoid": 1, "tanh": 2}

_p, _i, _l, _f = C.c_void_p, C.c_int, C.c_int64, C.c_float


class Rows(C.Structure):
    """mtpx_rows."""
    _fields_ = [("data", _p), ("row", _l), ("head", _l), ("map", _l)]


class RotaryRequest(C.Structure):
    """mtpx_rotary_request."""
    _fields_ = [("stream", _p), ("dtype", _i), ("rows", _l), ("heads", _i), ("dim", _i),
                ("rotated", _i), ("interleaved", _i), ("inverse", _i), ("x", Rows), ("y", Rows),
                ("positions", _p), ("position_dtype", _i), ("position_row", _l),
                ("position_axis", _l), ("axes", _i), ("freq", _p), ("axis", _p),
                ("forward", Rows), ("dpositions", _p)]


class AttentionRequest(C.Structure):
    """mtpx_diff_attention_request."""
    _fields_ = [("stream", _p), ("dtype", _i), ("sequences", _p), ("heads", _i),
                ("kv_heads", _i), ("dim", _i), ("causal", _i), ("scale", _f), ("q", Rows),
                ("k", Rows), ("v", Rows), ("key_mask", _p), ("lambda_", _p), ("out", Rows),
                ("out1", _p), ("lse", _p), ("dout", Rows), ("dq", Rows), ("dk", Rows),
                ("dv", Rows), ("dlambda", _p), ("workspace", _p), ("workspace_bytes", C.c_size_t)]


class CacheRequest(C.Structure):
    """mtpx_diff_attention_cache_request."""
    _fields_ = [("stream", _p), ("dtype", _i), ("sequences", _i), ("heads", _i),
                ("kv_heads", _i), ("dim", _i), ("capacity", _l), ("scale", _f), ("q", Rows),
                ("k", Rows), ("v", Rows), ("k_sequence", _l), ("v_sequence", _l),
                ("lengths", _p), ("lambda_", _p), ("out", Rows), ("workspace", _p),
                ("workspace_bytes", C.c_size_t)]


class NormRequest(C.Structure):
    """mtpx_norm_block_request."""
    _fields_ = [("stream", _p), ("dtype", _i), ("rows", _l), ("width", _i), ("kind", _i),
                ("gate_act", _i), ("residual_scale", _f), ("block_scale", _f), ("eps", _f),
                ("x", _p), ("y", _p), ("gate", _p), ("post_weight", _p), ("pre_weight", _p),
                ("x_row", _l), ("y_row", _l), ("gate_row", _l), ("s", _p), ("n", _p),
                ("s_row", _l), ("n_row", _l), ("stats", _p), ("ds", _p), ("dn", _p),
                ("ds_row", _l), ("dn_row", _l), ("dx", _p), ("dy", _p), ("dgate", _p),
                ("dpost_weight", _p), ("dpre_weight", _p), ("dx_row", _l), ("dy_row", _l),
                ("dgate_row", _l), ("workspace", _p), ("workspace_bytes", C.c_size_t)]


class HeadNormRequest(C.Structure):
    """mtpx_head_norm_rotary_request."""
    _fields_ = [("stream", _p), ("dtype", _i), ("rows", _l), ("heads", _i), ("kv_heads", _i),
                ("maps", _i), ("dim", _i), ("rotated", _i), ("kind", _i), ("interleaved", _i),
                ("eps", _f), ("q", Rows), ("k", Rows), ("q_out", Rows), ("k_out", Rows),
                ("q_weight", _p), ("k_weight", _p), ("positions", _p), ("position_dtype", _i),
                ("position_row", _l), ("position_axis", _l), ("axes", _i), ("freq", _p),
                ("axis", _p), ("dq_out", Rows), ("dk_out", Rows), ("dq", Rows), ("dk", Rows),
                ("dq_weight", _p), ("dk_weight", _p), ("dpositions", _p), ("workspace", _p),
                ("workspace_bytes", C.c_size_t)]


class Pages(C.Structure):
    """mtpx_pages."""
    _fields_ = [("k", Rows), ("v", Rows), ("k_page", _l), ("v_page", _l), ("pages", _l),
                ("page_rows", _i), ("table", _p), ("table_row", _l), ("table_width", _i)]


class AppendRequest(C.Structure):
    """mtpx_append_paged_request."""
    _fields_ = [("stream", _p), ("dtype", _i), ("rows", _l), ("sequences", _i), ("heads", _i),
                ("kv_heads", _i), ("dim", _i), ("rotated", _i), ("kind", _i), ("interleaved", _i),
                ("eps", _f), ("q", Rows), ("k", Rows), ("v", Rows), ("q_out", Rows),
                ("q_weight", _p), ("k_weight", _p), ("positions", _p), ("position_dtype", _i),
                ("position_row", _l), ("position_axis", _l), ("axes", _i), ("freq", _p),
                ("axis", _p), ("cache", Pages), ("offsets", _p), ("lengths", _p)]


class PagedRequest(C.Structure):
    """mtpx_diff_attention_paged_request."""
    _fields_ = [("stream", _p), ("dtype", _i), ("rows", _l), ("sequences", _i), ("max_rows", _i),
                ("heads", _i), ("kv_heads", _i), ("dim", _i), ("causal", _i), ("scale", _f),
                ("q", Rows), ("cache", Pages), ("offsets", _p), ("lengths", _p), ("lambda_", _p),
                ("out", Rows), ("workspace", _p), ("workspace_bytes", C.c_size_t)]


def _packer(cls):
    """The C layout of a request as one flat list of its fields: packing it
    takes a third of the time that filling the ctypes structure does, which
    counts in calls of a few microseconds."""
    codes = {_p: "P", _i: "i", _l: "q", _f: "f", C.c_size_t: "N"}
    # (the pages' structure ends with an int, padded to its strictest alignment)
    codes[Rows], codes[Pages] = "Pqqq", "PqqqPqqqqqqiPqi0q"
    fmt = "".join(codes[f] for _, f in cls._fields_)
    # (a structure's size is a multiple of its strictest alignment)
    s = struct.Struct("@" + fmt + "0P")
    assert s.size == C.sizeof(cls)
    return s.pack


_pack_rotary, _pack_attention, _pack_cache, _pack_norm, _pack_heads, _pack_append, _pack_paged = (
    _packer(c) for c in (RotaryRequest, AttentionRequest, CacheRequest, NormRequest,
                         HeadNormRequest, AppendRequest, PagedRequest))

_lib = None


def _ops():
    """The library with the operators' signatures."""
    global _lib
    if _lib is None:
        L = capi.lib()
        ctx, size = C.c_void_p, C.POINTER(C.c_size_t)
        L.mtpx_rotary.argtypes = [ctx, _p]
        L.mtpx_sequences_create.argtypes = [ctx, _i, C.POINTER(_l), C.POINTER(_l), C.POINTER(_p)]
        L.mtpx_sequences_destroy.argtypes = [_p]
        L.mtpx_sequences_destroy.restype = None
        for name, req in (("diff_attention", C.POINTER(AttentionRequest)),
                          ("diff_attention_cache", _p), ("norm_block", _p),
                          ("head_norm_rotary", _p), ("diff_attention_paged", _p)):
            getattr(L, "mtpx_" + name).argtypes = [ctx, req]
            getattr(L, "mtpx_%s_workspace" % name).argtypes = [ctx, req, size]
        L.mtpx_diff_attention_backward.argtypes = [ctx, C.POINTER(AttentionRequest)]
        L.mtpx_norm_block_backward.argtypes = [ctx, _p]
        L.mtpx_head_norm_rotary_backward.argtypes = [ctx, _p]
        L.mtpx_append_paged.argtypes = [ctx, _p]
        _lib = L
    return _lib


_native = None


def _calls():
    """Norms of heads and the serving calls as native steps (csrc/torch_calls.cpp).  They take a call
    that is plainly right, which is nearly all of them, and return None for any
    other: the checks here then say what is wrong with it, or take it if nothing
    is (a max_rows of numpy's type, say)."""
    global _native
    if _native is None:
        L = capi.lib()
        try:
            from . import _calls as native
        except ImportError as e:
            raise RuntimeError("mtpx/_calls.so does not fit this torch or is not built "
                               "(run imr-mlp_amd/build.py)") from e
        native.setup(*(C.cast(getattr(L, "mtpx_" + f), _p).value for f in
                       ("head_norm_rotary", "head_norm_rotary_backward", "head_norm_rotary_workspace",
                        "append_paged", "diff_attention_paged", "diff_attention_paged_workspace")))
        _native = native
    return _native


def _handle(ctx):
    return getattr(ctx.h, "value", None)


def _fail(what):
    raise MtpxError(capi.ERRORS_BY_NAME["MTPX_E_INVALID"], what)


def _tensor(ctx, t, name, shape=None, dtype=None):
    """Checks a device tensor (None in shape: any size) and returns it."""
    if not isinstance(t, torch.Tensor) or t.get_device() != ctx.device:
        _fail("%s is not a tensor on the context's device" % name)
    if dtype is not None and t.dtype is not dtype:
        _fail("%s is %s, not %s" % (name, t.dtype, dtype))
    if shape is not None and t.shape != shape:
        if t.dim() != len(shape) or any(w is not None and w != n for w, n in zip(shape, t.shape)):
            _fail("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    return t


def _strides(ctx, t, name, shape, dtype):
    """Strides of a tensor of this shape and type on the context's device whose
    last dimension is contiguous."""
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == ctx.device:
            s = t.stride()
            if s[-1] == 1 or shape[-1] <= 1:
                return s
    except AttributeError:
        pass
    _tensor(ctx, t, name, shape, dtype)  # says which
    _fail("the last dimension of %s is not contiguous" % name)


def _typed(ctx, t, name, dims):
    """The type code of a tensor of so many dimensions on the context's device."""
    if not isinstance(t, torch.Tensor) or t.get_device() != ctx.device:
        _fail("%s is not a tensor on the context's device" % name)
    code = DTYPES.get(t.dtype)
    if code is None:
        _fail("%s is %s, not float32, bfloat16 or float16" % (name, t.dtype))
    if t.dim() != dims:
        _fail("%s has %d dimensions, not %d" % (name, t.dim(), dims))
    return code


_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # (not there: no device either)


def _stream(ctx):
    return _stream_of(ctx.device)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _bytes(ctx, query, request, **sizes):
    """Workspace that a call of these sizes needs: asked for once per context."""
    key = (request, *sizes.values())
    size = ctx.workspaces.get(key)
    if size is None:
        n = C.c_size_t()
        ctx._check(query(ctx.h, C.byref(request(**sizes)), C.byref(n)), "workspace")
        size = n.value
        if len(ctx.workspaces) > 1000:  # (another thread may be reading them)
            ctx.workspaces.clear()
        ctx.workspaces[key] = size
    return size


def _workspace(ctx, size):
    return torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", ctx.device))


# ---- rotary positions ----------------------------------------------------------


def _rotary(ctx, x, positions, freq, axis, interleaved, inverse, out, forward, dpositions):
    dtype = _typed(ctx, x, "x", 3)
    shape = x.shape
    sx = _strides(ctx, x, "x", shape, x.dtype)
    rows, heads, dim = shape
    sp = _tensor(ctx, positions, "positions", (rows, None)).stride()
    ptype = POSITION_DTYPES.get(positions.dtype)
    if ptype is None:
        _fail("positions are %s, not float32, float64, int32 or int64" % positions.dtype)
    pairs = (freq.numel(),) if isinstance(freq, torch.Tensor) else (None,)
    _strides(ctx, freq, "freq", pairs, torch.float32)
    _strides(ctx, axis, "axis", pairs, torch.int32)
    if out is None:
        y, sy = x.new_empty(shape), (heads * dim, dim)
    else:
        y, sy = out, _strides(ctx, out, "out", shape, x.dtype)
    f, sf = None, (0, 0)
    if dpositions is not None:
        sf, f = _strides(ctx, forward, "x", shape, x.dtype), forward.data_ptr()
    req = _pack_rotary(
        _stream(ctx), dtype, rows, heads, dim, 2 * pairs[0], interleaved, inverse,
        x.data_ptr(), sx[0], sx[1], 0, y.data_ptr(), sy[0], sy[1], 0, positions.data_ptr(),
        ptype, sp[0], sp[1], positions.shape[1], freq.data_ptr(),
        axis.data_ptr(), f or 0, sf[0], sf[1], 0, 0 if dpositions is None else dpositions.data_ptr())
    ctx._check(_ops().mtpx_rotary(ctx.h, req), "rotary")
    return y


def rotary(ctx, x, positions, freq, axis, *, interleaved=False, inverse=False, out=None):
    """Turns the pairs of x [rows, heads, dim] by positions[row, axis[p]] *
    freq[p]: pair p is elements (p, p + R/2), or (2p, 2p + 1) with
    `interleaved`, R = 2 len(freq); elements from R on are copied.  positions
    [rows, axes] in float32, float64, int32 or int64; freq float32, axis
    int32.  out may be x."""
    return _rotary(ctx, x, positions, freq, axis, interleaved, inverse, out, None, None)


def rotary_backward(ctx, dy, positions, freq, axis, *, interleaved=False, x=None):
    """Gradient of x from that of the result: (dx, None), or (dx, dpositions)
    with the forward pass's x given (positions float32 or float64; a 32-bit sum
    for both)."""
    dpos = None
    if x is not None:
        dpos = torch.empty(positions.shape, dtype=positions.dtype, device=dy.device)
    dx = _rotary(ctx, dy, positions, freq, axis, interleaved, True, None, x, dpos)
    return dx, dpos


# ---- differential attention ------------------------------------------------------


class Sequences:
    """mtpx_sequences: the row ranges of a ragged batch.  q_offsets and
    k_offsets (default: the same) are n + 1 ascending row numbers on the
    host.  Creation allocates and waits for its upload: once per batch, not
    while a graph is recorded."""

    def __init__(self, ctx, q_offsets, k_offsets=None):
        self.h = None
        q = np.ascontiguousarray(q_offsets, np.int64)
        k = q if k_offsets is None else np.ascontiguousarray(k_offsets, np.int64)
        if q.ndim != 1 or q.size < 1 or q.shape != k.shape:
            _fail("offsets are n + 1 numbers")
        h = C.c_void_p()
        ptr = C.POINTER(_l)
        ctx._check(_ops().mtpx_sequences_create(ctx.h, q.size - 1, q.ctypes.data_as(ptr),
                                                k.ctypes.data_as(ptr), C.byref(h)), "sequences")
        self.h, self.q_rows, self.k_rows = h, int(q[-1]), int(k[-1])
        self._destroy = _ops().mtpx_sequences_destroy  # kept: this module's names may go first

    def close(self):
        """Ends the use of the handle; work that is queued keeps its tables, a
        recorded graph does not.  The next handle frees them, once the device
        has ended its work."""
        if getattr(self, "h", None):
            h, self.h = self.h, None
            self._destroy(h)

    def __del__(self):
        self.close()


_NO_ROWS = (0, 0, 0, 0)


def _attention(ctx, q, k, v, lam, seqs, causal, scale, key_mask, out=_NO_ROWS, out1=0, lse=0,
               dout=_NO_ROWS, dq=_NO_ROWS, dk=_NO_ROWS, dv=_NO_ROWS, dlam=0):
    """The checked request of either pass; results as (address, row, head and
    map stride) or addresses."""
    dtype, of = _typed(ctx, q, "q", 4), q.dtype
    rows, heads, _, dim = q.shape
    sq = _strides(ctx, q, "q", (rows, heads, 2, dim), of)
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        _fail("k is not [key rows, kv heads, 2, dim]")
    keys, kv, _, _ = k.shape
    sk = _strides(ctx, k, "k", (keys, kv, 2, dim), of)
    sv = _strides(ctx, v, "v", (keys, kv, 2 * dim), of)
    if seqs.h is None:
        _fail("the sequences are closed")
    if rows != seqs.q_rows or keys != seqs.k_rows:
        _fail("q and k have %d and %d rows, the sequences %d and %d" %
              (rows, keys, seqs.q_rows, seqs.k_rows))
    _strides(ctx, lam, "lam", (heads,), torch.float32)
    mask = 0
    if key_mask is not None:
        _tensor(ctx, key_mask, "key_mask", (keys,))
        if key_mask.dtype not in (torch.bool, torch.uint8) or not key_mask.is_contiguous():
            _fail("key_mask must be contiguous bool or uint8")
        mask = key_mask.data_ptr()
    return AttentionRequest.from_buffer_copy(_pack_attention(
        _stream(ctx), dtype, getattr(seqs.h, "value", seqs.h), heads, kv, dim, causal,
        dim ** -0.5 if scale is None else scale, q.data_ptr(), sq[0], sq[1], sq[2], k.data_ptr(),
        sk[0], sk[1], sk[2], v.data_ptr(), sv[0], sv[1], dim, mask, lam.data_ptr(), *out, out1,
        lse, *dout, *dq, *dk, *dv, dlam, 0, 0))


def diff_attention(ctx, q, k, v, lam, seqs, *, causal=False, scale=None, key_mask=None,
                   save=False, out=None):
    """(softmax(scale q0 k0^T) - lam softmax(scale q1 k1^T)) v per sequence and
    head: q [rows, heads, 2, dim], k [key rows, kv heads, 2, dim], v [key
    rows, kv heads, 2 dim], lam [heads] float32; scale defaults to dim^-1/2.
    Returns out [rows, heads, 2 dim], with save (out, saved) for
    diff_attention_backward."""
    _typed(ctx, q, "q", 4)
    rows, heads, _, dim = q.shape
    shape = (rows, heads, 2 * dim)
    if out is None:
        out, so = q.new_empty(shape), (heads * 2 * dim, 2 * dim)
    else:
        so = _strides(ctx, out, "out", shape, q.dtype)
    saved = None
    if save:
        saved = q.new_empty(shape), q.new_empty((2, heads, rows), dtype=torch.float32)
    req = _attention(ctx, q, k, v, lam, seqs, causal, scale, key_mask,
                     (out.data_ptr(), so[0], so[1], dim), *(s.data_ptr() for s in saved or ()))
    ctx._check(_ops().mtpx_diff_attention(ctx.h, req), "diff_attention")
    return (out, saved) if save else out


def diff_attention_backward(ctx, dout, q, k, v, lam, seqs, out, saved, *, causal=False,
                            scale=None, key_mask=None):
    """(dq, dk, dv, dlam) from the gradient of out and what the forward call
    returned and saved."""
    _typed(ctx, q, "q", 4)
    rows, heads, _, dim = q.shape
    shape, of = (rows, heads, 2 * dim), q.dtype
    sd = _strides(ctx, dout, "dout", shape, of)
    so = _strides(ctx, out, "out", shape, of)
    out1, lse = saved
    for t, name, s, kind in ((out1, "saved[0]", shape, of),
                             (lse, "saved[1]", (2, heads, rows), torch.float32)):
        _strides(ctx, t, name, s, kind)
        if not t.is_contiguous():
            _fail("%s must be contiguous" % name)
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    dlam = q.new_empty(heads, dtype=torch.float32)
    kv = k.shape[1]
    req = _attention(
        ctx, q, k, v, lam, seqs, causal, scale, key_mask, (out.data_ptr(), so[0], so[1], dim),
        out1.data_ptr(), lse.data_ptr(), (dout.data_ptr(), sd[0], sd[1], dim),
        (dq.data_ptr(), heads * 2 * dim, 2 * dim, dim), (dk.data_ptr(), kv * 2 * dim, 2 * dim, dim),
        (dv.data_ptr(), kv * 2 * dim, 2 * dim, dim), dlam.data_ptr())
    n = C.c_size_t()
    ctx._check(_ops().mtpx_diff_attention_workspace(ctx.h, req, C.byref(n)), "workspace")
    req.workspace_bytes = n.value
    w = _workspace(ctx, n.value)  # held until the kernels are queued
    req.workspace = w.data_ptr()
    ctx._check(_ops().mtpx_diff_attention_backward(ctx.h, req), "diff_attention_backward")
    return dq, dk, dv, dlam


def diff_attention_cache(ctx, q, k, v, lam, lengths, *, scale=None, out=None):
    """One row per sequence against a cache: q [sequences, heads, 2, dim],
    k [sequences, capacity, kv heads, 2, dim], v [sequences, capacity, kv
    heads, 2 dim], lengths [sequences] int32 on the device.  Returns
    [sequences, heads, 2 dim]."""
    dtype = _typed(ctx, q, "q", 4)
    of = q.dtype
    n, heads, _, dim = q.shape
    sq = _strides(ctx, q, "q", (n, heads, 2, dim), of)
    if not isinstance(k, torch.Tensor) or k.dim() != 5:
        _fail("k is not [sequences, capacity, kv heads, 2, dim]")
    _, cap, kv, _, _ = k.shape
    sk = _strides(ctx, k, "k", (n, cap, kv, 2, dim), of)
    sv = _strides(ctx, v, "v", (n, cap, kv, 2 * dim), of)
    _strides(ctx, lengths, "lengths", (n,), torch.int32)
    _strides(ctx, lam, "lam", (heads,), torch.float32)
    shape = (n, heads, 2 * dim)
    if out is None:
        out, so = q.new_empty(shape), (heads * 2 * dim, 2 * dim)
    else:
        so = _strides(ctx, out, "out", shape, of)
    size = _bytes(ctx, _ops().mtpx_diff_attention_cache_workspace, CacheRequest, dtype=dtype,
                  sequences=n, heads=heads, kv_heads=kv, dim=dim, capacity=cap)
    w = _workspace(ctx, size) if size else None  # held until the kernels are queued
    req = _pack_cache(
        _stream(ctx), dtype, n, heads, kv, dim, cap, dim ** -0.5 if scale is None else scale,
        q.data_ptr(), sq[0], sq[1], sq[2], k.data_ptr(), sk[1], sk[2], sk[3], v.data_ptr(), sv[1],
        sv[2], dim, sk[0], sv[0], lengths.data_ptr(), lam.data_ptr(), out.data_ptr(), so[0], so[1],
        dim, _ptr(w), size)
    ctx._check(_ops().mtpx_diff_attention_cache(ctx.h, req), "diff_attention_cache")
    return out


# ---- norms around a block ----------------------------------------------------------


def _norm(ctx, x, y, gate, post_weight, pre_weight, kind, gate_act, residual_scale, block_scale,
          eps, s, n, stats, ds=None, dn=None, dx=None, dy=None, dgate=None, dpost=None, dpre=None,
          work=None, work_bytes=0):
    """The checked and packed request of either pass; results are contiguous."""
    dtype, of = _typed(ctx, y, "y", 2), y.dtype
    shape = y.shape
    rows, width = shape
    sy = _strides(ctx, y, "y", shape, of)
    if kind not in NORMS or gate_act not in GATES:
        _fail("kind is one of %s, gate_act of %s" % (tuple(NORMS), tuple(GATES)))
    sx = (0,) if x is None else _strides(ctx, x, "x", shape, of)
    gate_row = 0
    if gate is not None:
        one = gate.dim() == 1
        sg = _strides(ctx, gate, "gate", (width,) if one else shape, of)
        if not one:
            gate_row = sg[0]
            if gate_row == 0:
                if rows > 1:
                    _fail("a gate shared by all rows is [width]")
                gate_row = width  # one row's stride is any
    if post_weight is not None:
        _strides(ctx, post_weight, "post_weight", (width,), of)
    if pre_weight is not None:
        _strides(ctx, pre_weight, "pre_weight", (width,), of)
    sds = (0,) if ds is None else _strides(ctx, ds, "ds", shape, of)
    sdn = (0,) if dn is None else _strides(ctx, dn, "dn", shape, of)
    return _pack_norm(
        _stream(ctx), dtype, rows, width, NORMS[kind], GATES[gate_act], residual_scale, block_scale,
        eps, _ptr(x), y.data_ptr(), _ptr(gate), _ptr(post_weight), _ptr(pre_weight), sx[0], sy[0],
        gate_row, _ptr(s), _ptr(n), width, width, _ptr(stats), _ptr(ds), _ptr(dn), sds[0], sdn[0],
        _ptr(dx), _ptr(dy), _ptr(dgate), _ptr(dpost), _ptr(dpre), width, width,
        width if gate_row else 0, _ptr(work), work_bytes)


def norm_block(ctx, x, y, gate=None, post_weight=None, pre_weight=None, *, kind="rms",
               gate_act="none", residual_scale=1.0, block_scale=1.0, eps=1e-6, save=False,
               next_norm=True):
    """s = residual_scale x + block_scale act(gate) (norm(y) post_weight) and
    n = norm(s) pre_weight, for the block output y and the residual x [rows,
    width] (x None: no residual; gate [rows, width], [width] or None; weights
    [width] or None).  Returns (s, n), with save (s, n, stats); without
    next_norm n is None."""
    if not isinstance(y, torch.Tensor):
        _fail("y is not a tensor")
    s = y.new_empty(y.shape)
    n = y.new_empty(y.shape) if next_norm else None
    stats = y.new_empty((len(y), 4), dtype=torch.float32) if save else None
    req = _norm(ctx, x, y, gate, post_weight, pre_weight, kind, gate_act, residual_scale,
                block_scale, eps, s, n, stats)
    ctx._check(_ops().mtpx_norm_block(ctx.h, req), "norm_block")
    return (s, n, stats) if save else (s, n)


def norm_block_backward(ctx, ds, dn, x, y, gate, post_weight, pre_weight, stats, *, kind="rms",
                        gate_act="none", residual_scale=1.0, block_scale=1.0, eps=1e-6):
    """(dx, dy, dgate, dpost_weight, dpre_weight) from the gradients of s and n
    (either may be None) and the forward pass's inputs and stats; None in the
    place of an input that was not given."""
    dtype = _typed(ctx, y, "y", 2)
    rows, width = y.shape
    _tensor(ctx, stats, "stats", (rows, 4), torch.float32)
    if not stats.is_contiguous():
        _fail("stats must be contiguous")

    def like(t):
        return None if t is None else t.new_empty(t.shape)

    dx, dy, dgate, dpost, dpre = like(x), like(y), like(gate), like(post_weight), like(pre_weight)
    size = _bytes(ctx, _ops().mtpx_norm_block_workspace, NormRequest, dtype=dtype, rows=rows,
                  width=width)
    w = _workspace(ctx, size)  # held until the kernels are queued
    req = _norm(ctx, x, y, gate, post_weight, pre_weight, kind, gate_act, residual_scale,
                block_scale, eps, None, None, stats, ds, dn, dx, dy, dgate, dpost, dpre, w, size)
    ctx._check(_ops().mtpx_norm_block_backward(ctx.h, req), "norm_block_backward")
    return dx, dy, dgate, dpost, dpre


# ---- norms of queries and keys, with their rotation ---------------------------------


def _turns(ctx, positions, freq, axis, rows):
    """The checked fields of a rotation, as a request has them, and how many
    elements of a head it turns."""
    shape = _tensor(ctx, positions, "positions", (rows, None)).shape
    sp = positions.stride()
    ptype = POSITION_DTYPES.get(positions.dtype)
    if ptype is None:
        _fail("positions are %s, not float32, float64, int32 or int64" % positions.dtype)
    pairs = (freq.numel(),) if isinstance(freq, torch.Tensor) else (0,)
    _strides(ctx, freq, "freq", pairs, torch.float32)
    _strides(ctx, axis, "axis", pairs, torch.int32)
    return 2 * pairs[0], (positions.data_ptr(), ptype, sp[0], sp[1], shape[1],
                          freq.data_ptr(), axis.data_ptr())


def _head_rows(ctx, t, name, shape, of):
    """Heads [rows, heads, dim] or [rows, heads, maps, dim] as a request has them."""
    s = _strides(ctx, t, name, shape, of)
    return (t.data_ptr(), s[0], s[1], s[2]) if len(s) == 4 else (t.data_ptr(), s[0], s[1], 0)


def _like(t):
    """An unwritten contiguous tensor of the same shape."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _whole(t, heads, maps, dim):
    """The same of a contiguous result."""
    return t.data_ptr(), heads * maps * dim, maps * dim, dim


def _heads_of(ctx, q, k):
    """Checks what q and k share: the type's code, rows, heads, kv heads, maps and
    dim, and k's shape."""
    dims = 4 if isinstance(q, torch.Tensor) and q.dim() == 4 else 3
    dtype, shape = _typed(ctx, q, "q", dims), q.shape
    if dims == 4:
        rows, heads, maps, dim = shape
        if maps not in (1, 2):
            _fail("q has %d maps, not 1 or 2" % maps)
    else:
        (rows, heads, dim), maps = shape, 1
    if k is None:
        return dtype, rows, heads, 0, maps, dim, None
    if not isinstance(k, torch.Tensor) or k.dim() != dims:
        _fail("k has not as many dimensions as q")
    kv = k.shape[1]
    if kv == 0:
        _fail("k has no heads")
    return dtype, rows, heads, kv, maps, dim, (rows, kv, maps, dim) if dims == 4 else (rows, kv, dim)


def _weight(ctx, w, name, dim, of):
    if w is None:
        return 0
    _strides(ctx, w, name, (dim,), of)
    return w.data_ptr()


def head_norm_rotary(ctx, q, k, q_weight, k_weight, positions, freq, axis, *, kind="rms",
                     eps=1e-6, interleaved=False):
    """Norms of queries and keys for each head, and their rotation: of q [rows,
    heads, dim] or [rows, heads, maps, dim] and k (the same with its own heads;
    None: q only) every head and map becomes norm(x) weight, turned as by
    rotary; weights [dim] or None, positions, freq and axis as there.  Returns
    (q, k)."""
    done = _calls().head_norm_rotary(_handle(ctx), ctx.device, _stream_of, q, k, q_weight, k_weight,
                                     positions, freq, axis, NORMS.get(kind), eps, interleaved)
    if done is not None:
        if type(done) is int:
            ctx._check(done, "head_norm_rotary")
        return done
    dtype, rows, heads, kv, maps, dim, k_shape = _heads_of(ctx, q, k)
    shape, of = q.shape, q.dtype
    if kind not in NORMS:
        _fail("kind is one of %s" % (tuple(NORMS),))
    rotated, turn = _turns(ctx, positions, freq, axis, rows)
    q_in, qo = _head_rows(ctx, q, "q", shape, of), _like(q)
    ko, k_in, k_out = None, _NO_ROWS, _NO_ROWS
    if k is not None:
        k_in, ko = _head_rows(ctx, k, "k", k_shape, of), _like(k)
        k_out = _whole(ko, kv, maps, dim)
    req = _pack_heads(
        _stream(ctx), dtype, rows, heads, kv, maps, dim, rotated, NORMS[kind], interleaved, eps,
        *q_in, *k_in, *_whole(qo, heads, maps, dim), *k_out,
        _weight(ctx, q_weight, "q_weight", dim, of), _weight(ctx, k_weight, "k_weight", dim, of),
        *turn, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, 0, 0, 0, 0, 0)
    ctx._check(_ops().mtpx_head_norm_rotary(ctx.h, req), "head_norm_rotary")
    return qo, ko


def head_norm_rotary_backward(ctx, dq, dk, q, k, q_weight, k_weight, positions, freq, axis, *,
                              kind="rms", eps=1e-6, interleaved=False, dpositions=False):
    """(dq, dk, dq_weight, dk_weight, dpositions) from the gradients of the
    results and the forward pass's inputs; None in the place of an input that
    was not given, and of the positions' without dpositions (which needs
    float32 or float64 ones; a 32-bit sum for both)."""
    done = _calls().head_norm_rotary_backward(
        _handle(ctx), ctx.device, _stream_of, dq, dk, q, k, q_weight, k_weight, positions, freq, axis,
        NORMS.get(kind), eps, interleaved, dpositions)
    if done is not None:
        if type(done) is int:
            ctx._check(done, "head_norm_rotary_backward")
        return done
    dtype, rows, heads, kv, maps, dim, k_shape = _heads_of(ctx, q, k)
    shape, of = q.shape, q.dtype
    if kind not in NORMS:
        _fail("kind is one of %s" % (tuple(NORMS),))
    rotated, turn = _turns(ctx, positions, freq, axis, rows)
    if (dk is None) != (k is None):
        _fail("dk is given with k")
    gq, gk, dpos = _like(q), None, None
    k_in, k_grad, k_out = _NO_ROWS, _NO_ROWS, _NO_ROWS
    if k is not None:
        gk = _like(k)
        k_in, k_grad = _head_rows(ctx, k, "k", k_shape, of), _head_rows(ctx, dk, "dk", k_shape, of)
        k_out = _whole(gk, kv, maps, dim)
    wq, wk = _weight(ctx, q_weight, "q_weight", dim, of), _weight(ctx, k_weight, "k_weight", dim, of)
    dwq = None if q_weight is None else q.new_empty(dim)
    dwk = None if k_weight is None else q.new_empty(dim)
    if dpositions:
        dpos = torch.empty(positions.shape, dtype=positions.dtype, device=q.device)
    size = _bytes(ctx, _ops().mtpx_head_norm_rotary_workspace, HeadNormRequest, rows=rows, dim=dim)
    w = q.new_empty(size, dtype=torch.uint8)  # held until the kernels are queued
    req = _pack_heads(
        _stream(ctx), dtype, rows, heads, kv, maps, dim, rotated, NORMS[kind], interleaved, eps,
        *_head_rows(ctx, q, "q", shape, of), *k_in, *_NO_ROWS, *_NO_ROWS, wq, wk, *turn,
        *_head_rows(ctx, dq, "dq", shape, of), *k_grad, *_whole(gq, heads, maps, dim), *k_out,
        _ptr(dwq), _ptr(dwk), _ptr(dpos), w.data_ptr(), size)
    ctx._check(_ops().mtpx_head_norm_rotary_backward(ctx.h, req), "head_norm_rotary_backward")
    return gq, gk, dwq, dwk, dpos


# ---- a cache in pages ------------------------------------------------------------------


def _pages(ctx, k_pages, v_pages, table, offsets, lengths, kv, dim, of):
    """The checked fields of a cache and its batch: (mtpx_pages, offsets, lengths, sequences)."""
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 5:
        _fail("k_pages is not [pages, page rows, kv heads, 2, dim]")
    n, page, *_ = k_pages.shape
    sk = _strides(ctx, k_pages, "k_pages", (n, page, kv, 2, dim), of)
    sv = _strides(ctx, v_pages, "v_pages", (n, page, kv, 2 * dim), of)
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        _fail("lengths are not [sequences]")
    seqs = lengths.shape[0]
    _strides(ctx, lengths, "lengths", (seqs,), torch.int32)
    _strides(ctx, offsets, "offsets", (seqs + 1,), torch.int32)
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        _fail("table is not [sequences, pages of a sequence]")
    width = table.shape[1]
    st = _strides(ctx, table, "table", (seqs, width), torch.int32)
    return (k_pages.data_ptr(), sk[1], sk[2], sk[3], v_pages.data_ptr(), sv[1], sv[2], dim, sk[0],
            sv[0], n, page, table.data_ptr(), st[0], width), offsets.data_ptr(), lengths.data_ptr(), seqs


def append_paged(ctx, k, v, k_pages, v_pages, table, offsets, lengths, positions, freq, axis, *,
                 q=None, kind="none", q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                 out=None):
    """Puts a batch's new rows into a cache: k [rows, kv heads, 2, dim], normed
    (kind "rms" or "layer", weights [dim] or None; "none": as it is) and turned
    by positions [rows, axes] as by head_norm_rotary, into k_pages [pages, page
    rows, kv heads, 2, dim], and v [rows, kv heads, 2 dim] into v_pages [pages,
    page rows, kv heads, 2 dim].  Sequence i has rows offsets[i] to offsets[i +
    1] - 1 and lengths[i] rows with them; its row t lies in page table[i, t //
    page rows].  offsets [sequences + 1], lengths [sequences] and table
    [sequences, width] are int32 on the device and are not read on the host.
    With q [rows, heads, 2, dim] its queries are normed and turned as well:
    returns them (in out, which may be q), else None.  Rows of no sequence are
    left as they are."""
    done = _calls().append_paged(_handle(ctx), ctx.device, _stream_of, k, v, k_pages, v_pages, table,
                                 offsets, lengths, positions, freq, axis, q, APPEND_NORMS.get(kind),
                                 q_weight, k_weight, eps, interleaved, out)
    if done is not None:
        if type(done) is int:
            ctx._check(done, "append_paged")
        return done if q is not None else None
    dtype = _typed(ctx, k, "k", 4)
    of = k.dtype
    rows, kv, _, dim = k.shape
    k_in = _head_rows(ctx, k, "k", (rows, kv, 2, dim), of)
    sv = _strides(ctx, v, "v", (rows, kv, 2 * dim), of)
    if kind not in APPEND_NORMS:
        _fail("kind is one of %s" % (tuple(APPEND_NORMS),))
    if kind == "none" and (q_weight is not None or k_weight is not None):
        _fail("weights without a norm")
    cache, off, length, seqs = _pages(ctx, k_pages, v_pages, table, offsets, lengths, kv, dim, of)
    rotated, turn = _turns(ctx, positions, freq, axis, rows)
    heads, q_in, q_out = 0, _NO_ROWS, _NO_ROWS
    if q is not None:
        _typed(ctx, q, "q", 4)
        heads = q.shape[1]
        shape = (rows, heads, 2, dim)
        q_in = _head_rows(ctx, q, "q", shape, of)
        if out is None:
            out = _like(q)
            q_out = _whole(out, heads, 2, dim)
        else:
            q_out = _head_rows(ctx, out, "out", shape, of)
    elif out is not None:
        _fail("out without q")
    req = _pack_append(
        _stream(ctx), dtype, rows, seqs, heads, kv, dim, rotated, APPEND_NORMS[kind], interleaved,
        eps, *q_in, *k_in, v.data_ptr(), sv[0], sv[1], dim, *q_out,
        _weight(ctx, q_weight, "q_weight", dim, of), _weight(ctx, k_weight, "k_weight", dim, of),
        *turn, *cache, off, length)
    ctx._check(_ops().mtpx_append_paged(ctx.h, req), "append_paged")
    return out


def _paged_sizes(page, width, **sizes):
    return PagedRequest(cache=Pages(page_rows=page, table_width=width), **sizes)


def diff_attention_paged(ctx, q, k_pages, v_pages, lam, table, offsets, lengths, *, causal=True,
                         scale=None, max_rows=None, out=None):
    """Differential attention of each sequence's new rows over its pages, where
    append_paged has put them already: q [rows, heads, 2, dim], the other
    arguments as there, lam [heads] float32.  Row j of m new ones sees the
    first lengths[i] - m + j + 1 rows of its sequence, without causal all of
    them.  max_rows: the most new rows of a sequence, where the caller knows it
    (1 in a plain decoding step), which saves work; rows of a sequence beyond it
    may be left unwritten.  Returns [rows, heads, 2 dim]; rows of no sequence are
    left as they are."""
    done = _calls().diff_attention_paged(_handle(ctx), ctx.device, _stream_of, q, k_pages, v_pages,
                                         lam, table, offsets, lengths, causal, scale, max_rows, out)
    if done is not None:
        if type(done) is int:
            ctx._check(done, "diff_attention_paged")
        return done
    dtype = _typed(ctx, q, "q", 4)
    of = q.dtype
    rows, heads, _, dim = q.shape
    sq = _strides(ctx, q, "q", (rows, heads, 2, dim), of)
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 5:
        _fail("k_pages is not [pages, page rows, kv heads, 2, dim]")
    kv = k_pages.shape[2]
    cache, off, length, seqs = _pages(ctx, k_pages, v_pages, table, offsets, lengths, kv, dim, of)
    _strides(ctx, lam, "lam", (heads,), torch.float32)
    if max_rows is None:
        max_rows = 0
    elif max_rows < 1:
        _fail("max_rows must be positive")
    else:
        max_rows = min(max_rows, max(rows, 1))
    shape = (rows, heads, 2 * dim)
    if out is None:
        out, so = q.new_empty(shape), (heads * 2 * dim, 2 * dim)
    else:
        so = _strides(ctx, out, "out", shape, of)
    key = (PagedRequest, dtype, rows, seqs, max_rows, heads, kv, dim, cache[11], cache[14])
    size = ctx.workspaces.get(key)
    if size is None:
        size = _bytes(ctx, _ops().mtpx_diff_attention_paged_workspace, _paged_sizes, dtype=dtype,
                      rows=rows, sequences=seqs, max_rows=max_rows, heads=heads, kv_heads=kv,
                      dim=dim, page=cache[11], width=cache[14])
        ctx.workspaces[key] = size
    w = q.new_empty(size, dtype=torch.uint8) if size else None  # held until the kernels are queued
    req = _pack_paged(
        _stream(ctx), dtype, rows, seqs, max_rows, heads, kv, dim, causal,
        dim ** -0.5 if scale is None else scale, q.data_ptr(), sq[0], sq[1], sq[2], *cache, off,
        length, lam.data_ptr(), out.data_ptr(), so[0], so[1], dim, _ptr(w), size)
    ctx._check(_ops().mtpx_diff_attention_paged(ctx.h, req), "diff_attention_paged")
    return out


# ---- autograd ------------------------------------------------------------------------


def _last_contiguous(t):
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


class _Refused(torch.autograd.Function):
    """Hands gradients on; refuses to be differentiated."""

    @staticmethod
    def forward(fn, grads, *inputs):
        fn.set_materialize_grads(False)
        return tuple(g.detach() for g in grads)

    @staticmethod
    def backward(fn, *unused):
        _fail("a second derivative of an operator on device tensors, which has first ones only")


def _learned(**values):
    """The names of arguments without a gradient that are asked for one:
    refused in the backward pass, as None in its place would say zero."""
    return [n for n, t in values.items() if isinstance(t, torch.Tensor) and t.requires_grad]


_STREAM = "mtpx.ops: stream"
_CREATED = 4096  # handles of created streams are addresses, those of the default ones (0, 1, 2) are not


def _recording():
    try:
        return torch.cuda.is_current_stream_capturing()
    except RuntimeError:  # no device
        return False


def _made_on(fn, node):
    """The stream that was current when an end of the graph at a leaf was made,
    on which autograd hands that leaf's gradient over."""
    try:
        at = _calls().stream_of(node)
    except RuntimeError:  # the native calls are not built: not known
        at = None
    if at is None:
        return _stream(fn.ctx)
    return torch.cuda.Stream(stream_id=at[0], device_index=at[1], device_type=at[2]).cuda_stream


def _mark_leaves(fn):
    """Notes at a graph's ends at its leaves on which stream they were made."""
    for node, _ in fn.next_functions:
        if type(node) is _Leaf and node.variable.is_cuda and _STREAM not in node.metadata:
            node.metadata[_STREAM] = _made_on(fn, node)


def _same_streams(fn):
    """Refuses a backward pass that is being recorded into a graph while another
    graph of the same leaves lives that was made on the default stream (an eager
    one, as a rule): autograd would hand the gradients over on that stream, which
    cannot be part of a recording, and ending it would end the process.  (Any other
    stream waits for the recording and is joined to it as the pass ends.)  A pass
    that is not recorded is asked nothing else: marks set by every forward pass
    took 0.9 to 1.6 us there, and 5 to 11 us of a pass with its gradients."""
    if not _recording():
        return
    _mark_leaves(fn)
    now = _stream(fn.ctx)
    for node, _ in fn.next_functions:
        made = node.metadata.get(_STREAM, now) if type(node) is _Leaf else now
        if made != now and made < _CREATED:
            _fail("a backward pass recorded while an earlier graph of the same leaves lives "
                  "that was made on the default stream: drop what still refers to that one first")


_Leaf = type(torch.zeros(1, requires_grad=True).expand(1).grad_fn.next_functions[0][0])


def _first_only(backward):
    """The kernels' gradients carry no graph.  Where autograd keeps one
    (create_graph), it would take them for constants, and a loss of them, as of
    forces, would lose its share of every other gradient without a word: they
    are tied to all that they depend on by a node that raises.  (torch's
    once_differentiable does so only if an incoming gradient has a graph.)"""
    @functools.wraps(backward)
    def once(fn, *grads):
        if fn.learned:
            _fail("%s requires a gradient and has none" % " and ".join(fn.learned))
        _same_streams(fn)
        with torch.no_grad():
            out = backward(fn, *grads)
        if not torch.is_grad_enabled():
            return out
        inputs = [t for t in (*grads, *fn.saved_tensors) if t is not None and t.requires_grad]
        if not inputs:
            return out
        tied = iter(_Refused.apply([t for t in out if t is not None], *inputs))
        return tuple(t if t is None else next(tied) for t in out)

    return once


class RotaryFn(torch.autograd.Function):
    """RotaryFn.apply(ctx, x, positions, freq, axis, interleaved): rotary with
    the gradients of x and of floating-point positions.  freq has none: one
    that requires it raises in the backward pass."""

    @staticmethod
    def forward(fn, ctx, x, positions, freq, axis, interleaved=False):
        fn.ctx, fn.interleaved, fn.learned = ctx, interleaved, _learned(freq=freq)
        keep = x if positions.requires_grad else None
        fn.save_for_backward(keep, positions, freq, axis)
        return rotary(ctx, x, positions, freq, axis, interleaved=interleaved)

    @staticmethod
    @_first_only
    def backward(fn, dy):
        x, positions, freq, axis = fn.saved_tensors
        dx, dpos = rotary_backward(fn.ctx, _last_contiguous(dy), positions, freq, axis,
                                   interleaved=fn.interleaved, x=x)
        return None, dx, dpos, None, None, None


class DiffAttentionFn(torch.autograd.Function):
    """DiffAttentionFn.apply(ctx, q, k, v, lam, seqs, causal, scale, key_mask),
    with the gradients of q, k, v and lam."""

    @staticmethod
    def forward(fn, ctx, q, k, v, lam, seqs, causal=False, scale=None, key_mask=None):
        out, saved = diff_attention(ctx, q, k, v, lam, seqs, causal=causal, scale=scale,
                                    key_mask=key_mask, save=True)
        fn.ctx, fn.seqs, fn.causal, fn.scale = ctx, seqs, causal, scale
        fn.learned = _learned(scale=scale)
        fn.save_for_backward(q, k, v, lam, out, *saved, key_mask)
        return out

    @staticmethod
    @_first_only
    def backward(fn, dout):
        q, k, v, lam, out, out1, lse, mask = fn.saved_tensors
        grads = diff_attention_backward(fn.ctx, _last_contiguous(dout), q, k, v, lam, fn.seqs,
                                        out, (out1, lse), causal=fn.causal, scale=fn.scale,
                                        key_mask=mask)
        return (None, *grads, None, None, None, None)


class NormBlockFn(torch.autograd.Function):
    """NormBlockFn.apply(ctx, x, y, gate, post_weight, pre_weight, options):
    (s, n) of norm_block with the keyword arguments in the dict options, which
    have no gradients."""

    @staticmethod
    def forward(fn, ctx, x, y, gate, post_weight, pre_weight, options):
        s, n, stats = norm_block(ctx, x, y, gate, post_weight, pre_weight, save=True, **options)
        fn.ctx, fn.options = ctx, {k: v for k, v in options.items() if k != "next_norm"}
        fn.learned = _learned(**options)
        fn.save_for_backward(x, y, gate, post_weight, pre_weight, stats)
        fn.set_materialize_grads(False)
        return s, n

    @staticmethod
    @_first_only
    def backward(fn, ds, dn):
        x, y, gate, post_weight, pre_weight, stats = fn.saved_tensors
        grads = norm_block_backward(fn.ctx, _last_contiguous(ds), _last_contiguous(dn), x, y,
                                    gate, post_weight, pre_weight, stats, **fn.options)
        return (None, *grads, None)


class HeadNormRotaryFn(torch.autograd.Function):
    """HeadNormRotaryFn.apply(ctx, q, k, q_weight, k_weight, positions, freq,
    axis, options): (q, k) of head_norm_rotary with the keyword arguments in the
    dict options, with the gradients of q, k, the weights and floating-point
    positions.  freq and the options have none."""

    @staticmethod
    def forward(fn, ctx, q, k, q_weight, k_weight, positions, freq, axis, options):
        fn.ctx, fn.options, fn.learned = ctx, dict(options), _learned(freq=freq, **options)
        fn.save_for_backward(q, k, q_weight, k_weight, positions, freq, axis)
        fn.set_materialize_grads(False)
        return head_norm_rotary(ctx, q, k, q_weight, k_weight, positions, freq, axis, **options)

    @staticmethod
    @_first_only
    def backward(fn, dq, dk):
        q, k, q_weight, k_weight, positions, freq, axis = fn.saved_tensors
        dq = torch.zeros_like(q) if dq is None else dq
        dk = torch.zeros_like(k) if dk is None and k is not None else dk
        grads = head_norm_rotary_backward(
            fn.ctx, _last_contiguous(dq), _last_contiguous(dk), q, k, q_weight, k_weight, positions,
            freq, axis, dpositions=positions.requires_grad, **fn.options)
        return (None, *grads, None, None, None)

"""Operators on device tensors (the last section of include/mtpx.h) for torch
tensors: rotary positions with several axes, differential attention over
ragged batches and over a cache, and the norms around a block with its gate
and residual scale.

Every function takes the Context first, queues its kernels on torch's current
stream of the tensors' device and returns without waiting; workspaces and
results come from torch's allocator, so a call can be captured into a graph.
Functions with gradients come twice: as a pair (f, f_backward) on plain
tensors, and as an autograd function (RotaryFn, DiffAttentionFn, NormBlockFn).
Gradients are first derivatives: differentiating one of them again (a loss of
forces that were taken through a block) raises.
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


def _packer(cls):
    """The C layout of a request as one flat list of its fields: packing it
    takes a third of the time that filling the ctypes structure does, which
    counts in calls of a few microseconds."""
    codes = {_p: "P", _i: "i", _l: "q", _f: "f", C.c_size_t: "N"}
    fmt = "".join("Pqqq" if f is Rows else codes[f] for _, f in cls._fields_)
    # (a structure's size is a multiple of its strictest alignment)
    s = struct.Struct("@" + fmt + "0P")
    assert s.size == C.sizeof(cls)
    return s.pack


_pack_rotary, _pack_attention, _pack_cache, _pack_norm = (
    _packer(c) for c in (RotaryRequest, AttentionRequest, CacheRequest, NormRequest))

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
                          ("diff_attention_cache", _p), ("norm_block", _p)):
            getattr(L, "mtpx_" + name).argtypes = [ctx, req]
            getattr(L, "mtpx_%s_workspace" % name).argtypes = [ctx, req, size]
        L.mtpx_diff_attention_backward.argtypes = [ctx, C.POINTER(AttentionRequest)]
        L.mtpx_norm_block_backward.argtypes = [ctx, _p]
        _lib = L
    return _lib


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
    if (not isinstance(t, torch.Tensor) or t.get_device() != ctx.device or t.dtype is not dtype or
            t.shape != shape):
        _tensor(ctx, t, name, shape, dtype)  # says which
    s = t.stride()
    if s[-1] != 1 and t.shape[-1] > 1:
        _fail("the last dimension of %s is not contiguous" % name)
    return s


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


def _stream(ctx):
    return torch._C._cuda_getCurrentRawStream(ctx.device)


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

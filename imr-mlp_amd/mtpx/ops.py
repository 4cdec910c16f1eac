"""Operators on device tensors (the last section of include/mtpx.h) for torch
tensors: rotary positions with several axes, differential attention over
ragged batches and over a cache, and the norms around a block with its gate
and residual scale.

Every function takes the Context first, queues its kernels on torch's current
stream of the tensors' device and returns without waiting; workspaces and
results come from torch's allocator, so a call can be captured into a graph.
Functions with gradients come twice: as a pair (f, f_backward) on plain
tensors, and as an autograd function (RotaryFn, DiffAttentionFn, NormBlockFn).
Tensors are float32, bfloat16 or float16; their last dimension has to be
contiguous, other strides are free.  There is no fallback: a missing library
or a refused argument raises.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import capi
from .capi import MtpxError  # noqa: F401 -- what the calls raise

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


_lib = None


def _ops():
    """The library with the operators' signatures."""
    global _lib
    if _lib is None:
        L = capi.lib()
        ctx, size = C.c_void_p, C.POINTER(C.c_size_t)
        L.mtpx_rotary.argtypes = [ctx, C.POINTER(RotaryRequest)]
        L.mtpx_sequences_create.argtypes = [ctx, _i, C.POINTER(_l), C.POINTER(_l), C.POINTER(_p)]
        L.mtpx_sequences_destroy.argtypes = [_p]
        L.mtpx_sequences_destroy.restype = None
        for name, req in (("diff_attention", AttentionRequest),
                          ("diff_attention_cache", CacheRequest), ("norm_block", NormRequest)):
            getattr(L, "mtpx_" + name).argtypes = [ctx, C.POINTER(req)]
            getattr(L, "mtpx_%s_workspace" % name).argtypes = [ctx, C.POINTER(req), size]
        L.mtpx_diff_attention_backward.argtypes = [ctx, C.POINTER(AttentionRequest)]
        L.mtpx_norm_block_backward.argtypes = [ctx, C.POINTER(NormRequest)]
        _lib = L
    return _lib


def _fail(what):
    raise MtpxError(capi.ERRORS_BY_NAME["MTPX_E_INVALID"], what)


def _tensor(ctx, t, name, shape=None, dtype=None):
    """Checks a device tensor (None in shape: any size) and returns it."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.device.index != ctx.device:
        _fail("%s is not a tensor on the context's device" % name)
    if dtype is not None and t.dtype != dtype:
        _fail("%s is %s, not %s" % (name, t.dtype, dtype))
    if shape is not None and (t.dim() != len(shape) or
                              any(w is not None and w != n for w, n in zip(shape, t.shape))):
        _fail("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    return t


def _inner(t, name):
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _fail("the last dimension of %s is not contiguous" % name)
    return t


def _typed(ctx, t, name):
    _tensor(ctx, t, name)
    if t.dtype not in DTYPES:
        _fail("%s is %s, not float32, bfloat16 or float16" % (name, t.dtype))
    return DTYPES[t.dtype]


def _stream(ctx):
    return torch.cuda.current_stream(ctx.device).cuda_stream


def _heads(t):
    """[rows][heads][dim]"""
    return Rows(t.data_ptr(), t.stride(0), t.stride(1), 0)


def _maps(t):
    """[rows][heads][2][dim]"""
    return Rows(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _wide(t):
    """[rows][heads][2 dim] as two maps side by side"""
    return Rows(t.data_ptr(), t.stride(0), t.stride(1), t.shape[2] // 2)


def _workspace(ctx, query, req):
    n = C.c_size_t()
    ctx._check(query(ctx.h, C.byref(req), C.byref(n)), "workspace")
    w = torch.empty(n.value, dtype=torch.uint8, device=torch.device("cuda", ctx.device))
    req.workspace, req.workspace_bytes = w.data_ptr(), n.value
    return w


# ---- rotary positions ----------------------------------------------------------


def _rotary(ctx, x, positions, freq, axis, interleaved, inverse, out, forward, dpositions):
    dtype = _typed(ctx, x, "x")
    rows, heads, dim = _tensor(ctx, x, "x", (None, None, None)).shape
    _inner(x, "x")
    _tensor(ctx, positions, "positions", (rows, None))
    if positions.dtype not in POSITION_DTYPES:
        _fail("positions are %s, not float32, float64, int32 or int64" % positions.dtype)
    _tensor(ctx, freq, "freq", (None,), torch.float32)
    _tensor(ctx, axis, "axis", tuple(freq.shape), torch.int32)
    if not freq.is_contiguous() or not axis.is_contiguous():
        _fail("freq and axis must be contiguous")
    y = torch.empty((rows, heads, dim), dtype=x.dtype, device=x.device) if out is None else out
    if out is not None:
        _inner(_tensor(ctx, out, "out", (rows, heads, dim), x.dtype), "out")
    req = RotaryRequest(_stream(ctx), dtype, rows, heads, dim, 2 * freq.shape[0],
                        int(interleaved), int(inverse), _heads(x), _heads(y),
                        positions.data_ptr(), POSITION_DTYPES[positions.dtype],
                        positions.stride(0), positions.stride(1), positions.shape[1],
                        freq.data_ptr(), axis.data_ptr())
    if dpositions is not None:
        _inner(_tensor(ctx, forward, "x", (rows, heads, dim), x.dtype), "x")
        req.forward, req.dpositions = _heads(forward), dpositions.data_ptr()
    ctx._check(_ops().mtpx_rotary(ctx.h, C.byref(req)), "rotary")
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
    with the forward pass's x given (positions float32 or float64)."""
    dpos = None
    if x is not None:
        dpos = torch.empty(positions.shape, dtype=positions.dtype, device=dy.device)
    dx = _rotary(ctx, dy, positions, freq, axis, interleaved, True, None, x, dpos)
    return dx, dpos


# ---- differential attention ------------------------------------------------------


class Sequences:
    """mtpx_sequences: the row ranges of a ragged batch.  q_offsets and
    k_offsets (default: the same) are n + 1 ascending row numbers on the
    host."""

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

    def close(self):
        """Frees the tables, after the work queued on the device has ended."""
        if getattr(self, "h", None):
            _ops().mtpx_sequences_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


def _attention(ctx, q, k, v, lam, seqs, causal, scale, key_mask):
    dtype = _typed(ctx, q, "q")
    heads, dim = _tensor(ctx, q, "q", (None, None, 2, None)).shape[1::2]
    kv = _tensor(ctx, k, "k", (None, None, 2, dim), q.dtype).shape[1]
    _tensor(ctx, v, "v", (k.shape[0], kv, 2 * dim), q.dtype)
    if seqs.h is None:
        _fail("the sequences are closed")
    if q.shape[0] != seqs.q_rows or k.shape[0] != seqs.k_rows:
        _fail("q and k have %d and %d rows, the sequences %d and %d" %
              (q.shape[0], k.shape[0], seqs.q_rows, seqs.k_rows))
    _tensor(ctx, lam, "lam", (heads,), torch.float32)
    if not lam.is_contiguous():
        _fail("lam must be contiguous")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _inner(t, name)
    if key_mask is not None:
        _tensor(ctx, key_mask, "key_mask", (k.shape[0],))
        if key_mask.dtype not in (torch.bool, torch.uint8) or not key_mask.is_contiguous():
            _fail("key_mask must be contiguous bool or uint8")
    return AttentionRequest(_stream(ctx), dtype, seqs.h, heads, kv, dim, int(causal),
                            dim ** -0.5 if scale is None else scale, _maps(q), _maps(k), _wide(v),
                            None if key_mask is None else key_mask.data_ptr(), lam.data_ptr())


def diff_attention(ctx, q, k, v, lam, seqs, *, causal=False, scale=None, key_mask=None,
                   save=False, out=None):
    """(softmax(scale q0 k0^T) - lam softmax(scale q1 k1^T)) v per sequence and
    head: q [rows, heads, 2, dim], k [key rows, kv heads, 2, dim], v [key
    rows, kv heads, 2 dim], lam [heads] float32; scale defaults to dim^-1/2.
    Returns out [rows, heads, 2 dim], with save (out, saved) for
    diff_attention_backward."""
    req = _attention(ctx, q, k, v, lam, seqs, causal, scale, key_mask)
    rows, heads, _, dim = q.shape
    if out is None:
        out = torch.empty((rows, heads, 2 * dim), dtype=q.dtype, device=q.device)
    else:
        _inner(_tensor(ctx, out, "out", (rows, heads, 2 * dim), q.dtype), "out")
    req.out = _wide(out)
    saved = None
    if save:
        saved = (torch.empty((rows, heads, 2 * dim), dtype=q.dtype, device=q.device),
                 torch.empty((2, heads, rows), dtype=torch.float32, device=q.device))
        req.out1, req.lse = saved[0].data_ptr(), saved[1].data_ptr()
    ctx._check(_ops().mtpx_diff_attention(ctx.h, C.byref(req)), "diff_attention")
    return (out, saved) if save else out


def diff_attention_backward(ctx, dout, q, k, v, lam, seqs, out, saved, *, causal=False,
                            scale=None, key_mask=None):
    """(dq, dk, dv, dlam) from the gradient of out and what the forward call
    returned and saved."""
    req = _attention(ctx, q, k, v, lam, seqs, causal, scale, key_mask)
    rows, heads, _, dim = q.shape
    shape = (rows, heads, 2 * dim)
    _inner(_tensor(ctx, dout, "dout", shape, q.dtype), "dout")
    _inner(_tensor(ctx, out, "out", shape, q.dtype), "out")
    out1, lse = saved
    _tensor(ctx, out1, "saved[0]", shape, q.dtype)
    _tensor(ctx, lse, "saved[1]", (2, heads, rows), torch.float32)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=q.device)
    dv = torch.empty(v.shape, dtype=v.dtype, device=q.device)
    dlam = torch.empty(heads, dtype=torch.float32, device=q.device)
    req.out, req.dout, req.out1, req.lse = _wide(out), _wide(dout), out1.data_ptr(), lse.data_ptr()
    req.dq, req.dk, req.dv, req.dlambda = _maps(dq), _maps(dk), _wide(dv), dlam.data_ptr()
    w = _workspace(ctx, _ops().mtpx_diff_attention_workspace, req)  # noqa: F841 -- kept until queued
    ctx._check(_ops().mtpx_diff_attention_backward(ctx.h, C.byref(req)), "diff_attention_backward")
    return dq, dk, dv, dlam


def diff_attention_cache(ctx, q, k, v, lam, lengths, *, scale=None, out=None):
    """One row per sequence against a cache: q [sequences, heads, 2, dim],
    k [sequences, capacity, kv heads, 2, dim], v [sequences, capacity, kv
    heads, 2 dim], lengths [sequences] int32 on the device.  Returns
    [sequences, heads, 2 dim]."""
    dtype = _typed(ctx, q, "q")
    n, heads, _, dim = _tensor(ctx, q, "q", (None, None, 2, None)).shape
    cap, kv = _tensor(ctx, k, "k", (n, None, None, 2, dim), q.dtype).shape[1:3]
    _tensor(ctx, v, "v", (n, cap, kv, 2 * dim), q.dtype)
    _tensor(ctx, lengths, "lengths", (n,), torch.int32)
    _tensor(ctx, lam, "lam", (heads,), torch.float32)
    if not lam.is_contiguous() or not lengths.is_contiguous():
        _fail("lam and lengths must be contiguous")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _inner(t, name)
    if out is None:
        out = torch.empty((n, heads, 2 * dim), dtype=q.dtype, device=q.device)
    else:
        _inner(_tensor(ctx, out, "out", (n, heads, 2 * dim), q.dtype), "out")
    req = CacheRequest(_stream(ctx), dtype, n, heads, kv, dim, cap,
                       dim ** -0.5 if scale is None else scale, _maps(q),
                       Rows(k.data_ptr(), k.stride(1), k.stride(2), k.stride(3)),
                       Rows(v.data_ptr(), v.stride(1), v.stride(2), dim), k.stride(0),
                       v.stride(0), lengths.data_ptr(), lam.data_ptr(), _wide(out))
    w = _workspace(ctx, _ops().mtpx_diff_attention_cache_workspace, req)  # noqa: F841
    ctx._check(_ops().mtpx_diff_attention_cache(ctx.h, C.byref(req)), "diff_attention_cache")
    return out


# ---- norms around a block ----------------------------------------------------------


def _row(t):
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0))


def _norm(ctx, x, y, gate, post_weight, pre_weight, kind, gate_act, residual_scale, block_scale,
          eps):
    dtype = _typed(ctx, y, "y")
    rows, width = _tensor(ctx, y, "y", (None, None)).shape
    _inner(y, "y")
    if kind not in NORMS or gate_act not in GATES:
        _fail("kind is one of %s, gate_act of %s" % (tuple(NORMS), tuple(GATES)))
    if x is not None:
        _inner(_tensor(ctx, x, "x", (rows, width), y.dtype), "x")
    gate_row = 0
    if gate is not None:
        _inner(_tensor(ctx, gate, "gate", (width,) if gate.dim() == 1 else (rows, width), y.dtype),
               "gate")
        if gate.dim() == 2:
            gate_row = gate.stride(0)
            if gate_row == 0:
                _fail("a gate shared by all rows is [width]")
    for w, name in ((post_weight, "post_weight"), (pre_weight, "pre_weight")):
        if w is not None:
            _inner(_tensor(ctx, w, name, (width,), y.dtype), name)
    px, sx = _row(x)
    return NormRequest(_stream(ctx), dtype, rows, width, NORMS[kind], GATES[gate_act],
                       residual_scale, block_scale, eps, px, y.data_ptr(),
                       None if gate is None else gate.data_ptr(),
                       None if post_weight is None else post_weight.data_ptr(),
                       None if pre_weight is None else pre_weight.data_ptr(), sx, y.stride(0),
                       gate_row)


def norm_block(ctx, x, y, gate=None, post_weight=None, pre_weight=None, *, kind="rms",
               gate_act="none", residual_scale=1.0, block_scale=1.0, eps=1e-6, save=False,
               next_norm=True):
    """s = residual_scale x + block_scale act(gate) (norm(y) post_weight) and
    n = norm(s) pre_weight, for the block output y and the residual x [rows,
    width] (x None: no residual; gate [rows, width], [width] or None; weights
    [width] or None).  Returns (s, n), with save (s, n, stats); without
    next_norm n is None."""
    req = _norm(ctx, x, y, gate, post_weight, pre_weight, kind, gate_act, residual_scale,
                block_scale, eps)
    s = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    n = torch.empty_like(s) if next_norm else None
    (req.s, req.s_row), (req.n, req.n_row) = _row(s), _row(n)
    stats = None
    if save:
        stats = torch.empty((y.shape[0], 4), dtype=torch.float32, device=y.device)
        req.stats = stats.data_ptr()
    ctx._check(_ops().mtpx_norm_block(ctx.h, C.byref(req)), "norm_block")
    return (s, n, stats) if save else (s, n)


def norm_block_backward(ctx, ds, dn, x, y, gate, post_weight, pre_weight, stats, *, kind="rms",
                        gate_act="none", residual_scale=1.0, block_scale=1.0, eps=1e-6):
    """(dx, dy, dgate, dpost_weight, dpre_weight) from the gradients of s and n
    (either may be None) and the forward pass's inputs and stats; None in the
    place of an input that was not given."""
    req = _norm(ctx, x, y, gate, post_weight, pre_weight, kind, gate_act, residual_scale,
                block_scale, eps)
    _tensor(ctx, stats, "stats", (y.shape[0], 4), torch.float32)
    if not stats.is_contiguous():
        _fail("stats must be contiguous")
    for t, name in ((ds, "ds"), (dn, "dn")):
        if t is not None:
            _inner(_tensor(ctx, t, name, y.shape, y.dtype), name)
    req.stats = stats.data_ptr()
    (req.ds, req.ds_row), (req.dn, req.dn_row) = _row(ds), _row(dn)

    def like(t):
        return None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)

    dx, dy, dgate, dpost, dpre = like(x), like(y), like(gate), like(post_weight), like(pre_weight)
    (req.dx, req.dx_row), (req.dy, req.dy_row) = _row(dx), _row(dy)
    if dgate is not None:
        req.dgate, req.dgate_row = dgate.data_ptr(), dgate.stride(0) if dgate.dim() == 2 else 0
    if dpost is not None:
        req.dpost_weight = dpost.data_ptr()
    if dpre is not None:
        req.dpre_weight = dpre.data_ptr()
    w = _workspace(ctx, _ops().mtpx_norm_block_workspace, req)  # noqa: F841
    ctx._check(_ops().mtpx_norm_block_backward(ctx.h, C.byref(req)), "norm_block_backward")
    return dx, dy, dgate, dpost, dpre


# ---- autograd ------------------------------------------------------------------------


def _last_contiguous(t):
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


class RotaryFn(torch.autograd.Function):
    """RotaryFn.apply(ctx, x, positions, freq, axis, interleaved): rotary with
    the gradients of x and of floating-point positions."""

    @staticmethod
    def forward(fn, ctx, x, positions, freq, axis, interleaved=False):
        fn.ctx, fn.interleaved = ctx, interleaved
        keep = x if positions.requires_grad else None
        fn.save_for_backward(keep, positions, freq, axis)
        return rotary(ctx, x, positions, freq, axis, interleaved=interleaved)

    @staticmethod
    def backward(fn, dy):
        x, positions, freq, axis = fn.saved_tensors
        dx, dpos = rotary_backward(fn.ctx, _last_contiguous(dy), positions, freq, axis,
                                   interleaved=fn.interleaved, x=x)
        return None, dx, dpos, None, None, None


class DiffAttentionFn(torch.autograd.Function):
    """DiffAttentionFn.apply(ctx, q, k, v, lam, seqs, causal, scale, key_mask)."""

    @staticmethod
    def forward(fn, ctx, q, k, v, lam, seqs, causal=False, scale=None, key_mask=None):
        out, saved = diff_attention(ctx, q, k, v, lam, seqs, causal=causal, scale=scale,
                                    key_mask=key_mask, save=True)
        fn.ctx, fn.seqs, fn.causal, fn.scale = ctx, seqs, causal, scale
        fn.save_for_backward(q, k, v, lam, out, *saved, key_mask)
        return out

    @staticmethod
    def backward(fn, dout):
        q, k, v, lam, out, out1, lse, mask = fn.saved_tensors
        grads = diff_attention_backward(fn.ctx, _last_contiguous(dout), q, k, v, lam, fn.seqs,
                                        out, (out1, lse), causal=fn.causal, scale=fn.scale,
                                        key_mask=mask)
        return (None, *grads, None, None, None, None)


class NormBlockFn(torch.autograd.Function):
    """NormBlockFn.apply(ctx, x, y, gate, post_weight, pre_weight, options):
    norm_block with the keyword arguments in the dict options."""

    @staticmethod
    def forward(fn, ctx, x, y, gate, post_weight, pre_weight, options):
        s, n, stats = norm_block(ctx, x, y, gate, post_weight, pre_weight, save=True, **options)
        fn.ctx, fn.options = ctx, options
        fn.save_for_backward(x, y, gate, post_weight, pre_weight, stats)
        fn.set_materialize_grads(False)
        return s, n

    @staticmethod
    def backward(fn, ds, dn):
        x, y, gate, post_weight, pre_weight, stats = fn.saved_tensors
        grads = norm_block_backward(fn.ctx, _last_contiguous(ds), _last_contiguous(dn), x, y,
                                    gate, post_weight, pre_weight, stats, **fn.options)
        return (None, *grads, None)

"""The gated linear recurrence h_t = gate_t * h_{t-1} + x_t over many sequences, its gradient and its single step.

It is what compositing along a ray is -- C = alpha c + (1 - alpha) C_behind, from the last hit to the first -- and what
layers with a decaying state run over long sequences.  For decoders and losses outside the fused render path:

    t, hits = renderer.Render(O, v, t_min, size)                             # (16, size), slot-major
    _, colour, saved = recurrence.scan((1 - alpha).T[..., None], (alpha[..., None] * c).transpose(0, 1), background,
                                       reverse=True, states=False, training=True)
    dgate, dx, dbackground = recurrence.scan_backward(gate, x, saved, None, dcolour, background, reverse=True)

No reference counterpart (the reference composites inside its kernels only).
"""
from __future__ import annotations

import torch

from . import _lib, _ops

_FLOATS = tuple(_ops.TYPE_CODE)
_F32 = (torch.float32,)


def _dense(t):
    """t, or a copy of it whose last dimension is dense."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _like(t, width, dtype):
    """An uninitialised tensor with t's leading dimensions in t's memory order."""
    if t.dim() == 3 and t.stride(0) < t.stride(1) and t.shape[0] > 1:
        return torch.empty((t.shape[1], t.shape[0], width), dtype=dtype, device=t.device).transpose(0, 1)
    return torch.empty(t.shape[:-1] + (width,), dtype=dtype, device=t.device)


def _strides(t):
    """(per sequence, per step) in elements; a single step's stride means nothing."""
    if t is None:
        return 0, 0
    return (t.stride(0) if t.dim() == 3 else 0), (t.stride(-2) if t.shape[-2] > 1 else 0)


def _inputs(gate, x, state, offsets):
    """Checks; returns (gate, x, offsets, seqs)."""
    _ops.need(x, "x", _FLOATS)
    dev = x.device
    _ops.need(gate, "gate", (x.dtype, torch.float32), dev)
    if offsets is None:
        if x.dim() != 3 or x.shape[2] < 1:
            raise ValueError(f"x: shape {tuple(x.shape)}, expected (sequences, steps, width)")
        seqs = x.shape[0]
    else:
        _ops.need(offsets, "offsets", tuple(_ops.INDEX_CODE), dev)
        if x.dim() != 2 or x.shape[1] < 1:
            raise ValueError(f"x: shape {tuple(x.shape)}, expected (rows, width) with offsets")
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError(f"offsets: shape {tuple(offsets.shape)}, expected (sequences + 1,)")
        seqs, offsets = offsets.numel() - 1, offsets.contiguous()
    if gate.dim() != x.dim() or gate.shape[:-1] != x.shape[:-1] or gate.shape[-1] < 1 or x.shape[-1] % gate.shape[-1]:
        raise ValueError(f"gate: shape {tuple(gate.shape)}, expected {tuple(x.shape[:-1])} + (groups,), groups dividing "
                         f"{x.shape[-1]}")
    if seqs * x.shape[-1] >= 2 ** 30 or x.shape[-2] >= 2 ** 30:
        raise ValueError(f"x: {seqs} sequences of {x.shape[-1]} channels, {x.shape[-2]} steps, at most 2^30 channels in all and "
                         "2^30 steps")
    _ends(state, "state", seqs, x)
    return _dense(gate), _dense(x), offsets, seqs


def _ends(t, name, seqs, x):
    if t is not None:
        _ops.need(t, name, _F32, x.device)
        _ops.need_shape(t, name, (seqs, x.shape[-1]))


def _launch(lib, backward, what, seqs, reverse, gate, x, state, offsets, h=None, last=None, saved=None, dh=None, dlast=None, dgate=None,
            dx=None, dstate=None):
    p, dev, steps = _ops.ptr, x.device, x.shape[-2]
    head = (gate.data_ptr(), x.data_ptr(), p(state), p(offsets), p(h), p(last), p(saved), p(dh), p(dlast), p(dgate), p(dx), p(dstate))
    tail = (seqs, steps, *_strides(gate), *_strides(x), *_strides(h), *_strides(dh), *_strides(dgate), *_strides(dx), x.shape[-1],
            gate.shape[-1], _ops.TYPE_CODE[gate.dtype], _ops.TYPE_CODE[x.dtype],
            0 if offsets is None else _ops.INDEX_CODE[offsets.dtype], 1 if reverse else 0)
    ws, nbytes = None, 0
    if backward or steps > _lib.RECURRENCE_SPAN:  # a forward of one span needs none
        nbytes = lib.flare_recurrence_workspace(_lib.PACK_RECURRENCE.pack(*head, 0, 0, *tail), backward)
        ws = _ops.workspace(nbytes, dev)
    a = _lib.PACK_RECURRENCE.pack(*head, p(ws), nbytes, *tail)
    _lib.check((lib.flare_recurrence_backward if backward else lib.flare_recurrence_forward)(a, _ops.stream(dev)), what)


def scan(gate, x, state=None, offsets=None, reverse=False, states=True, training=False):
    """Runs the recurrence; returns (h, last, saved).

    x: (sequences, steps, width) f32, f16 or bf16, any strides with a dense last dimension (others are copied).  gate:
    (sequences, steps, groups), of x's type or f32; each gate is shared by width / groups consecutive channels.
    state: (sequences, width) f32, what precedes the first step, None for 0.  reverse: from the last step to the first.
    With offsets (sequences + 1,) int32 or int64, non-decreasing, x is (rows, width) and gate (rows, groups), and
    sequence s is rows offsets[s] to offsets[s + 1]; it may be empty.  Rows of no sequence get zeros.
    h: every state, of x's shape and type (None if not states); last: the final states (sequences, width) f32; saved:
    what scan_backward needs (None if not training).  The recurrence runs in 32 bits, h is rounded once.  Time is
    cut into stretches, and the product of a stretch's gates is a float: where it is too small, the state that enters the
    stretch counts as 0 behind it; where it is too large (gates above 1), a state other than 0 gives infinity or NaN behind it
    even if single steps would stay finite.  A tensor's steps are less than 2 GB apart
    (FlareError).
    """
    lib = _lib.load()
    gate, x, offsets, seqs = _inputs(gate, x, state, offsets)
    state = None if state is None else state.contiguous()
    dev, width = x.device, x.shape[-1]
    with _ops.on(dev):
        h = _like(x, width, x.dtype) if states else None
        last = torch.empty((seqs, width), dtype=torch.float32, device=dev)
        saved = None
        if training:
            n = lib.flare_recurrence_saved(seqs, x.shape[-2], width, 0 if offsets is None else 1)
            saved = torch.empty(n, dtype=torch.float32, device=dev)
        _launch(lib, 0, "scan", seqs, reverse, gate, x, state, offsets, h, last, saved)
    return h, last, saved


def scan_backward(gate, x, saved, dh=None, dlast=None, state=None, offsets=None, reverse=False):
    """Gradients of `scan` with the same gate, x, state, offsets and reverse: (dgate, dx, dstate).

    saved: from scan(..., training=True).  dh: the gradient of h, of x's shape and type, dlast: that of last,
    (sequences, width) f32; None for 0.  dgate and dx have the types of gate and x and are rounded once; dstate is
    (sequences, width) f32, None without a state.  Sums run in a fixed order, so results repeat bit for bit.
    """
    lib = _lib.load()
    gate, x, offsets, seqs = _inputs(gate, x, state, offsets)
    state = None if state is None else state.contiguous()
    dev, width = x.device, x.shape[-1]
    _ops.need(saved, "saved", _F32, dev)
    n = lib.flare_recurrence_saved(seqs, x.shape[-2], width, 0 if offsets is None else 1)
    if saved.numel() != n or not saved.is_contiguous():
        raise ValueError(f"saved: {saved.numel()} elements, expected the {n} of scan(..., training=True)")
    if dh is not None:
        _ops.need(dh, "dh", (x.dtype,), dev)
        dh = _dense(_ops.need_shape(dh, "dh", x.shape))
    _ends(dlast, "dlast", seqs, x)
    dlast = None if dlast is None else dlast.contiguous()
    with _ops.on(dev):
        dgate, dx = _like(gate, gate.shape[-1], gate.dtype), _like(x, width, x.dtype)
        dstate = None if state is None else torch.empty_like(state)
        _launch(lib, 1, "scan_backward", seqs, reverse, gate, x, state, offsets, None, None, saved, dh, dlast, dgate, dx, dstate)
    return dgate, dx, dstate


def step(gate, x, state, out=None):
    """One step for every sequence, for a caller that keeps the state: out = gate * state + x, f32 (sequences, width),
    written in place of `state` unless another tensor is given; returns it in x's type (a new tensor).

    x: (sequences, width) f32, f16 or bf16; gate: (sequences, groups), of x's type or f32.  What is written may be one of
    the inputs, element for element, and overlaps them in no other way (FlareError).
    """
    lib = _lib.load()
    _ops.need(x, "x", _FLOATS)
    dev = x.device
    _ops.need(gate, "gate", (x.dtype, torch.float32), dev)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x: shape {tuple(x.shape)}, expected (sequences, width)")
    seqs, width = x.shape
    if gate.dim() != 2 or gate.shape[0] != seqs or gate.shape[1] < 1 or width % gate.shape[1]:
        raise ValueError(f"gate: shape {tuple(gate.shape)}, expected ({seqs}, groups), groups dividing {width}")
    if seqs * width >= 2 ** 30:
        raise ValueError(f"x: {seqs} sequences of {width} channels, at most 2^30 channels in all")
    out = state if out is None else out
    for t, name in ((state, "state"), (out, "out")):
        _ops.need_shape(_ops.need(t, name, _F32, dev), name, x.shape)
        if not t.is_contiguous():
            raise ValueError(f"{name}: tensor must be contiguous")
    gate, x = _dense(gate), _dense(x)
    with _ops.on(dev):
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
        # one step of `seqs` sequences: the rows are the sequences
        a = _lib.PACK_RECURRENCE.pack(gate.data_ptr(), x.data_ptr(), state.data_ptr(), 0, h.data_ptr(), out.data_ptr(), 0, 0, 0, 0, 0, 0,
                                      0, 0, seqs, 1, gate.stride(0), 0, x.stride(0), 0, width, 0, 0, 0, 0, 0, 0, 0, width,
                                      gate.shape[1], _ops.TYPE_CODE[gate.dtype], _ops.TYPE_CODE[x.dtype], 0, 0)
        _lib.check(lib.flare_recurrence_forward(a, _ops.stream(dev)), "step")
    return h

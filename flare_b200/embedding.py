"""Rows of a descriptor table for a list of hits, with scaling, and the table's gradient.

For decoders, losses and feature maps that a caller writes outside the fused render path: `Render`'s hit lists name
primitives, -1 where a ray has no further hit, and `lookup` fetches their descriptor rows, `lookup_backward` turns the
gradients of the fetched rows into the table's:

    t, hits = renderer.Render(O, v, t_min, size)                      # (16, size), -1 padded
    rows = embedding.lookup(scene.cond, hits, weight)                 # (16, size, 96)
    ...
    dcond, dweight = embedding.lookup_backward(drows, scene.cond, hits, weight)   # f32, as the optimizer takes them

No reference counterpart (the reference reads descriptors inside its decoder kernels only).
"""
from __future__ import annotations

import torch

from . import _lib, _ops
from .microscale import Micro4

_FLOATS = tuple(_ops.TYPE_CODE)
_INDICES = tuple(_ops.INDEX_CODE)
MAX_ROWS, MAX_ENTRIES = 2 ** 31 - 2, 2 ** 31 - 8193  # of lookup_backward


def _entries(idx, weight, device):
    _ops.need(idx, "idx", _INDICES, device)
    if weight is not None:
        _ops.need(weight, "weight", (torch.float32,), device)
        _ops.need_shape(weight, "weight", idx.shape)
        weight = weight.contiguous()
    return idx.contiguous(), weight


def lookup(table, idx, weight=None, scale=1.0, dtype=None):
    """scale * weight[i] * table[idx[i]] for every entry of idx: a new tensor of shape idx.shape + (width,).

    table: (rows, width) f32, f16 or bf16, or a `Micro4`; rows may be strided.  idx: int32 or int64 of any shape; an
    index outside [0, rows) names no row and gives zeros whatever its weight, as Render's -1 does.  weight: f32 of
    idx's shape or None (1).  dtype: the result's, by default the table's (f16 for a Micro4).  Products are formed in
    32 bits and rounded once.  Runs on the current stream of the table's device.
    """
    lib = _lib.load()
    micro = isinstance(table, Micro4)
    if micro:
        device, (n_rows, width) = table.codes.device, table.shape
    else:
        _ops.need(table, "table", _FLOATS)
        if table.dim() != 2:
            raise ValueError(f"table: shape {tuple(table.shape)}, expected (rows, width)")
        device, (n_rows, width) = table.device, table.shape
        table = _ops.rows(table)
    dtype = dtype or (torch.float16 if micro else table.dtype)
    if dtype not in _ops.TYPE_CODE:
        raise ValueError(f"dtype: {dtype}, expected one of {', '.join(str(d) for d in _FLOATS)}")
    idx, weight = _entries(idx, weight, device)
    with _ops.on(device):
        out = torch.empty(idx.shape + (width,), dtype=dtype, device=device)
        a = _lib.PACK_LOOKUP.pack(
            (table.codes if micro else table).data_ptr(), table.scales.data_ptr() if micro else 0, idx.data_ptr(), _ops.ptr(weight),
            out.data_ptr(), n_rows, idx.numel(), 0 if micro else table.stride(0), width, width,
            _ops.MICRO if micro else _ops.TYPE_CODE[table.dtype], _ops.INDEX_CODE[idx.dtype], _ops.TYPE_CODE[dtype], scale)
        _lib.check(lib.flare_lookup(a, _ops.stream(device)), "lookup")
    return out


def lookup_backward(dout, table, idx, weight=None, scale=1.0, need_table=True, need_weight=None):
    """Gradients of `lookup` with the same table, idx, weight and scale: (dtable (rows, width) f32, dweight f32 of
    idx's shape), each None where it is not asked for (need_weight: by default whether there is a weight).

    dout: idx.shape + (width,), f32, f16 or bf16, of any type whatever the table's.  The entries of a row are added in
    32 bits in an order that the sizes fix (ascending within stretches of 32 to 256 sorted entries, whose sums are then
    added), so results repeat bit for bit; rows that no entry names get zeros.  A Micro4 table
    has no gradient: ValueError.
    """
    lib = _lib.load()
    _ops.need(table, "table", _FLOATS)
    if table.dim() != 2:
        raise ValueError(f"table: shape {tuple(table.shape)}, expected (rows, width)")
    device, (n_rows, width) = table.device, table.shape
    table = _ops.rows(table)
    idx, weight = _entries(idx, weight, device)
    _ops.need(dout, "dout", _FLOATS, device)
    _ops.need_shape(dout, "dout", tuple(idx.shape) + (width,))
    n = idx.numel()
    if n_rows > MAX_ROWS or n > MAX_ENTRIES:
        raise ValueError(f"lookup_backward: {n_rows} rows and {n} entries, at most {MAX_ROWS} and {MAX_ENTRIES}")
    dout = _ops.rows(dout)
    need_weight = weight is not None if need_weight is None else need_weight
    with _ops.on(device):
        dtable = torch.empty((n_rows, width), dtype=torch.float32, device=device) if need_table else None
        dweight = torch.empty(idx.shape, dtype=torch.float32, device=device) if need_weight else None
        ws = _ops.workspace(lib.flare_lookup_workspace(n_rows, n, width) if need_table else 0, device)
        a = _lib.PACK_LOOKUP_GRAD.pack(
            dout.data_ptr(), table.data_ptr(), idx.data_ptr(), _ops.ptr(weight), _ops.ptr(dtable), _ops.ptr(dweight), _ops.ptr(ws),
            n_rows, n, dout.stride(0) if n else width, table.stride(0), 0 if ws is None else ws.numel(), width,
            _ops.TYPE_CODE[table.dtype], _ops.INDEX_CODE[idx.dtype], _ops.TYPE_CODE[dout.dtype], scale)
        _lib.check(lib.flare_lookup_backward(a, _ops.stream(device)), "lookup_backward")
    return dtable, dweight

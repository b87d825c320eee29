"""Matrices held in 4 bits an element with a power-of-two scale per 32 (microscaled 4-bit floats), and their product.

A 96-wide f16 descriptor takes 192 bytes; held here it takes 52, in memory and in each row that `embedding.lookup` reads.
`quantize` makes a `Micro4` from a tensor, `Micro4.dequantize` reads it back, and `product` multiplies two of them on the
tensor cores.  The renderer's inference methods take one as `conditioning_variable` too, but expand the whole table to f16 at
every call (a pass over it and as much memory again while the call runs): for many frames `dequantize` it once.  Inference only: none of them has a
gradient.  No reference counterpart.
"""
from __future__ import annotations

import torch

from . import _lib, _ops

BLOCK = 32  # elements that share a scale
_FLOATS = tuple(_ops.TYPE_CODE)
_BYTES = (torch.uint8,)


class Micro4:
    """A (rows, width) matrix in 4 bits an element.

    codes (rows, 16 * blocks) uint8, blocks = ceil(width / 32): two elements a byte, the even one in the low four
    bits, each a sign bit and the magnitude 0, .5, 1, 1.5, 2, 3, 4 or 6; zero past `width`.  scales (rows, 4 *
    ceil(blocks / 4)) uint8: a block's elements are multiplied by 2^(byte - 127), byte 255 stands for NaN; bytes past
    `blocks` are not used.  Both contiguous.
    """

    __slots__ = ("codes", "scales", "width")

    def __init__(self, codes, scales, width: int):
        """Checks and keeps the two tensors."""
        width = int(width)
        blocks = -(-width // BLOCK)
        _ops.need(codes, "codes", _BYTES)
        _ops.need(scales, "scales", _BYTES, codes.device)
        if width < 1 or codes.dim() != 2:
            raise ValueError(f"codes: shape {tuple(codes.shape)} for a width of {width}")
        rows = codes.shape[0]
        _ops.need_shape(codes, "codes", (rows, 16 * blocks))
        _ops.need_shape(scales, "scales", (rows, (blocks + 3) // 4 * 4))
        if not codes.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError("codes: tensor must be contiguous and aligned to 16 bytes")
        if not scales.is_contiguous() or scales.data_ptr() % 4:
            raise ValueError("scales: tensor must be contiguous and aligned to 4 bytes")
        self.codes, self.scales, self.width = codes, scales, width

    @property
    def shape(self):
        return self.codes.shape[0], self.width

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float16):
        """The (rows, width) values, rounded to f32, f16 or bf16."""
        lib = _lib.load()
        if dtype not in _ops.TYPE_CODE:
            raise ValueError(f"dtype: {dtype}, expected one of {', '.join(str(d) for d in _FLOATS)}")
        with _ops.on(self.device):
            out = torch.empty(self.shape, dtype=dtype, device=self.device)
            _lib.check(lib.flare_micro_dequantize(_ops.ptr(self.codes), _ops.ptr(self.scales), self.shape[0], self.width,
                                                  _ops.ptr(out), _ops.TYPE_CODE[dtype], self.width,
                                                  _ops.stream(self.device)), "dequantize")
        return out


def quantize(x) -> Micro4:
    """The 4-bit form of a (rows, width) tensor, f32, f16 or bf16, width >= 1; rows may be strided.

    A block's scale is 2^(floor(log2 of its largest magnitude) - 2); elements go to the nearest value, ties to the even
    code, and to 6 scales at most.  A block that holds an infinity or a NaN becomes NaN.
    """
    lib = _lib.load()
    _ops.need(x, "x", _FLOATS)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x: shape {tuple(x.shape)}, expected (rows, width)")
    rows, width = x.shape
    x = _ops.rows(x)
    blocks = -(-width // BLOCK)
    with _ops.on(x.device):
        codes = torch.empty((rows, 16 * blocks), dtype=torch.uint8, device=x.device)
        scales = torch.empty((rows, -(-blocks // 4) * 4), dtype=torch.uint8, device=x.device)
        _lib.check(lib.flare_micro_quantize(_ops.ptr(x), _ops.TYPE_CODE[x.dtype], rows, width, x.stride(0),
                                            _ops.ptr(codes), _ops.ptr(scales), _ops.stream(x.device)), "quantize")
    q = Micro4.__new__(Micro4)  # made here, so there is nothing to check
    q.codes, q.scales, q.width = codes, scales, width
    return q


def product(x, w: Micro4, dtype=torch.bfloat16, check=False):
    """x (m, k) times the transpose of w (n, k): a new (m, n) tensor of f32, f16 or bf16, accumulated in 32 bits.

    x: a `Micro4`, or an f32, f16 or bf16 tensor that is quantized first (up to 16 rows inside the product).  check: wait for
    the product and raise FlareError if a wait inside the kernel ran out (without it such a tile is NaN).
    """
    lib = _lib.load()
    if not isinstance(w, Micro4):
        raise ValueError(f"w: expected a Micro4, got {type(w).__name__}")
    dev = w.codes.device
    plain = None
    if not isinstance(x, Micro4):
        _ops.need(x, "x", _FLOATS, dev)
        if x.dim() != 2:
            raise ValueError(f"x: shape {tuple(x.shape)}, expected (m, {w.width})")
        if x.shape[0] <= _lib.PRODUCT_ROWS:
            plain = _ops.rows(x)  # quantized on the way
        else:
            x = quantize(x)
    if dtype not in _ops.TYPE_CODE:
        raise ValueError(f"dtype: {dtype}, expected one of {', '.join(str(d) for d in _FLOATS)}")
    (m, k), n = x.shape, w.codes.shape[0]
    if k != w.width:
        raise ValueError(f"x has {k} columns, w has {w.width}")
    if x.device != dev:
        raise ValueError(f"w: tensor on {dev}, expected {x.device}")
    with _ops.on(dev):
        out = torch.empty((m, n), dtype=dtype, device=dev)
        ws = _ops.workspace(lib.flare_micro_product_workspace(m, n, k), dev)
        status = torch.zeros(1, dtype=torch.int32, device=dev) if check else None
        a, scales, p, stride, code = (x.codes.data_ptr(), x.scales.data_ptr(), 0, 0, 0) if plain is None else (
            0, 0, plain.data_ptr(), plain.stride(0), _ops.TYPE_CODE[plain.dtype])
        a = _lib.PACK_PRODUCT.pack(a, scales, w.codes.data_ptr(), w.scales.data_ptr(), p, out.data_ptr(), _ops.ptr(ws), _ops.ptr(status),
                                   m, n, n, stride, 0 if ws is None else ws.numel(), k, _ops.TYPE_CODE[dtype], code)
        _lib.check(lib.flare_micro_product(a, _ops.stream(dev)), "product")
    if check and int(status):
        raise _lib.FlareError(f"product: device reported error bits 0x{int(status):x} (tensor-core wait timeout)")
    return out

"""Microscaled 4-bit matrices: quantisation, values, lookup and product against a 64-bit restatement (GPU), refusals (CPU)."""
import numpy as np
import pytest
import torch

import ops_reference as ref
from flare_b200 import _lib, embedding, microscale

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _same(got, want):
    assert got.shape == want.shape
    assert np.array_equal(np.nan_to_num(ref.f64(got), nan=-1e300), np.nan_to_num(want, nan=-1e300))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,pad", [(1, 1, 0), (3, 31, 0), (5, 32, 0), (7, 33, 0), (100, 96, 0), (9, 129, 0), (4, 1000, 0), (6, 96, 8),
                                            (6, 40, 3)])
@pytest.mark.parametrize("x", [F32, F16, BF16])
def test_quantize(rows, width, pad, x):
    g = torch.Generator().manual_seed(width)
    t = (torch.randn(rows, width + pad, generator=g) * torch.exp(4 * torch.randn(rows, 1, generator=g))).to(x)
    q = microscale.quantize(t.to(DEV)[:, :width])
    want, scales = ref.quantize(ref.f64(t[:, :width]))
    nb = -(-width // 32)
    assert np.array_equal(q.scales.cpu().numpy()[:, :nb], scales) and not q.scales[:, nb:].any()
    codes = q.codes.cpu().numpy()
    assert np.array_equal(ref.values(codes, q.scales.cpu().numpy(), width), want)
    assert np.array_equal(np.signbit(ref.values(codes, q.scales.cpu().numpy(), width)), np.signbit(want))
    past = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)[:, width:]
    assert not past.any()
    _same(q.dequantize(F32), want)
    for t in (F16, BF16):
        _same(q.dequantize(t), ref.f64(torch.from_numpy(want).float().to(t)))


@pytest.mark.gpu
def test_quantize_every_tie_and_border():
    v = torch.tensor([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99])
    v = torch.cat([v, torch.nextafter(v, v + 1), torch.nextafter(v, v - 1)])
    x = torch.zeros(len(v), 2, 32)
    x[:, 0, 0] = 4.0  # a scale of 1
    x[:, 0, 1], x[:, 0, 2] = v, -v
    x[:, 1] = x[:, 0] * 2.0 ** 20
    x = x.reshape(len(v), 64)
    q = microscale.quantize(x.to(DEV))
    want, scales = ref.quantize(ref.f64(x))
    assert np.array_equal(q.scales.cpu().numpy()[:, :2], scales)
    _same(q.dequantize(F32), want)


@pytest.mark.gpu
def test_quantize_ends_of_the_range():
    big, small = torch.finfo(F32).max, 2.0 ** -149
    x = torch.zeros(9, 32)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[4, 5] = big, small, 2.0 ** -126, -0.0, 2.0 ** -125
    x[5, 3], x[6, 4], x[7, 5] = float("nan"), float("inf"), -float("inf")
    x[5:8, 0] = 1.0
    x[8] = torch.linspace(-2.0 ** -140, 2.0 ** -127, 32)
    q = microscale.quantize(x.to(DEV))
    want, scales = ref.quantize(ref.f64(x))
    assert np.array_equal(q.scales.cpu().numpy()[:, 0], scales[:, 0])
    assert q.scales[:, 0].tolist()[5:8] == [255] * 3 and q.scales[3, 0] == 0
    _same(q.dequantize(F32), want)
    assert torch.isnan(q.dequantize(BF16)[5:8]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 6, 12, 32, 96, 100, 1023])
@pytest.mark.parametrize("out", [F32, F16, BF16])
def test_lookup_reads_a_4_bit_table(width, out):
    g = torch.Generator().manual_seed(width)
    q = microscale.quantize(torch.randn(50, width, generator=g).to(DEV))
    idx = torch.randint(-1, 52, (77,), generator=g)
    w = torch.rand(77, generator=g)
    got = embedding.lookup(q, idx.to(DEV), w.to(DEV), 0.5, dtype=out)
    want = ref.lookup(ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), width), idx.numpy(), ref.f64(w), 0.5)
    ref.close(got, want, 3 * ref.U * np.abs(want))
    assert embedding.lookup(q, idx.to(DEV)).dtype == F16
    with pytest.raises(ValueError):
        embedding.lookup_backward(got, q, idx.to(DEV))


def test_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        microscale.quantize(torch.zeros(2, 3))
    with pytest.raises(ValueError, match="x: dtype"):
        microscale.quantize(torch.zeros(2, 3, dtype=torch.float64))
    with pytest.raises(ValueError, match="codes"):
        microscale.Micro4(torch.zeros(2, 3), torch.zeros(2, 4), 3)


@pytest.mark.gpu
def test_refusals_on_the_device():
    q = microscale.quantize(torch.ones(4, 40, device=DEV))
    for bad in (lambda: microscale.quantize(torch.ones(4, device=DEV)), lambda: microscale.quantize(torch.ones(4, 0, device=DEV)),
                lambda: q.dequantize(torch.float64),
                lambda: microscale.Micro4(q.codes, q.scales, 65), lambda: microscale.Micro4(q.codes[:2], q.scales, 40),
                lambda: microscale.Micro4(q.codes[:, :16], q.scales, 32)):
        with pytest.raises(ValueError):
            bad()


def test_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    assert lib.flare_micro_quantize(None, 0, 1, 4, 4, None, None, None) == 1 and b"NULL" in lib.flare_last_error()
    assert lib.flare_micro_quantize(None, 3, 1, 4, 4, None, None, None) == 1 and b"type" in lib.flare_last_error()
    assert lib.flare_micro_dequantize(None, None, 1, 0, None, 0, 4, None) == 1
    assert lib.flare_micro_dequantize(16, 16, 1, 8, 16, 0, 4, None) == 1 and b"overlap" in lib.flare_last_error()

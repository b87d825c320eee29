"""Microscaled 4-bit matrices: quantisation, values, lookup and product against a 64-bit restatement (GPU), refusals (CPU)."""
import ctypes
import os
import shutil
import subprocess

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
                                            (6, 40, 3), (5, 16, 0), (5, 48, 0), (9, 80, 16), (3, 1008, 0)])
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


def _product(m, n, k, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    a, b = ((torch.randn(r, k, generator=g) * torch.exp(spread * torch.randn(r, 1, generator=g))).to(DEV) for r in (m, n))
    qa, qb = microscale.quantize(a), microscale.quantize(b)
    va, vb = (ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), k) for q in (qa, qb))
    # products are exact; an addition may truncate (a whole step of 2^-23) what it adds to sums of magnitudes
    return qa, qb, va @ vb.T, (k + 2) * 2 * ref.U * (np.abs(va) @ np.abs(vb).T)


SIZES = [(1, 1, 1), (1, 1, 33), (3, 5, 64), (128, 128, 256), (129, 64, 96), (1, 300, 500), (300, 1, 4000), (200, 260, 1000),
         (130, 513, 31), (4, 1000, 4096), (1000, 7, 128), (257, 129, 2049), (5, 2000, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k, out):
    qa, qb, want, err = _product(m, n, k, spread=0.3)
    got = microscale.product(qa, qb, dtype=out, check=True)
    assert got.dtype == out
    ref.close(got, want, err)
    assert torch.equal(got, microscale.product(qa, qb, dtype=out))


@pytest.mark.gpu
def test_product_of_whole_numbers_is_exact():
    """Codes and scales whose products and sums are small whole numbers: any order and any place of an element that is
    taken wrongly shows."""
    g = torch.Generator().manual_seed(5)
    for m, n, k in ((300, 280, 520), (2, 700, 1030), (513, 64, 96), (4500, 2100, 1290), (2100, 4481, 2600), (70_000, 50, 96),
                    (90_001, 64, 96), (45_000, 128, 250), (12, 60_003, 31), (76_000, 17, 129)):
        lev = torch.tensor([0.0, 1.0, 2.0, 3.0, 4.0, -1.0, -2.0])
        a, b = lev[torch.randint(0, 7, (m, k), generator=g)], lev[torch.randint(0, 7, (n, k), generator=g)]
        for t in (a, b):
            t[:, ::32] = 4.0  # every block's scale is 1 ...
            for c in range(0, k, 32):  # ... times a power of two that differs from block to block and row to row
                t[:, c:c + 32] *= 2.0 ** ((torch.arange(t.shape[0])[:, None] + c // 32) % 3).float()
        got = microscale.product(a.to(DEV), microscale.quantize(b.to(DEV)), dtype=F32)
        assert torch.equal(got.cpu(), a @ b.T)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2500, 2401, 600), (2333, 2600, 1000), (300, 20_000, 4096), (3001, 2000, 2049)])
def test_product_of_many_wide_tiles_is_exact(m, n, k):
    """Tiles of 192 columns, several per block, scale rows of whole 16 bytes and not: small whole numbers, so equality."""
    g = torch.Generator().manual_seed(m)
    a, b = (torch.randint(-1, 2, (r, k), generator=g).float() for r in (m, n))
    for t in (a, b):
        t[:, ::32] = 4.0  # every block's scale is 1 ...
        t *= 2.0 ** torch.randint(0, 3, (t.shape[0], (k + 31) // 32), generator=g).repeat_interleave(32, 1)[:, :k]  # ... or 2 or 4
    got = microscale.product(microscale.quantize(a.to(DEV)), microscale.quantize(b.to(DEV)), dtype=F32, check=True)
    assert torch.equal(got.cpu(), a @ b.T)  # sums below 2^24


@pytest.mark.gpu
def test_product_of_a_tensor_quantizes_it():
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(50, 70, generator=g).to(DEV).half(), microscale.quantize(torch.randn(30, 70, generator=g).to(DEV))
    assert torch.equal(microscale.product(x, w), microscale.product(microscale.quantize(x), w))
    wide = torch.randn(50, 100, generator=g).to(DEV)
    assert torch.equal(microscale.product(wide[:, 7:77], w), microscale.product(wide[:, 7:77].contiguous(), w))


@pytest.mark.gpu
@pytest.mark.parametrize("x", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 700, 1030), (4, 5, 33), (16, 300, 256), (16, 3, 4096), (7, 129, 250), (3, 20_011, 300), (9, 40, 31)])
def test_product_of_a_few_rows_quantizes_them_on_the_way(m, n, k, x):
    g = torch.Generator().manual_seed(m)
    t = (torch.randn(m, k + 8, generator=g) * torch.exp(3 * torch.randn(m, 1, generator=g))).to(x).to(DEV)
    w = microscale.quantize(torch.randn(n, k, generator=g).to(DEV))
    for v in (t[:, :k], t[:, 3:k + 3], t[:, :k].contiguous()):
        got = microscale.product(v, w, dtype=F32, check=True)
        want = microscale.product(microscale.quantize(v), w, dtype=F32)
        # the same codes and scales; sums over K may run in another order
        va, vb = (ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), k) for q in (microscale.quantize(v), w))
        err = (k + 2) * 2 * ref.U * (np.abs(va) @ np.abs(vb).T)
        ref.close(got, va @ vb.T, err)
        ref.close(got, ref.f64(want), 2 * err)
    bad = t[:, :k].clone()
    bad[0, k // 2] = float("inf")
    assert torch.isnan(microscale.product(bad, w)[0]).all() and torch.isfinite(microscale.product(bad, w)[1:]).all()


@pytest.mark.gpu
def test_product_passes_nan_and_range():
    a, b = torch.randn(140, 96), torch.randn(33, 96)
    a[3, 40], b[7, 70] = float("nan"), float("inf")
    got = microscale.product(a.to(DEV), microscale.quantize(b.to(DEV)), dtype=F32).cpu()
    want = torch.zeros(140, 33, dtype=torch.bool)
    want[3], want[:, 7] = True, True
    assert torch.equal(torch.isnan(got), want)
    big = microscale.quantize(torch.full((2, 32), 2.0 ** 100, device=DEV))
    assert torch.isinf(microscale.product(big, big, dtype=F32)).all()
    half = microscale.quantize(torch.full((2, 32), 2.0 ** 10, device=DEV))
    assert torch.isinf(microscale.product(half, half, dtype=F16)).all()
    assert (microscale.product(half, half, dtype=F32) == 2.0 ** 25).all()


@pytest.mark.gpu
def test_product_of_nothing():
    none, some = microscale.quantize(torch.zeros(0, 40, device=DEV)), microscale.quantize(torch.ones(3, 40, device=DEV))
    assert microscale.product(none, some).shape == (0, 3) and microscale.product(some, none).shape == (3, 0)
    assert none.dequantize().shape == (0, 40)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    x, w = torch.randn(200, 512, device=DEV).bfloat16(), microscale.quantize(torch.randn(300, 512, device=DEV))
    want = microscale.product(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = microscale.product(x, w)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = microscale.product(x, w)
        back = microscale.quantize(x).dequantize()
    x.mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want * 2) and torch.equal(back, microscale.quantize(x).dequantize())


def test_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        microscale.quantize(torch.zeros(2, 3))
    with pytest.raises(ValueError, match="x: dtype"):
        microscale.quantize(torch.zeros(2, 3, dtype=torch.float64))
    with pytest.raises(ValueError, match="codes"):
        microscale.Micro4(torch.zeros(2, 3), torch.zeros(2, 4), 3)
    with pytest.raises(ValueError, match="Micro4"):
        microscale.product(torch.zeros(2, 3), torch.zeros(2, 3))


@pytest.mark.gpu
def test_refusals_on_the_device():
    q = microscale.quantize(torch.ones(4, 40, device=DEV))
    other = microscale.quantize(torch.ones(4, 41, device=DEV))
    for bad in (lambda: microscale.quantize(torch.ones(4, device=DEV)), lambda: microscale.quantize(torch.ones(4, 0, device=DEV)),
                lambda: q.dequantize(torch.float64), lambda: microscale.product(q, other), lambda: microscale.product(q, q, dtype=torch.int8),
                lambda: microscale.Micro4(q.codes, q.scales, 65), lambda: microscale.Micro4(q.codes[:2], q.scales, 40),
                lambda: microscale.Micro4(q.codes[:, :16], q.scales, 32), lambda: microscale.product(torch.ones(2, 39, device=DEV), q),
                lambda: microscale.product(torch.ones(40, device=DEV), q), lambda: microscale.product(torch.ones(99, 39, device=DEV), q)):
        with pytest.raises(ValueError):
            bad()


def test_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    assert lib.flare_micro_quantize(None, 0, 1, 4, 4, None, None, None) == 1 and b"NULL" in lib.flare_last_error()
    assert lib.flare_micro_quantize(None, 3, 1, 4, 4, None, None, None) == 1 and b"type" in lib.flare_last_error()
    assert lib.flare_micro_dequantize(None, None, 1, 0, None, 0, 4, None) == 1
    assert lib.flare_micro_dequantize(16, 16, 1, 8, 16, 0, 4, None) == 1 and b"overlap" in lib.flare_last_error()
    assert lib.flare_micro_product(None, None) == 1
    a = _lib.ProductArgs(m=1, n=1, k=0)
    assert lib.flare_micro_product(ctypes.byref(a), None) == 1
    a = _lib.ProductArgs(m=1, n=1, k=32, out_stride=1)
    assert lib.flare_micro_product(ctypes.byref(a), None) == 1 and b"NULL" in lib.flare_last_error()
    a = _lib.ProductArgs(m=17, n=1, k=32, out_stride=1, x=16, x_stride=32, b_codes=16, b_scales=16, out=16)
    assert lib.flare_micro_product(ctypes.byref(a), None) == 1 and b"17 rows" in lib.flare_last_error()
    a = _lib.ProductArgs(m=1, n=1, k=32, out_stride=1, a_codes=8, b_codes=16, a_scales=16, b_scales=16, out=16)
    assert lib.flare_micro_product(ctypes.byref(a), None) == 1 and b"aligned" in lib.flare_last_error()


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_blocks_that_share_a_tile_cover_k_and_run_at_once(tmp_path):
    """Over all numbers of stages, tiles and columns; a short K is not shared, a long one is."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flare_b200", "csrc")
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text("""#include <cstdio>
#include "product_plan.h"
using namespace flare;
int main() {
    const int columns[] = {1, 4, 16, 24, 64}, most[] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
    for (int all = 1; all <= 300; ++all)
        for (long long tiles = 1; tiles <= 200; ++tiles)
            for (int c : columns)
                for (int way = 0; way < (c <= 16 ? 6 : 3); ++way) {
                    const bool plain = way > 2;
                    const int S = parts_of_k(all, tiles, c, plain, (Store)(way % 3)), per = part_of_k(all, S);
                    const bool once = S == 1 || tiles <= most[S] || (!plain && per == 2 && tiles * S <= 148);
                    if (S < 1 || S > 8 || !once || (long long)S * per < all || (S > 1 && per % 2)) {
                        std::printf("%d stages, %lld tiles, %d columns, way %d: %d parts of %d;", all, tiles, c, way, S, per);
                        return 1;
                    }
                }
    std::printf("%d %d %d %d %d", parts_of_k(4, 8, 64, false, Store::columns), parts_of_k(2, 32, 4, true, Store::columns),
                parts_of_k(16, 32, 4, true, Store::columns), parts_of_k(32, 8, 64, false, Store::columns),
                parts_of_k(32, 16, 64, false, Store::rows_of_16));
}
""")
    subprocess.run(["g++", "-std=c++17", "-I", csrc, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "1 1 4 8 6", out.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("stages", [2, 6, 7, 10, 14, 16, 18, 26])
@pytest.mark.parametrize("n", [65, 1900, 2600, 3300])
@pytest.mark.parametrize("m", [2, 40, 61])
def test_product_of_parts_of_k_is_exact(m, n, stages):
    """1 to 8 blocks share a tile, some without a stage of their own; K ends inside one.  Small whole numbers, so equality."""
    g = torch.Generator().manual_seed(stages)
    k = 256 * stages - 37
    a, b = (torch.randint(-2, 3, (r, k), generator=g).float() for r in (m, n))
    for t in (a, b):
        t[:, ::32] = 4.0  # every block's scale is 1
    want = a @ b.T  # sums below 2^24
    w = microscale.quantize(b.to(DEV))
    for x in (a.to(DEV), microscale.quantize(a.to(DEV))):
        assert torch.equal(microscale.product(x, w, dtype=F32, check=True).cpu(), want)
    assert torch.equal(microscale.product(w, x, dtype=F32, check=True).cpu(), want.T)  # the tiles' rows are the output's

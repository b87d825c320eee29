"""Row lookup with scaling and its gradient against a 64-bit restatement (GPU), refusals (CPU)."""
import ctypes
import os

import numpy as np
import pytest
import torch

import ops_reference as ref
from flare_b200 import _lib, embedding

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _case(rows, width, n, table=F16, index=torch.int32, weight=True, seed=0, hot=0.0, empty=0.2, pad=0, shape=None):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(rows, width + pad, generator=g).to(table)[:, :width]
    idx = torch.randint(0, max(rows, 1), (n,), generator=g)
    idx = torch.where(torch.rand(n, generator=g) < hot, idx % 2, idx)
    idx = torch.where(torch.rand(n, generator=g) < empty, -1, idx).to(index)
    w = torch.rand(n, generator=g) + 0.1 if weight else None
    if shape:
        idx, w = idx.reshape(shape), None if w is None else w.reshape(shape)
    return t, idx, w


def _to(*ts):
    # a strided table keeps its strides on the device
    return [None if t is None else t.to(DEV) if t.is_contiguous() else
            torch.as_strided(torch.empty(t.shape[0] * t.stride(0), dtype=t.dtype, device=DEV), t.shape, t.stride()).copy_(t)
            for t in ts]


FORWARD = [
    dict(rows=1, width=1, n=1), dict(rows=7, width=3, n=5, table=F32), dict(rows=50, width=96, n=1000),
    dict(rows=50, width=96, n=33, table=BF16, index=torch.int64, weight=False), dict(rows=300, width=32, n=257, table=F32),
    dict(rows=20, width=1023, n=40, table=BF16), dict(rows=20, width=2050, n=13), dict(rows=9, width=12, n=100),
    dict(rows=9, width=96, n=100, pad=8), dict(rows=9, width=96, n=100, pad=3), dict(rows=9, width=6, n=100, pad=1, table=F32),
    dict(rows=40, width=96, n=48, shape=(16, 3)), dict(rows=3, width=8, n=20, empty=1.0), dict(rows=9, width=150, n=70, pad=1),
    dict(rows=30, width=771, n=50, table=F32, weight=False), dict(rows=30, width=64, n=50, pad=1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("c", FORWARD, ids=str)
@pytest.mark.parametrize("out", [None, F32, F16, BF16])
def test_lookup(c, out):
    t, idx, w = _case(**c)
    tg, ig, wg = _to(t, idx, w)
    got = embedding.lookup(tg, ig, wg, 0.75, dtype=out)
    assert got.dtype == (out or t.dtype) and got.shape == idx.shape + (t.shape[1],)
    want = ref.lookup(ref.f64(t), idx.numpy(), ref.f64(w), 0.75).reshape(got.shape)
    ref.close(got, want, 2 * ref.U * np.abs(want))
    assert not got[(ig < 0)].any()


@pytest.mark.gpu
def test_lookup_rows_that_do_not_exist_give_zeros_whatever_they_are_multiplied_with():
    t = torch.full((4, 5), float("inf"), device=DEV)
    idx = torch.tensor([-1, 4, 2, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    w = torch.tensor([float("nan"), float("inf"), 1.0, 1.0, 1.0], device=DEV)
    got = embedding.lookup(t, idx, w)
    assert torch.isinf(got[2]).all() and not got[[0, 1, 3, 4]].any()
    big = torch.tensor([2 ** 40, -2 ** 40, 1], device=DEV)
    got = embedding.lookup(torch.ones(4, 5, device=DEV), big)
    assert not got[:2].any() and (got[2] == 1).all()
    dt, dw = embedding.lookup_backward(torch.ones(5, 5, device=DEV), t, idx, w)
    assert (dt[2] == 1).all() and not dt[[0, 1, 3]].any() and torch.isinf(dw[2]) and not dw[[0, 1, 3, 4]].any()


@pytest.mark.gpu
def test_lookup_of_nothing():
    t = torch.ones(4, 5, device=DEV)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert embedding.lookup(t, none).shape == (0, 5)
    dt, dw = embedding.lookup_backward(torch.empty(0, 5, device=DEV), t, none, need_weight=True)
    assert dt.shape == (4, 5) and not dt.any() and dw.shape == (0,)
    idx = torch.tensor([0, -1], device=DEV)
    empty = torch.empty(0, 5, device=DEV)
    assert not embedding.lookup(empty, idx).any()
    dt, dw = embedding.lookup_backward(torch.ones(2, 5, device=DEV), empty, idx, need_weight=True)
    assert dt.shape == (0, 5) and not dw.any()


BACKWARD = [
    dict(rows=1, width=1, n=1, empty=0.0), dict(rows=5, width=3, n=400, table=F32), dict(rows=40, width=96, n=3000),
    dict(rows=5000, width=96, n=700, index=torch.int64), dict(rows=70000, width=8, n=5000, table=F32),
    dict(rows=300, width=37, n=9000, table=BF16, hot=0.8), dict(rows=2, width=96, n=2000, hot=1.0, empty=0.0),
    dict(rows=2, width=64, n=255, empty=0.0), dict(rows=1, width=64, n=256, empty=0.0), dict(rows=1, width=64, n=257, empty=0.0),
    dict(rows=3, width=260, n=5000, table=F32, weight=False), dict(rows=9, width=1023, n=700, table=BF16),
    dict(rows=50, width=4, n=4097, table=F32), dict(rows=12, width=16, n=64, empty=1.0), dict(rows=9, width=24, n=100, pad=8),
    dict(rows=40, width=96, n=48, shape=(16, 3)), dict(rows=100_000, width=5, n=17_000), dict(rows=300, width=96, n=16_383, hot=0.5),
    dict(rows=2000, width=20, n=40_000, table=F32, hot=0.3), dict(rows=70, width=200, n=3000), dict(rows=50, width=192, n=2000, table=BF16),
    dict(rows=50, width=256, n=900, pad=8), dict(rows=50, width=128, n=900, table=F32), dict(rows=50, width=132, n=900, table=F32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("c", BACKWARD, ids=str)
def test_lookup_backward(c):
    t, idx, w = _case(**c)
    g = torch.Generator().manual_seed(1)
    dout = torch.randn(*idx.shape, t.shape[1], generator=g).to(t.dtype)
    tg, ig, wg, dg = _to(t, idx, w, dout)
    dt, dw = embedding.lookup_backward(dg, tg, ig, wg, 0.75, need_weight=True)
    want, err, wantw, errw = ref.lookup_backward(ref.f64(dout), ref.f64(t), idx.numpy(), ref.f64(w), 0.75)
    assert dt.dtype == dw.dtype == F32 and dw.shape == idx.shape
    ref.close(dt, want, err, "dtable")
    ref.close(dw.reshape(-1), wantw, errw, "dweight")
    again, _ = embedding.lookup_backward(dg, tg, ig, wg, 0.75)
    assert torch.equal(again, dt)  # a fixed order of every sum
    only, none = embedding.lookup_backward(dg, tg, ig, wg, 0.75, need_weight=False)
    assert none is None and torch.equal(only, dt)
    none, onlyw = embedding.lookup_backward(dg, tg, ig, wg, 0.75, need_table=False, need_weight=True)
    assert none is None
    ref.close(onlyw.reshape(-1), wantw, errw, "dweight alone")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1023, 1025, 4097, 8192, 8193, 16_384, 16_385, 32_769, 100_000, 160_000, 400_000, 700_000])
def test_lookup_backward_many_equal_entries(n):
    """Rows of 0, 1 and thousands of entries, runs that end inside a chunk: whole numbers sum exactly, so equality."""
    g = torch.Generator().manual_seed(n)
    idx = torch.cat([torch.zeros(n // 2, dtype=torch.int64), torch.randint(1, 5, (n // 4,), generator=g),
                     torch.arange(7, 7 + n - n // 2 - n // 4)])[torch.randperm(n, generator=g)]
    dout = torch.randint(-3, 4, (n, 10), generator=g).float()
    rows = int(idx.max()) + 3
    dt, _ = embedding.lookup_backward(dout.to(DEV), torch.zeros(rows, 10, device=DEV), idx.to(DEV))
    want = torch.zeros(rows, 10).index_add_(0, idx, dout)
    assert torch.equal(dt.cpu(), want)


@pytest.mark.gpu
def test_rows_of_no_columns():
    idx = torch.tensor([[0, 2], [-1, 1]], device=DEV)
    table, w = torch.zeros(3, 0, device=DEV), torch.ones(2, 2, device=DEV)
    out = embedding.lookup(table, idx, w)
    assert out.shape == (2, 2, 0)
    dt, dw = embedding.lookup_backward(out, table, idx, w)
    assert dt.shape == (3, 0) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.gpu
def test_gradient_agrees_with_differences():
    t, idx, w = _case(rows=6, width=5, n=20, table=F32)
    g = torch.Generator().manual_seed(2)
    d = torch.randn(20, 5, generator=g)
    tg, ig, wg, dg = _to(t, idx, w, d)
    dt, dw = embedding.lookup_backward(dg, tg, ig, wg, 0.5)
    loss = lambda a, b: float((ref.lookup(a, idx.numpy(), b, 0.5) * ref.f64(d)).sum())  # noqa: E731
    a, b = ref.f64(t), ref.f64(w)
    for p, c in ((0, 0), (3, 4), (5, 2)):
        up, dn = a.copy(), a.copy()
        up[p, c] += 0.5
        dn[p, c] -= 0.5
        # linear in the table: the difference has no error but the 32-bit sum's (at most 20 terms of size 5)
        assert abs(loss(up, b) - loss(dn, b) - float(dt[p, c])) < 22 * ref.U * 100
    for i in (0, 7, 19):
        up, dn = b.copy(), b.copy()
        up[i] += 0.5
        dn[i] -= 0.5
        assert abs(loss(a, up) - loss(a, dn) - float(dw[i])) < 7 * ref.U * 100


@pytest.mark.gpu
def test_broadcast_and_strided_gradients():
    t, idx, _ = _case(rows=6, width=8, n=30, table=F32, empty=0.0)
    tg, ig = _to(t, idx)
    one = torch.ones(1, 1, device=DEV).expand(30, 8)  # the gradient of a sum
    dt, _ = embedding.lookup_backward(one, tg, ig)
    assert torch.equal(dt.cpu(), torch.bincount(idx.long(), minlength=6).float()[:, None].expand(6, 8))
    wide = torch.randn(30, 20, device=DEV)
    a, _ = embedding.lookup_backward(wide[:, 3:11], tg, ig)
    b, _ = embedding.lookup_backward(wide[:, 3:11].contiguous(), tg, ig)
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    t, idx, w = _case(rows=5000, width=96, n=20_000)
    tg, ig, wg = _to(t, idx, w)
    d = torch.randn(20_000, 96, device=DEV).half()
    out, (dt, dw) = embedding.lookup(tg, ig, wg), embedding.lookup_backward(d, tg, ig, wg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2, (dt2, dw2) = embedding.lookup(tg, ig, wg), embedding.lookup_backward(d, tg, ig, wg)
    torch.cuda.synchronize()
    assert torch.equal(out, out2) and torch.equal(dt, dt2) and torch.equal(dw, dw2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out3, (dt3, dw3) = embedding.lookup(tg, ig, wg), embedding.lookup_backward(d, tg, ig, wg)
    ig.copy_(ig.flip(0))
    d.copy_(d.flip(0))
    wg.copy_(wg.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out3, out.flip(0)) and torch.equal(dw3, dw.flip(0))
    eager, _ = embedding.lookup_backward(d, tg, ig, wg)
    assert torch.equal(dt3, eager)


def test_refusals():
    t, idx, w = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    with pytest.raises(ValueError, match="CUDA"):
        embedding.lookup(t, idx, w)
    with pytest.raises(ValueError, match="table: dtype"):
        embedding.lookup(t.double(), idx)
    with pytest.raises(ValueError, match="expected a torch.Tensor"):
        embedding.lookup([1.0], idx)
    with pytest.raises(ValueError, match="table"):
        embedding.lookup_backward(torch.zeros(3, 8), object(), idx)


@pytest.mark.gpu
def test_refusals_on_the_device():
    t, idx, w = torch.zeros(4, 8, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, device=DEV)
    d = torch.zeros(3, 8, device=DEV)
    for bad in (lambda: embedding.lookup(t[0], idx), lambda: embedding.lookup(t, idx.float()), lambda: embedding.lookup(t, idx.cpu()),
                lambda: embedding.lookup(t, idx, w[:2]), lambda: embedding.lookup(t, idx, w.half()),
                lambda: embedding.lookup(t, idx, dtype=torch.float64), lambda: embedding.lookup_backward(d[:2], t, idx),
                lambda: embedding.lookup_backward(d.double(), t, idx), lambda: embedding.lookup_backward(d[:, :4], t, idx)):
        with pytest.raises(ValueError):
            bad()


def test_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    assert lib.flare_lookup(None, None) == 1 and b"NULL" in lib.flare_last_error()
    a = _lib.LookupArgs(n=1, rows=1, width=4, out_stride=4, table_type=7)
    assert lib.flare_lookup(ctypes.byref(a), None) == 1 and b"table type" in lib.flare_last_error()
    a.table_type = 0
    assert lib.flare_lookup(ctypes.byref(a), None) == 1 and b"NULL buffer" in lib.flare_last_error()
    a.n = 0
    assert lib.flare_lookup(ctypes.byref(a), None) == 0
    b = _lib.LookupGradArgs(n=2 ** 31, rows=1, width=4)
    assert lib.flare_lookup_backward(ctypes.byref(b), None) == 1
    b = _lib.LookupGradArgs(n=5, rows=3, width=4, dout=16, index=16, dtable=16, dout_stride=4)
    assert lib.flare_lookup_backward(ctypes.byref(b), None) == 1 and b"workspace" in lib.flare_last_error()
    assert lib.flare_lookup_workspace(3, 5, 4) > 0 and lib.flare_lookup_workspace(0, 5, 4) == 0


def test_one_bound_on_the_number_of_entries():
    lib = _lib.load()
    for n, why in ((embedding.MAX_ENTRIES, b"NULL buffer"), (embedding.MAX_ENTRIES + 1, b"entries")):
        a = _lib.LookupGradArgs(n=n, rows=1, width=4)
        assert lib.flare_lookup_backward(ctypes.byref(a), None) == 1 and why in lib.flare_last_error()
    for rows, why in ((embedding.MAX_ROWS, b"NULL buffer"), (embedding.MAX_ROWS + 1, b"rows")):
        a = _lib.LookupGradArgs(n=1, rows=rows, width=4)
        assert lib.flare_lookup_backward(ctypes.byref(a), None) == 1 and why in lib.flare_last_error()
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "flare_b200.h")
    text = " ".join(open(header).read().replace("\n *", " ").split())
    assert f"rows < 2^31 - {2 ** 31 - 1 - embedding.MAX_ROWS}, n < 2^31 - {2 ** 31 - 1 - embedding.MAX_ENTRIES}." in text

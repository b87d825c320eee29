"""The operators where 32-bit numbers end and where nothing has run before: outputs of more than one launch, elements past 2^31,
a first call inside a graph's capture.  Whole numbers of few bits, so that results are exact in any order."""
import os
import subprocess
import sys

import pytest
import torch

from flare_b200 import embedding, microscale, recurrence

DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def _give_memory_back():
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


def _ends(n, width=1 << 16):
    """Slices of [0, n): its ends and the stretch around every multiple of 2^30."""
    at = {0, n - width} | {k - width // 2 for k in range(2 ** 30, n, 2 ** 30)}
    return [slice(max(0, a), min(n, a + width)) for a in sorted(at)]


@pytest.mark.gpu
def test_lookup_of_more_entries_than_a_launch_takes():
    n = 2 ** 30 + 1000
    table = torch.arange(1000, device=DEV, dtype=F16)[:, None]
    idx = torch.randint(-1, 1000, (n,), dtype=torch.int32, device=DEV)
    out = embedding.lookup(table, idx)
    for s in _ends(n):
        i = idx[s].long()
        assert torch.equal(out[s, 0], torch.where(i < 0, 0, table[i.clamp(min=0), 0]))


@pytest.mark.gpu
def test_lookup_of_a_table_past_2_to_the_31_elements():
    rows, width, n = 22_400_000, 96, 4000
    assert rows * width > 2 ** 31
    table = torch.empty(rows, width, dtype=F16, device=DEV)
    table.copy_((torch.arange(rows, device=DEV) % 251).to(F16)[:, None])
    table[:, 1] = 1.0
    g = torch.Generator(device=DEV).manual_seed(1)
    idx = torch.cat([torch.randint(rows - 3000, rows, (n // 2,), device=DEV, generator=g),
                     torch.randint(0, rows, (n // 2,), device=DEV, generator=g)])
    out = embedding.lookup(table, idx)
    assert torch.equal(out, table[idx])
    dout = torch.randint(-3, 4, (n, width), device=DEV, generator=g).to(F16)
    dt, dw = embedding.lookup_backward(dout, table, idx, need_weight=True)
    named, inverse = idx.unique(return_inverse=True)
    want = torch.zeros(named.numel(), width, device=DEV).index_add_(0, inverse, dout.float())
    assert torch.equal(dt[named], want)
    assert int(dt.any(1).sum()) == int(want.any(1).sum())  # every other row is zero
    assert torch.equal(dw, (dout.float() * table[idx].float()).sum(1))  # sums below 96 * 3 * 251


@pytest.mark.gpu
def test_recurrence_past_2_to_the_31_elements():
    B, T, D = 1_420_000, 16, 96
    assert B * T * D > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randint(-2, 3, (T, B, D), device=DEV, generator=g, dtype=torch.int8).to(F16).transpose(0, 1)
    gate = torch.randint(0, 2, (T, B, 1), device=DEV, generator=g).float().transpose(0, 1)
    dlast = torch.randint(-2, 3, (B, D), device=DEV, generator=g).float()
    _, last, saved = recurrence.scan(gate, x, reverse=True, states=False, training=True)
    dgate, dx, _ = recurrence.scan_backward(gate, x, saved, None, dlast, reverse=True)
    for s in (slice(0, 500), slice(B - 500, B)):
        xs, gs = x[s].contiguous(), gate[s].contiguous()
        _, want, sv = recurrence.scan(gs, xs, reverse=True, states=False, training=True)
        wg, wx, _ = recurrence.scan_backward(gs, xs, sv, None, dlast[s].contiguous(), reverse=True)
        assert torch.equal(last[s], want) and torch.equal(dgate[s], wg) and torch.equal(dx[s], wx)
        h = torch.zeros(500, D, device=DEV)
        for t in range(T - 1, -1, -1):
            h = gs[:, t] * h + xs[:, t].float()
        assert torch.equal(last[s], h)


@pytest.mark.gpu
def test_quantize_of_more_rows_than_a_launch_takes():
    rows = 2 ** 28 + 100  # four pieces a row
    level = torch.tensor([1.0, -1.5, 2.0, 3.0, 0.0, -8.0], device=DEV, dtype=F16)  # alone in their blocks: exact
    x = level.repeat(rows // 6 + 1)[:rows, None]
    back = microscale.quantize(x).dequantize()
    for s in _ends(rows) + [slice(rows // 2, rows // 2 + 65536)]:
        assert torch.equal(back[s], x[s])


@pytest.mark.gpu
def test_product_past_2_to_the_31_outputs():
    m, n, k = 70_000, 31_000, 40
    assert m * n > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(3)
    a, b = (torch.randint(-1, 2, (r, k), device=DEV, generator=g).float() for r in (m, n))
    a[:, ::32] = b[:, ::32] = 4.0
    out = microscale.product(microscale.quantize(a), microscale.quantize(b), dtype=F16, check=True)
    for s in (slice(0, 300), slice(m - 300, m), slice(2 ** 31 // n - 100, 2 ** 31 // n + 100)):
        assert torch.equal(out[s].float(), a[s] @ b.T)  # whole numbers below 100


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4000, 16_384, 16_385, 70_000])
@pytest.mark.parametrize("rows", [1, 5, 1023, 1024, 2 ** 20 + 5, embedding.MAX_ROWS])
def test_lookup_gradient_of_every_number_of_digits(rows, n):
    """Row numbers of 1 to 31 bits, up to the most rows there may be."""
    g = torch.Generator(device=DEV).manual_seed(4)
    idx = torch.randint(0, rows, (n,), device=DEV, generator=g)
    idx[::7], idx[1::7], idx[3] = rows - 1, 0, -1
    idx[5::50] = rows  # no row
    dout = torch.randint(-3, 4, (n, 1), device=DEV, generator=g).float()
    dt, _ = embedding.lookup_backward(dout, torch.empty(rows, 1, dtype=F16, device=DEV), idx)
    some = (idx >= 0) & (idx < rows)
    named, inverse = idx[some].unique(return_inverse=True)
    want = torch.zeros(named.numel(), 1, device=DEV).index_add_(0, inverse, dout[some])
    assert torch.equal(dt[named], want)
    dt[named] = 0
    assert not dt.any()


FIRST = """
import torch
from flare_b200 import embedding, microscale, recurrence
torch.manual_seed(0)
d = "cuda"
table, idx, w = torch.randn({rows}, 96, device=d).half(), torch.randint(-1, {rows}, ({n},), device=d), torch.rand({n}, device=d)
dout = torch.randn({n}, 96, device=d).half()
gate, x, s = torch.rand(1, 4000, 64, device=d), torch.randn(1, 4000, 64, device=d), torch.randn(1, 64, device=d)
layer = microscale.Micro4(torch.randint(0, 256, (70, 48), device=d).byte(), torch.full((70, 4), 127, device=d).byte(), 96)
def run():
    out = [embedding.lookup(table, idx, w), *embedding.lookup_backward(dout, table, idx, w)]
    h, last, saved = recurrence.scan(gate, x, s, training=True)
    out += [h, last, *recurrence.scan_backward(gate, x, saved, x, s, s), recurrence.step(gate[0], x[0], x[0].clone())]
    q = microscale.quantize(table)
    return out + [q.dequantize(), microscale.product(q, layer), microscale.product(table[:5], layer), embedding.lookup(q, idx)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
torch.cuda.synchronize()
want = run()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(bool(a.any()) for a in got)
print("same")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(500, 3000), (50_000, 40_000)])
def test_first_calls_are_captured(rows, n):
    """In a process of its own, in which no operator has run before the capture."""
    r = subprocess.run([sys.executable, "-c", FIRST.format(rows=rows, n=n)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]

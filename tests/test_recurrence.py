"""The gated linear recurrence, its gradient and its single step against a 64-bit restatement (GPU), refusals (CPU)."""
import ctypes

import numpy as np
import pytest
import torch

import ops_reference as ref
from flare_b200 import _lib, recurrence

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _case(layout, B, T, D, G, x=F32, gate=None, seed=0, cuts=None, pad=0):
    """Tensors on the device; time: step-major in memory; packed: T rows in all, cut at random or at `cuts`."""
    g = torch.Generator().manual_seed(seed)
    lead = {"batch": (B, T), "time": (T, B), "packed": (T,)}[layout]
    a = torch.sigmoid(torch.randn(*lead, G, generator=g) * 2 + 1.5)
    a = torch.where(torch.rand(*lead, G, generator=g) < 0.05, 0.0, a).to(gate or x)  # a gate of 0 ends what came before
    v, dh = (torch.randn(*lead, D + pad, generator=g).to(x)[..., :D] for _ in range(2))
    off = None
    if layout == "packed":
        off = torch.tensor([0] + sorted(torch.randint(0, T + 1, (B,), generator=g).tolist()) if cuts is None else cuts,
                           dtype=torch.int32)
    s, dl = torch.randn(B, D, generator=g), torch.randn(B, D, generator=g)
    back = (lambda t: t.transpose(0, 1)) if layout == "time" else (lambda t: t)

    def dev(t):  # with its strides
        full = torch.empty(t.shape[:-1] + (D + pad,), dtype=t.dtype, device=DEV)[..., :t.shape[-1]] if pad and t.shape[-1] == D else \
            torch.empty(t.shape, dtype=t.dtype, device=DEV)
        return back(full.copy_(t))

    return dict(gate=dev(a), x=dev(v), dh=dev(dh), offsets=None if off is None else off.to(DEV), state=s.to(DEV), dlast=dl.to(DEV))


def _check(c, reverse=False, state=True, use_dh=True, use_dlast=True):
    s = c["state"] if state else None
    dh, dl = c["dh"] if use_dh else None, c["dlast"] if use_dlast else None
    off = None if c["offsets"] is None else c["offsets"].cpu().numpy()
    want = ref.scan(ref.f64(c["gate"]), ref.f64(c["x"]), ref.f64(s), off, reverse, ref.f64(dh), ref.f64(dl))
    kw = dict(offsets=c["offsets"], reverse=reverse)
    h, last, saved = recurrence.scan(c["gate"], c["x"], s, training=True, **kw)
    dg, dx, ds = recurrence.scan_backward(c["gate"], c["x"], saved, dh, dl, s, **kw)
    assert h.dtype == dx.dtype == c["x"].dtype and dg.dtype == c["gate"].dtype and last.dtype == F32
    assert (ds is None) == (s is None)
    for name, got in dict(h=h, last=last, dgate=dg, dx=dx, dstate=ds).items():
        if got is not None:
            ref.close(got, *want[name], name)
    h2, last2, none = recurrence.scan(c["gate"], c["x"], s, states=False, **kw)
    assert h2 is None and none is None and torch.equal(last2, last)
    again = recurrence.scan_backward(c["gate"], c["x"], saved, dh, dl, s, **kw)
    assert torch.equal(again[0], dg) and torch.equal(again[1], dx)
    return h, last, dg, dx, ds


SHAPES = [
    # layout, sequences, steps, width, groups
    ("batch", 1, 1, 1, 1), ("batch", 3, 16, 4, 1), ("batch", 3, 17, 4, 4), ("batch", 2, 15, 96, 1), ("batch", 5, 33, 6, 2),
    ("time", 50, 16, 96, 1), ("time", 7, 42, 4, 1), ("time", 3, 100, 64, 64), ("batch", 1, 1000, 32, 32),
    ("batch", 1, 5000, 64, 64), ("batch", 2, 2500, 10, 1), ("batch", 1, 4099, 40, 2), ("time", 4, 300, 70, 1),
    ("batch", 2, 40, 160, 1), ("batch", 2, 40, 321, 1), ("batch", 1, 700, 260, 2), ("batch", 300, 20, 33, 11),
    ("batch", 2, 20, 1300, 1), ("time", 300, 31, 96, 1), ("batch", 130, 18, 100, 5), ("packed", 300, 2000, 24, 1),
    ("packed", 9, 200, 8, 2), ("packed", 5, 3000, 16, 16), ("packed", 40, 100, 5, 1), ("packed", 3, 9000, 130, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32)], ids=["f32", "bf16", "f16-f32"])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan_and_gradient(shape, reverse, types):
    _check(_case(*shape, x=types[0], gate=types[1]), reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("opts", [dict(state=False), dict(use_dh=False), dict(use_dlast=False), dict(use_dh=False, use_dlast=False)],
                         ids=str)
@pytest.mark.parametrize("shape", [("time", 5, 40, 12, 3), ("batch", 1, 3000, 16, 16), ("packed", 6, 500, 8, 1)], ids=str)
def test_optional_inputs(shape, opts):
    _check(_case(*shape, x=BF16), True, **opts)


@pytest.mark.gpu
@pytest.mark.parametrize("cuts", [[0, 0, 0, 0], [0, 50, 50, 50], [7, 9, 9, 40], [0, 16, 32, 33], [50, 50], [0]], ids=str)
@pytest.mark.parametrize("reverse", [False, True])
def test_packed_empty_sequences_and_rows_of_none(cuts, reverse):
    c = _case("packed", len(cuts) - 1, 50, 12, 3, cuts=cuts)
    h, last, dg, dx, ds = _check(c, reverse)
    out = torch.ones(50, dtype=torch.bool)
    for a, b in zip(cuts[:-1], cuts[1:]):
        out[a:b] = False
        if a == b:
            s = cuts[:-1].index(a) if cuts.count(a) == 2 else None
            if s is not None:
                assert torch.equal(last[s], c["state"][s]) and torch.equal(ds[s], c["dlast"][s])
    assert not h[out.to(DEV)].any() and not dg[out.to(DEV)].any() and not dx[out.to(DEV)].any()


@pytest.mark.gpu
def test_packed_rows_of_none_are_not_read():
    c = _case("packed", 2, 60, 8, 8, cuts=[3, 20, 44])
    want = recurrence.scan(c["gate"], c["x"], c["state"], c["offsets"], training=True)
    for t in (c["gate"], c["x"], c["dh"]):
        t[:3] = float("nan")
        t[44:] = float("inf")
    got = recurrence.scan(c["gate"], c["x"], c["state"], c["offsets"], training=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dg, dx, ds = recurrence.scan_backward(c["gate"], c["x"], got[2], c["dh"], c["dlast"], c["state"], c["offsets"])
    assert torch.isfinite(dg).all() and torch.isfinite(dx).all() and torch.isfinite(ds).all()


@pytest.mark.gpu
def test_packed_equals_dense():
    B, T, D = 6, 37, 24
    c = _case("batch", B, T, D, 3, x=BF16)
    off = torch.arange(B + 1, dtype=torch.int64, device=DEV) * T
    a = recurrence.scan(c["gate"], c["x"], c["state"], reverse=True)
    b = recurrence.scan(c["gate"].reshape(B * T, 3), c["x"].reshape(B * T, D), c["state"], off, reverse=True)
    assert torch.equal(a[0].reshape(B * T, D), b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_offsets_outside_the_rows_stay_inside():
    c = _case("packed", 3, 40, 8, 8, cuts=[-5, 10, 90, 20])
    h, last, saved = recurrence.scan(c["gate"], c["x"], c["state"], c["offsets"], training=True)
    recurrence.scan_backward(c["gate"], c["x"], saved, c["dh"], c["dlast"], c["state"], c["offsets"])
    torch.cuda.synchronize()
    want = recurrence.scan(c["gate"][:10], c["x"][:10], c["state"][:1], torch.tensor([0, 10], device=DEV))
    assert torch.equal(last[0], want[1][0])


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,steps", [(0, 5), (3, 0), (0, 0)])
def test_nothing_to_step(seqs, steps):
    x, g = torch.zeros(seqs, steps, 4, device=DEV), torch.zeros(seqs, steps, 1, device=DEV)
    s, dl = torch.randn(seqs, 4, device=DEV), torch.randn(seqs, 4, device=DEV)
    h, last, saved = recurrence.scan(g, x, s, training=True)
    assert h.shape == x.shape and torch.equal(last, s)
    dg, dx, ds = recurrence.scan_backward(g, x, saved, None, dl, s)
    assert dg.shape == g.shape and dx.shape == x.shape and torch.equal(ds, dl)
    _, last, _ = recurrence.scan(g, x)
    assert not last.any()


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 2, 3, 8])
@pytest.mark.parametrize("x", [F32, F16])
def test_padded_rows(pad, x):
    _check(_case("batch", 3, 50, 24, 4, x=x, pad=pad))
    _check(_case("time", 3, 50, 24, 24, x=x, pad=pad), True)


@pytest.mark.gpu
def test_strides_that_are_copied_or_broadcast():
    c = _case("batch", 3, 20, 8, 4)
    x = c["x"].permute(0, 2, 1).contiguous().permute(0, 2, 1)  # channels apart
    a, b = recurrence.scan(c["gate"], x, c["state"]), recurrence.scan(c["gate"], c["x"], c["state"])
    assert torch.equal(a[0], b[0])
    g = c["gate"][:, :1].expand(3, 20, 4)  # one gate for all steps
    a, b = recurrence.scan(g, c["x"], training=True), recurrence.scan(g.contiguous(), c["x"])
    assert torch.equal(a[0], b[0])
    da = recurrence.scan_backward(g, c["x"], a[2], c["dh"][:, :1].expand(3, 20, 8), None)
    db = recurrence.scan_backward(g.contiguous(), c["x"], a[2], c["dh"][:, :1].expand(3, 20, 8).contiguous(), None)
    assert torch.equal(da[0], db[0]) and torch.equal(da[1], db[1])


@pytest.mark.gpu
def test_gates_above_one_over_a_state_of_zero():
    """200 gates of 2 leave the range of a float in product; a state that is 0 until the last steps stays 0."""
    x = torch.zeros(1, 200, 4, device=DEV)
    x[:, 198] = 1.0
    h, last, _ = recurrence.scan(torch.full((1, 200, 1), 2.0, device=DEV), x)
    assert not h[:, :198].any() and (h[:, 198] == 1).all() and (last == 2).all()


@pytest.mark.gpu
def test_gradient_agrees_with_differences():
    c = _case("batch", 2, 25, 6, 2)
    out = _check(c)
    a = {k: ref.f64(c[k]) for k in ("gate", "x", "state", "dh", "dlast")}

    def loss(**over):
        v = a | over
        r = ref.scan(v["gate"], v["x"], v["state"], None, False)
        return (r["h"][0] * v["dh"]).sum() + (r["last"][0] * v["dlast"]).sum()

    eps = 1e-6
    for name, got, at in (("gate", out[2], (0, 3, 1)), ("gate", out[2], (1, 24, 0)), ("x", out[3], (0, 0, 5)), ("x", out[3], (1, 24, 2)),
                          ("state", out[4], (1, 4))):
        up, dn = a[name].copy(), a[name].copy()
        up[at] += eps
        dn[at] -= eps
        want = (loss(**{name: up}) - loss(**{name: dn})) / (2 * eps)
        # 32-bit sums of at most 25 x 3 terms of size 20; the difference quotient's own error is eps^2 and 1e-16 / eps
        assert abs(float(got[at]) - want) < 200 * ref.U * 75 * 20, (name, at)


@pytest.mark.gpu
@pytest.mark.parametrize("B,D,G,x,gate", [(1, 1, 1, F32, F32), (64, 1024, 1024, BF16, BF16), (5, 33, 11, F16, F32), (3, 96, 1, F16, F16)])
def test_step(B, D, G, x, gate):
    c = _case("batch", B, 4, D, G, x=x, gate=gate)
    h, last, _ = recurrence.scan(c["gate"], c["x"], c["state"])
    s, other = c["state"].clone(), torch.empty_like(c["state"])
    for t in range(4):
        assert torch.equal(recurrence.step(c["gate"][:, t], c["x"][:, t], s, out=other), h[:, t])
        assert torch.equal(recurrence.step(c["gate"][:, t], c["x"][:, t], s), h[:, t])
        assert torch.equal(s, other)
    assert torch.equal(s, last)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    c = _case("batch", 1, 3000, 96, 3, x=BF16)

    def both():
        h, last, saved = recurrence.scan(c["gate"], c["x"], c["state"], training=True)
        return (h, last) + recurrence.scan_backward(c["gate"], c["x"], saved, c["dh"], c["dlast"], c["state"])

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(both())
    c["x"].mul_(0.5)
    want = both()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, o))


def test_refusals():
    x, g = torch.zeros(2, 3, 8), torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        recurrence.scan(g, x)
    with pytest.raises(ValueError, match="x: dtype"):
        recurrence.scan(g, x.double())
    with pytest.raises(ValueError):
        recurrence.step(g, x, None)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, g, s = torch.zeros(2, 3, 8, device=DEV), torch.zeros(2, 3, 4, device=DEV), torch.zeros(2, 8, device=DEV)
    off = torch.tensor([0, 3, 6], device=DEV)
    for bad in (lambda: recurrence.scan(g[:, :2], x), lambda: recurrence.scan(g[..., :3], x), lambda: recurrence.scan(g.half(), x),
                lambda: recurrence.scan(g, x, s[:1]), lambda: recurrence.scan(g, x, s.half()), lambda: recurrence.scan(g, x, offsets=off),
                lambda: recurrence.scan(g[0], x[0], offsets=off.float()), lambda: recurrence.scan(g[0], x[0]),
                lambda: recurrence.scan_backward(g, x, torch.zeros(3, device=DEV)), lambda: recurrence.scan_backward(g, x, None),
                lambda: recurrence.scan_backward(g, x, torch.zeros(0, device=DEV), dh=x.half()),
                lambda: recurrence.scan_backward(g, x, torch.zeros(0, device=DEV), dlast=s[:1]),
                lambda: recurrence.step(g[:, 0], x[:, 0], s[:1]), lambda: recurrence.step(g[:, 0], x[:, 0], None)):
        with pytest.raises(ValueError):
            bad()


def test_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    A = _lib.RecurrenceArgs
    for fn in (lib.flare_recurrence_forward, lib.flare_recurrence_backward):
        assert fn(None, None) == 1 and b"NULL" in lib.flare_last_error()
        for a, why in ((A(width=4, groups=3), b"groups"), (A(width=4, groups=4, x_type=1, gate_type=2), b"gates"),
                       (A(width=4, groups=4, x_type=9), b"type"), (A(width=4, groups=4, seqs=2, steps=5), b"NULL"),
                       (A(width=2 ** 20, groups=1, seqs=2 ** 12), b"sequences")):
            assert fn(ctypes.byref(a), None) == 1 and why in lib.flare_last_error(), why
        assert fn(ctypes.byref(A(width=4, groups=4, seqs=0, steps=5)), None) == 0
    assert lib.flare_recurrence_saved(3, 16, 4, 0) == 0 and lib.flare_recurrence_saved(3, 17, 4, 0) == 12


def _dense_args(gate, x, **more):
    B, T, D = x.shape
    return _lib.RecurrenceArgs(gate=gate.data_ptr(), x=x.data_ptr(), seqs=B, steps=T, gate_s=gate.stride(0), gate_t=gate.stride(1),
                               x_s=T * D, x_t=D, h_s=T * D, h_t=D, dh_s=T * D, dh_t=D, dgate_s=gate.stride(0), dgate_t=gate.stride(1),
                               dx_s=T * D, dx_t=D, width=D, groups=gate.shape[2], **more)


def test_c_entry_takes_a_copy_of_a_state_kept_in_place():
    """Blocks that share a sequence all read its state, one writes the new one: in place they need room for a copy."""
    lib = _lib.load()
    x, gate, ends = torch.zeros(1, 5000, 64), torch.zeros(1, 5000, 64), torch.zeros(3, 64)
    p = [t.data_ptr() for t in ends]
    for backward, (old, new) in ((0, ("state", "last")), (1, ("dlast", "dstate"))):
        apart = lib.flare_recurrence_workspace(ctypes.byref(_dense_args(gate, x, **{old: p[0], new: p[1]})), backward)
        place = lib.flare_recurrence_workspace(ctypes.byref(_dense_args(gate, x, **{old: p[0], new: p[0]})), backward)
        assert apart > 0 and place == apart + 4 * 64
        fn = lib.flare_recurrence_backward if backward else lib.flare_recurrence_forward
        for part in (p[0] + 64, p[0] - 4):
            a = _dense_args(gate, x, **{old: p[0], new: part})
            a.dgate = a.dx = a.saved = 16
            assert fn(ctypes.byref(a), None) == 1 and f"{new} overlaps {old}".encode() in lib.flare_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 5000, 64, 64), (1, 5000, 64, 1), (3, 40, 33, 11), (2, 9, 96, 1)], ids=str)
def test_c_entry_keeps_a_state_in_place(shape):
    B, T, D, G = shape
    lib = _lib.load()
    c = _case("batch", *shape)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def call(fn, backward, **more):
        a = _dense_args(c["gate"], c["x"], **{k: v.data_ptr() for k, v in more.items()})
        ws = torch.empty(max(16, lib.flare_recurrence_workspace(ctypes.byref(a), backward)), dtype=torch.uint8, device=DEV)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(fn(ctypes.byref(a), stream), "recurrence")

    h, last, saved = recurrence.scan(c["gate"], c["x"], c["state"], training=True)
    want = recurrence.scan_backward(c["gate"], c["x"], saved, c["dh"], c["dlast"], c["state"])
    h2, saved2, state = torch.empty_like(h), torch.empty_like(saved), c["state"].clone()
    call(lib.flare_recurrence_forward, 0, state=state, last=state, h=h2, saved=saved2)
    assert torch.equal(h2, h) and torch.equal(state, last) and torch.equal(saved2, saved)
    dg, dx, ends = torch.empty_like(c["gate"]), torch.empty_like(c["x"]), c["dlast"].clone()
    call(lib.flare_recurrence_backward, 1, state=c["state"], saved=saved, dh=c["dh"], dlast=ends, dstate=ends, dgate=dg, dx=dx)
    assert torch.equal(dg, want[0]) and torch.equal(dx, want[1]) and torch.equal(ends, want[2])


def test_c_entry_refuses_a_step_over_part_of_its_inputs():
    """Addresses only: whatever is not refused is not run."""
    lib = _lib.load()
    B, D, at = 4, 10, 1 << 20  # last: 160 bytes from `at`

    def why(gate=at - 4096, gate_s=2, groups=2, gate_type=0, x=at + 4096, x_s=D, x_type=0, state=at + 65536):
        a = _lib.RecurrenceArgs(gate=gate, x=x, state=state, last=at, seqs=B, steps=1, gate_s=gate_s, x_s=x_s, width=D, groups=groups,
                                gate_type=gate_type, x_type=x_type, offsets_type=7)  # the check behind these
        assert lib.flare_recurrence_forward(ctypes.byref(a), None) == 1
        return lib.flare_last_error().decode().split(": ")[1]

    free = "unknown offsets type 7"
    for kw, want in ((dict(), free), (dict(state=at), free), (dict(state=at + 4), "last overlaps state"), (dict(x=at), free),
                     (dict(x=at, x_s=12), "last overlaps x"), (dict(x=at + 4), "last overlaps x"), (dict(x=at + 160), free),
                     (dict(x=at - 160), free), (dict(x=at - 156), "last overlaps x"), (dict(x=at, x_type=1), "last overlaps x"),
                     (dict(x=at - 40, x_s=50), free), (dict(x=at - 40, x_s=49), "last overlaps x"), (dict(x=at - 36, x_s=0), "last overlaps x"),
                     (dict(x=at - 40, x_s=0), free), (dict(gate=at), "last overlaps gate"), (dict(gate=at, groups=D, gate_s=D), free),
                     (dict(gate=at - 4 * 8, gate_s=2), free), (dict(gate=at - 4 * 8, gate_s=3), "last overlaps gate")):
        assert why(**kw) == want, kw


@pytest.mark.gpu
def test_step_writes_over_an_input_only_as_a_whole():
    g = torch.Generator().manual_seed(3)
    buf, gate = torch.randn(200, generator=g).to(DEV), torch.rand(4, 2, generator=g).to(DEV)
    state, x = buf[:40].view(4, 10), buf[100:140].view(4, 10)
    for o in (buf[1:41].view(4, 10), buf[30:70].view(4, 10)):
        with pytest.raises(_lib.FlareError, match="last overlaps state"):
            recurrence.step(gate, x, state, out=o)
    with pytest.raises(_lib.FlareError, match="last overlaps x"):
        recurrence.step(gate, x, state, out=buf[90:130].view(4, 10))
    with pytest.raises(_lib.FlareError, match="last overlaps x"):
        recurrence.step(gate, buf[5:45].view(4, 10), state)
    with pytest.raises(_lib.FlareError, match="last overlaps gate"):
        recurrence.step(buf[160:168].view(4, 2), x, state, out=buf[160:].view(4, 10))
    for gt in (gate, torch.rand(4, 10, generator=g).to(DEV)):
        want = recurrence.step(gt, x, state, out=torch.empty_like(state))
        for into in ("state", "x", "gate"):
            t = dict(gate=gt.clone(), x=x.clone(), state=state.clone())
            if t[into].shape == state.shape:
                assert torch.equal(recurrence.step(**t, out=t[into]), want) and torch.equal(t[into], want)
    twice = state.clone()
    assert torch.equal(recurrence.step(gate, twice, twice), recurrence.step(gate, state, state, out=torch.empty_like(state)))

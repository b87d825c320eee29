"""The operators as a caller with a decoder of its own runs them: Render's hits, the hit primitives' descriptor rows, a layer
over them, compositing back to front, and the gradients of the descriptors, the opacities and the background."""
import pytest
import torch

import ops_reference as ref
from flare_b200 import embedding, microscale, recurrence

DEV = "cuda"


def _hits(n, side):
    from flare_b200.renderer import CPyOptiXFLARERenderer
    from flare_b200.scene import camera_rays, make_scene
    sc = make_scene(n, 11).to(DEV)
    O, v = camera_rays(side, side, 60.0, eye=(0.0, 0.0, 3.0))
    r = CPyOptiXFLARERenderer(8, 11.3449, side * side)
    r.SetGeometry(*[t.contiguous() for t in sc.activated()])
    _, hits = r.Render(O.to(DEV), v.to(DEV), torch.zeros(side * side, device=DEV), side * side)
    return sc, r, O.to(DEV), v.to(DEV), hits


def _forward(rows, hits, alpha, W, background):
    """Own decoder: colour = sigmoid(rows W^T); composited from the last hit."""
    colour = torch.sigmoid(rows.to(W.dtype) @ W.T)
    al = torch.where(hits >= 0, alpha, 0.0)
    return colour, al


@pytest.mark.gpu
def test_training_step_outside_the_renderer():
    sc, _, _, _, hits = _hits(2000, 24)
    R = hits.shape[1]
    assert (hits < 0).any() and (hits >= 0).any()
    g = torch.Generator().manual_seed(4)
    W = (torch.randn(4, 96, generator=g) * 0.3).to(DEV)
    alpha, background = (torch.rand(16, R, generator=g) * 0.9).to(DEV), torch.rand(R, 4, generator=g).to(DEV)
    dC = torch.randn(R, 4, generator=g).to(DEV)

    rows = embedding.lookup(sc.cond, hits, scale=2.0, dtype=torch.float32)
    colour, al = _forward(rows, hits, alpha, W, background)
    gate, x = (1.0 - al)[..., None].transpose(0, 1), (al[..., None] * colour).transpose(0, 1)
    _, C, saved = recurrence.scan(gate, x, background, reverse=True, states=False, training=True)
    dgate, dx, dbg = recurrence.scan_backward(gate, x, saved, None, dC, background, reverse=True)
    dx, dgate = dx.transpose(0, 1), dgate.transpose(0, 1)[..., 0]
    dalpha = torch.where(hits >= 0, (dx * colour).sum(-1) - dgate, 0.0)
    drows = (al[..., None] * dx * colour * (1 - colour)) @ W
    dcond, _ = embedding.lookup_backward(drows, sc.cond, hits, scale=2.0)

    E = sc.cond.double().cpu().requires_grad_()
    a64, b64, h = alpha.double().cpu().requires_grad_(), background.double().cpu().requires_grad_(), hits.cpu().long()
    col = torch.sigmoid(2.0 * E[h.clamp(min=0)] @ W.double().cpu().T)
    am = torch.where(h >= 0, a64, 0.0)
    acc = b64
    for k in range(15, -1, -1):
        acc = am[k][:, None] * col[k] + (1 - am[k])[:, None] * acc
    (acc * dC.double().cpu()).sum().backward()
    # 16 hits, 96-wide 32-bit products and a sigmoid in between: some hundred roundings of terms of the result's size
    for got, want in ((C, acc.detach()), (dcond, E.grad), (dalpha, a64.grad), (dbg, b64.grad)):
        err = (got.double().cpu() - want).norm() / want.norm()
        assert err < 300 * ref.U, err


@pytest.mark.gpu
def test_inference_over_4_bit_descriptors():
    """Table, layer and compositing from 4 bits: as the same steps over the values they stand for."""
    sc, r, O, v, hits = _hits(2000, 24)
    R, n = hits.shape[1], sc.n
    table = microscale.quantize(sc.cond)
    rows = embedding.lookup(table, hits)
    assert torch.equal(rows, embedding.lookup(table.dequantize(), hits))
    layer = microscale.quantize(sc.A1[:, 32:].contiguous())
    per_primitive = microscale.product(table, layer, dtype=torch.float32)  # the descriptors' part of a first layer
    err = 98 * 2 * ref.U * (table.dequantize(torch.float32).abs() @ layer.dequantize(torch.float32).abs().T).cpu().double().numpy()
    ref.close(per_primitive, ref.f64(table.dequantize(torch.float32)) @ ref.f64(layer.dequantize(torch.float32)).T, err)
    y = embedding.lookup(per_primitive, hits)
    al = torch.where(hits >= 0, 0.3, 0.0)
    h, last, _ = recurrence.scan((1 - al).T[..., None], (al[..., None] * y).transpose(0, 1), reverse=True)
    want = torch.zeros(R, 64, device=DEV)
    for k in range(15, -1, -1):
        want = al[k][:, None] * y[k] + (1 - al[k])[:, None] * want
    assert (last - want).abs().max() < 64 * ref.U * y.abs().max() and torch.equal(h[:, 0], last)

    def image(cond):
        out = torch.zeros(R, 3, device=DEV)
        r.Forward_inference(cond, sc.features, sc.A1, sc.b1, sc.A2, sc.b2, sc.A3, sc.b3, O, v, out, 0.1, 0.2, 0.3, sc.m, sc.s, sc.q,
                            sc.RGBA, sc.k, 1e-4)
        return out

    got = image(table)
    assert torch.equal(got, image(table.dequantize())) and got.any()
    z = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    with pytest.raises(ValueError, match="4-bit"):
        r.Forward_training(table, sc.features, sc.A1, sc.b1, sc.A2, sc.b2, sc.A3, sc.b3, O, v, z(R, 3), 0.1, 0.2, 0.3, sc.m, sc.s, sc.q,
                           sc.RGBA, sc.k, 1e-4, z(R, 4), -0.1, 1.0, z(R, 2), z(R, 3), z(R, 4))


@pytest.mark.gpu
def test_two_calls_at_once():
    """The same operators on two streams at a time, each with workspaces of its own."""
    sc, _, _, _, hits = _hits(2000, 24)
    d = torch.randn(16, hits.shape[1], 96, device=DEV)
    gate = torch.rand(1, 4000, 64, device=DEV)
    x = torch.randn(1, 4000, 64, device=DEV)

    def work():
        a = embedding.lookup_backward(d, sc.cond, hits, need_weight=True)
        h, last, saved = recurrence.scan(gate, x, training=True)
        return a + (h, last) + recurrence.scan_backward(gate, x, saved, x)[:2] + (microscale.product(sc.cond, microscale.quantize(sc.A1[:, 32:])),)

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(want, outs))

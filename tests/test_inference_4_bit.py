"""Every inference method takes 4-bit descriptors and gives what it gives for the values they stand for (GPU)."""
import pytest
import torch

from flare_b200 import microscale
from flare_b200.scene import camera_rays, make_scene

DEV = "cuda"


def _case(kind, side=24):
    sc = make_scene(2000, 12, decoder=kind).to(DEV)
    O, v = camera_rays(side, side, 60.0, eye=(0.0, 0.0, 3.0))
    return sc, O.to(DEV), v.to(DEV), side * side


def _calls(kind):
    """name -> f(cond): the method's outputs."""
    from flare_b200.renderer import CPyOptiXFLARERenderer
    sc, O, v, R = _case(kind)
    r = CPyOptiXFLARERenderer(8, 11.3449, R)
    r.SetGeometry(*[t.contiguous() for t in sc.activated()])
    dec = (sc.features, sc.A1, sc.b1, sc.A2, sc.b2, sc.A3, sc.b3)
    geo = (sc.m, sc.s, sc.q, sc.RGBA, sc.k)
    z = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    colours = torch.rand(sc.n, 3, generator=torch.Generator().manual_seed(1)).to(DEV)

    def inference(c):
        out = z(R, 3)
        r.Forward_inference(c, *dec, O, v, out, 0.1, 0.2, 0.3, *geo, 1e-4)
        return [out]

    def geometry(c):
        out = [z(R, 3), z(R, 3), z(R), z(R)]
        r.Forward_inference_with_geometry(c, *dec, O, v, *out, 0.1, 0.2, 0.3, *geo, 1e-4)
        return out

    def pca(c):
        out = z(R, 3)
        r.Forward_pca(c, *dec, colours, O, v, out, 0.1, 0.2, 0.3, *geo, 1e-4)
        return [out]

    def median(c):
        out = z(R, 2)
        r.GetMedianDepth(c, *dec, O, v, *geo, 1e-4, out)
        return [out]

    def training(c):
        r.Forward_training(c, *dec, O, v, z(R, 3), 0.1, 0.2, 0.3, *geo, 1e-4, z(R, 4), -0.1, 1.0, z(R, 2), z(R, 3), z(R, 4))

    return sc, {"inference": inference, "geometry": geometry, "pca": pca, "median": median}, training


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["lut_pe", "grid_sh"])
def test_inference_methods(kind):
    sc, calls, training = _calls(kind)
    table = microscale.quantize(sc.cond)
    for name, f in calls.items():
        got, want = f(table), f(table.dequantize())
        # bits, as the index of a median depth is a whole number's
        assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(got, want)), name
        assert got[0].any(), name
    with pytest.raises(ValueError, match="4-bit"):
        training(table)
    for bad in (microscale.quantize(sc.cond[:, :31].contiguous()), microscale.quantize(sc.cond[:-1])):
        with pytest.raises(ValueError, match="conditioning_variable"):
            calls["inference"](bad)


@pytest.mark.gpu
def test_viewer():
    from flare_b200.viewer import CPyFlareViewerRenderer
    from oracle import viewer_oracle
    sc, O, v, R = _case("lut_pe")
    r = CPyFlareViewerRenderer(8, 11.3449, R, 2)
    sph, mat = (torch.from_numpy(t) for t in viewer_oracle.default_spheres())
    r.SetGeometry(*[t.contiguous() for t in sc.activated()], sph)

    def image(cond):
        out = torch.zeros(R, 3, device=DEV)
        r.Forward(cond, sc.features, sc.RGBA[:, :3].contiguous(), sc.A1, sc.b1, sc.A2, sc.b2, sc.A3, sc.b3, O, v, out, 0.2, 0.3, 0.4,
                  sc.m, sc.s, sc.q, sc.RGBA[:, 3].contiguous(), sc.k, 0.01, mat, torch.from_numpy(viewer_oracle.default_lights()), 1e-4,
                  0.55, 0.06, 0.06, 0.07)
        return out

    table = microscale.quantize(sc.cond)
    got = image(table)
    assert torch.equal(got, image(table.dequantize())) and got.any()

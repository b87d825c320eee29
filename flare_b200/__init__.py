"""flare_b200: B200-native (sm_100a) implementation of FlaRe's differentiable render path.

Public API: `flare_b200.renderer.CPyOptiXFLARERenderer` / `GenerateRays` (the reference extension's
interface), `flare_b200.scene` (seeded synthetic workloads), `flare_b200.dp` (data-parallel step), and for decoders
outside the renderer `flare_b200.embedding` (row lookup and its gradient), `flare_b200.recurrence` (the gated linear
recurrence) and `flare_b200.microscale` (4-bit matrices).
The native library is built with `python -m flare_b200.build`.
"""
__version__ = "0.1.0"

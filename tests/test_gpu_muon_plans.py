"""Every way in which newton_schulz launches its products: tiles of 64, 128, 192 and 256 for each of them, sums over long
rows whole and in parts, matrices of at most 64 rows beside ones that take wider tiles -- for split fp16 operands (prec 0)
and single ones (prec 1).  Which call takes which way is mms_muon_plan's answer; tests/test_cpu_muon_plans.py checks that
CASES take every way that ordinary sizes do.

Tolerances: test_gpu_muon.tolerance for prec 0; half a step of bfloat16, 2^-8, for prec 1."""
import pytest
import torch

from test_gpu_muon import gradient, iterate, rel, tolerance

pytestmark = pytest.mark.gpu

CASES = [
    [(40, 70)], [(1, 900)], [(132, 1623)], [(129, 138)],
    [(32, 345, 364)], [(99, 39), (288, 15), (32, 377, 338)],
    [(4, 3, 718), (8, 486, 591), (2, 936)],
    [(4288, 515)], [(641, 6038)],
    [(32, 522, 646), (265, 67), (4, 263, 13)],
    [(16, 947, 909)],
    [(16, 1187, 1229), (3, 1843)],
    [(32, 644, 1145), (32, 2, 4968)],
    [(16, 1, 1870), (2, 188, 345)],
    [(32, 142, 199), (8, 65, 12), (4, 138, 739)],
    [(32, 1052, 130), (49, 92), (4, 4, 2109)],
    [(16, 2825, 131), (16, 167, 328), (40, 307)],
    [(32, 129, 1586)],
    [(32, 323, 370), (16, 1281), (2475, 9)],
]


@pytest.fixture()
def gen(dev):
    return torch.Generator(device="cuda").manual_seed(41)


@pytest.mark.parametrize("prec", [0, 1])
@pytest.mark.parametrize("shapes", CASES, ids=str)
def test_every_plan(dev, gen, shapes, prec):
    from multimodalstudio_amd import hip_ops
    mats = [gradient(s, gen, torch.float32) for s in shapes]
    outs = hip_ops.newton_schulz(mats, prec=prec)
    for g, out in zip(mats, outs):
        want = iterate(g, torch.float64)
        assert rel(out, want) <= (tolerance(g, want) if prec == 0 else 2.0 ** -8), tuple(g.shape)
    assert all(torch.equal(x, y) for x, y in zip(outs, hip_ops.newton_schulz(mats, prec=prec)))


@pytest.mark.parametrize("shapes", [[(32, 522, 646), (265, 67)], [(16, 1187, 1229), (3, 1843)], [(641, 6038)]], ids=str)
def test_step_with_every_tile(dev, gen, shapes):
    """Weights, gradient and momentum through the wide tiles' last launch: rows that are no whole 16 bytes, tall and wide."""
    from multimodalstudio_amd import hip_ops
    from test_gpu_muon import check_step, reference_step
    ps = [torch.randn(s, device="cuda", generator=gen) for s in shapes]
    ms = [gradient(s, gen, torch.float32) for s in shapes]
    gs = [gradient(s, gen, torch.float32) for s in shapes]
    want = [reference_step(p, g, m, 0.02, 0.95, True, 0.1) for p, g, m in zip(ps, gs, ms)]
    hip_ops.muon_step(ps, gs, ms, lr=0.02)
    for p, m, w in zip(ps, ms, want):
        check_step(p, m, w, torch.float32)

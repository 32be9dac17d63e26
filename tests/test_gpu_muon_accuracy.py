"""The accuracy that hip_ops.newton_schulz and muon_step give where nothing is said: that of float32 products, for
matrices held in bfloat16 too.

Tolerance of a rounded result.  v is the value before its rounding, w the definition's, e = |v - w| <= the float32
iteration's tolerance (test_gpu_muon.tolerance).  Where v and w round alike, |round(v) - w| = |round(w) - w|; where they
do not, w is within e of the border, so |round(v) - w| <= half a step + e and |round(w) - w| >= half a step - e.  So
|round(v) - w| <= |round(w) - w| + 2 e for each entry, and in the Frobenius norm."""
import pytest
import torch

from test_gpu_muon import gradient, iterate, reference_step, rel, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gen(dev):
    return torch.Generator(device="cuda").manual_seed(31)


@pytest.mark.parametrize("shape", [(3, 64), (129, 129), (257, 300), (1024, 1030), (3, 1000, 2049), (2000, 900)], ids=str)
def test_bfloat16_results_are_rounded_once(dev, gen, shape):
    from multimodalstudio_amd import hip_ops
    g = gradient(shape, gen, torch.bfloat16)
    want = iterate(g, torch.float64)
    bound = rel(want.bfloat16(), want) + 2 * tolerance(g.float(), want)
    assert rel(hip_ops.newton_schulz(g), want) <= bound
    assert torch.equal(hip_ops.newton_schulz(g), hip_ops.newton_schulz(g, prec=0))


def test_bfloat16_weights_are_rounded_once(dev, gen):
    from multimodalstudio_amd import hip_ops
    shapes = [(300, 200), (1024, 1030), (2, 700, 1100)]
    ps = [torch.randn(s, device="cuda", generator=gen).bfloat16() for s in shapes]
    gs = [gradient(s, gen, torch.bfloat16) for s in shapes]
    ms = [gradient(s, gen, torch.float32) for s in shapes]
    want = [reference_step(p, g, m, 0.02, 0.95, True, 0.1) for p, g, m in zip(ps, gs, ms)]
    hip_ops.muon_step(ps, gs, ms, lr=0.02, weight_decay=0.1)
    for p, (wp, _, update, u) in zip(ps, want):
        # before the rounding: the update's error, a float32 product and sum, the float32 of 1 - lr wd
        off = tolerance(u.float(), iterate(u, torch.float64)) * float(update.norm()) + 2.0 ** -23 * float(wp.norm())
        assert float((p.double() - wp).norm()) <= float((wp.bfloat16().double() - wp).norm()) + 2 * off

"""The accuracy that hip_ops.newton_schulz and muon_step give where nothing is said: that of float32 products, for
matrices held in bfloat16 too.

Tolerance of a rounded result.  v is the value before its rounding, w the definition's, e = |v - w| <= the float32
iteration's tolerance (test_gpu_muon.tolerance).  Where v and w round alike, |round(v) - w| = |round(w) - w|; where they
do not, w is within e of the border, so |round(v) - w| <= half a step + e and |round(w) - w| >= half a step - e.  So
|round(v) - w| <= |round(w) - w| + 2 e for each entry, and in the Frobenius norm.

Uneven gradients.  An entry of 2^-23 of the norm or more keeps 22 bits as an operand, so test_gpu_muon.tolerance's 12 half
steps of float32 hold for any part of the result against the same part of a float32 iteration."""
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


def part_error(x, want, rows):
    return float((x.double()[..., rows, :] - want[..., rows, :]).norm() / want[..., rows, :].norm())


# tiles of every width (a call's matrices share theirs)
@pytest.mark.parametrize("shape", [(60, 100), (256, 256), (512, 1024), (6, 512, 1024), (2048, 2048), (4, 2048, 2500), (900, 250)],
                         ids=str)
@pytest.mark.parametrize("kind", ["entry 1e6", "entry 4e6", "row 1e4", "spread"])
def test_uneven_gradients_keep_their_small_parts(dev, gen, shape, kind):
    """One entry or one row far larger than the rest, and rows that fall off over six decades: the rest by itself."""
    from multimodalstudio_amd import hip_ops
    g = torch.randn(shape, device="cuda", generator=gen)
    r = shape[-2]
    rest = [i for i in range(r) if i != 3]
    if kind.startswith("entry"):
        g[..., 3, 5] = float(kind.split()[1])
    elif kind.startswith("row"):
        g[..., 3, :] *= 1e4
    else:
        g *= torch.logspace(0, -6, r, device="cuda")[:, None]
        rest = list(range(r // 2, r))
    want = iterate(g, torch.float64)
    single = iterate(g, torch.float32)
    out = hip_ops.newton_schulz(g)
    for rows in (list(range(r)), rest):
        assert part_error(out, want, rows) <= 12 * max(part_error(single, want, rows), 4 * 2.0 ** -24)


@pytest.mark.parametrize("steps,coeff", [(3, (6.0, 0.0, 0.0)), (2, (20.0, -60.0, 45.0)), (1, (1e6, -1e4, 0.0))])
def test_coefficients_that_grow(dev, gen, steps, coeff):
    """Iterates and products of some hundreds or thousands: the operands' units make room for them.  (The gradient's
    largest singular value is its norm, which is what the coefficients meet.)"""
    from multimodalstudio_amd import hip_ops
    for shape in ((50, 90), (900, 1100)):
        g = torch.randn(shape[0], 1, device="cuda", generator=gen) * torch.randn(1, shape[1], device="cuda", generator=gen)
        want = iterate(g, torch.float64, steps=steps, coeff=coeff)
        out = hip_ops.newton_schulz(g, steps=steps, coefficients=coeff)
        assert rel(out, want) <= tolerance(g, want, steps=steps, coeff=coeff)


def test_coefficients_out_of_range_are_refused(dev):
    from multimodalstudio_amd import hip_ops
    g = torch.ones(6, 8, device="cuda")
    for steps, coeff in ((5, (300.0, 0.0, 0.0)), (2, (3.0, -7e4, 0.0)), (12, (4.0, 1.0, 1.0))):
        with pytest.raises(RuntimeError, match="coefficients"):
            hip_ops.newton_schulz(g, steps=steps, coefficients=coeff)
        with pytest.raises(RuntimeError, match="coefficients"):
            hip_ops.muon_step([g.clone()], [g], [torch.zeros_like(g)], lr=0.1, steps=steps, coefficients=coeff)

"""Muon's operators (hip_ops.newton_schulz, hip_ops.muon_step) against the definition in 64 bits.

Tolerances.  The result's error is measured in the Frobenius norm over the result's.
  float32: operands are split into two fp16 values that keep 22 bits, and a product drops lo * lo: up to 3 * 2^-22 per
    product, 12 half steps of float32 (2^-24) where a float32 product has at least one.  So 12 times the error of the
    same iteration in float32, and not less than 12 times that of 15 roundings that add up at random (4 * 2^-24).
  bfloat16: the result's own rounding is at most a half step 2^-8 (2^-8 / sqrt(3) and less in the norm), and the fp16
    products below it must leave the sum of both under that half step.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

COEFF = (3.4445, -4.7750, 2.0315)


def iterate(g, dtype, steps=5, coeff=COEFF, eps=1e-7):
    """X = G / max(|G|, eps); X <- a X + (b A + c A A) X, in ``dtype``."""
    x = g.to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    x = (x.mT if tall else x).contiguous()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    a, b, c = coeff
    for _ in range(steps):
        gram = torch.matmul(x, x.mT.contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.mT.contiguous() if tall else x


def rel(x, want):
    return float((x.double() - want).norm() / want.norm().clamp(min=1e-300))


def tolerance(g, want, **kw):
    if g.dtype == torch.bfloat16:
        return 2.0 ** -8
    return 12 * max(rel(iterate(g, torch.float32, **kw), want), 4 * 2.0 ** -24)


def gradient(shape, gen, dtype, scale=1e-3):
    """Strong directions whose strength falls like 1 / i over noise."""
    *lead, m, n = shape
    k = max(1, min(16, m, n))
    u = torch.randn(*lead, m, k, device="cuda", generator=gen) / torch.arange(1, k + 1, device="cuda")
    g = torch.matmul(u, torch.randn(*lead, k, n, device="cuda", generator=gen))
    return (scale * (g + 0.3 * torch.randn(*lead, m, n, device="cuda", generator=gen))).to(dtype)


@pytest.fixture()
def gen(dev):
    return torch.Generator(device="cuda").manual_seed(11)


DTYPES = [torch.float32, torch.bfloat16]
# one row, one column, one value; below, at and over the tiles' sides; wide, tall, stacks; the three tile sizes (a
# call's matrices use 128- and 256-wide tiles once they have 192 of them)
# (That was the choice once.  Four tile sizes, by the expected end of the launch: test_gpu_muon_plans.py has them all.)
SHAPES = [(1, 1), (1, 5), (5, 1), (1, 4097), (2, 2), (3, 64), (64, 64), (65, 63), (64, 257), (129, 128), (256, 71),
          (257, 256), (256, 317), (5, 100, 40), (2, 3, 33, 70), (4, 1000, 900), (13, 1024, 1030), (9, 1500, 1100)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalisation(dev, gen, shape, dtype):
    from multimodalstudio_amd import hip_ops
    g = gradient(shape, gen, dtype)
    keep = g.clone()
    out = hip_ops.newton_schulz(g)
    assert out.shape == g.shape and out.dtype == dtype and out.is_contiguous() and torch.equal(g, keep)
    want = iterate(g, torch.float64)
    assert rel(out, want) <= tolerance(g, want)
    assert torch.equal(out, hip_ops.newton_schulz(g))


# sums over long rows are split over blocks: one tile and many, stacks, tall, beside short ones that are not split
LONG = [[(1, 20000)], [(40, 5000)], [(4096, 17)], [(3, 130, 2100)], [(300, 4096)], [(700, 8192)], [(1024, 16384)],
        [(60, 9000), (2000, 33), (50, 60), (3, 3), (2, 7, 3000)]]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shapes", LONG, ids=str)
def test_long_rows(dev, gen, shapes, dtype):
    from multimodalstudio_amd import hip_ops
    mats = [gradient(s, gen, dtype) for s in shapes]
    outs = hip_ops.newton_schulz(mats)
    for g, out in zip(mats, outs):
        want = iterate(g, torch.float64)
        assert rel(out, want) <= tolerance(g, want), tuple(g.shape)
    # whichever block adds a tile's parts: the same bits, in a replayed graph too
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(outs, hip_ops.newton_schulz(mats)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = hip_ops.newton_schulz(mats)
    for _ in range(3):
        for x in again:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, again))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_matrices_in_one_call(dev, gen, dtype):
    """More matrices than one launch holds, of every tile size, with empty ones between them: each as if alone."""
    from multimodalstudio_amd import hip_ops
    shapes = [(7 + 5 * i, 90 - i) for i in range(60)] + [(0, 5), (0, 4, 4), (5, 0)] + [(3, 1200, 1300), (12, 600, 700)]
    mats = [gradient(s, gen, dtype) if math.prod(s) else torch.empty(s, device="cuda", dtype=dtype) for s in shapes]
    outs = hip_ops.newton_schulz(mats)
    for g, out in zip(mats, outs):
        assert out.shape == g.shape
        if g.numel():
            want = iterate(g, torch.float64)
            assert rel(out, want) <= tolerance(g, want), tuple(g.shape)
    assert hip_ops.newton_schulz([]) == []


def test_mixed_types_keep_theirs(dev, gen):
    from multimodalstudio_amd import hip_ops
    mats = [gradient((40, 60), gen, torch.bfloat16), gradient((70, 30), gen, torch.float32)]
    for g, out in zip(mats, hip_ops.newton_schulz(mats)):
        want = iterate(g, torch.float64)
        assert out.dtype == g.dtype and rel(out, want) <= tolerance(g, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layouts(dev, gen, dtype):
    """Rows of a wider buffer, a transposed view, every second matrix of a stack, an expanded matrix."""
    from multimodalstudio_amd import hip_ops
    base = gradient((6, 70, 130), gen, dtype)
    views = [base[0][:, 3:100], base[1].mT, base[::2], base[2][::2, :33], base[3][:, ::2], base[4][:1].expand(5, 130)]
    for v in views:
        want = iterate(v, torch.float64)
        assert rel(hip_ops.newton_schulz(v), want) <= tolerance(v, want)
    assert rel(hip_ops.newton_schulz([base[1].mT])[0], iterate(base[1], torch.float64).mT) <= \
        tolerance(base[1], iterate(base[1], torch.float64))


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_any_scale(dev, gen, scale):
    """The norm is summed in double: the result does not depend on the gradient's scale (eps is below all of them)."""
    from multimodalstudio_amd import hip_ops
    g = gradient((50, 80), gen, torch.float32, 1.0)
    want = iterate(g * scale, torch.float64, eps=1e-60)
    assert rel(hip_ops.newton_schulz(g * scale, eps=1e-60), want) <= tolerance(g, iterate(g, torch.float64))


def test_eps_bounds_the_norm(dev, gen):
    """A gradient below eps stays small: X = G / eps, and each step multiplies small singular values by a = 3.4445 (the
    cubic and quintic terms only take away there), so |result| <= a^5 |G| / eps = 485 |G| / eps."""
    from multimodalstudio_amd import hip_ops
    g = gradient((50, 80), gen, torch.float32, 1e-14)
    want = iterate(g, torch.float64, eps=1e-7)
    assert want.norm() <= 485 * g.norm() / 1e-7 < 0.01 and rel(hip_ops.newton_schulz(g, eps=1e-7), want) <= 2.0 ** -11


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_zeros_nan_and_infinity_stay_in_their_matrix(dev, gen, dtype):
    from multimodalstudio_amd import hip_ops
    g = gradient((5, 70, 90), gen, dtype)
    alone = hip_ops.newton_schulz(g)
    g[1] = 0.0
    g[2, 3, 4] = float("nan")
    g[3, 69, 89] = float("inf")
    out = hip_ops.newton_schulz(g)
    assert torch.equal(out[0], alone[0]) and torch.equal(out[4], alone[4])
    assert (out[1] == 0).all() and out[2].isnan().all() and out[3].isnan().all()


@pytest.mark.parametrize("steps,coeff", [(1, COEFF), (3, (2.0, -1.5, 0.5)), (10, (2.0, -1.5, 0.5)), (2, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients(dev, gen, steps, coeff):
    from multimodalstudio_amd import hip_ops
    for shape in ((60, 130), (130, 60)):
        g = gradient(shape, gen, torch.float32)
        want = iterate(g, torch.float64, steps=steps, coeff=coeff)
        out = hip_ops.newton_schulz(g, steps=steps, coefficients=coeff)
        assert rel(out, want) <= tolerance(g, want, steps=steps, coeff=coeff)


def test_precisions(dev, gen):
    """prec 1 keeps a float32 result within bfloat16's half step; prec 0 leaves bfloat16 its own rounding alone."""
    from multimodalstudio_amd import hip_ops
    g = gradient((13, 1024, 1024), gen, torch.float32)
    want = iterate(g, torch.float64)
    assert tolerance(g, want) < rel(hip_ops.newton_schulz(g, prec=1), want) <= 2.0 ** -8
    h = g.bfloat16()
    assert rel(hip_ops.newton_schulz(h, prec=0), iterate(h, torch.float64)) <= 2.0 ** -8 / math.sqrt(3.0)


# ---- the step ---------------------------------------------------------------------------------------------------
def reference_step(p, g, m, lr, mu, nesterov, wd, adjust=None, clip=1.0):
    from multimodalstudio_amd import hip_ops
    g = g.double() * clip
    m2 = m.double() + (1.0 - mu) * (g - m.double())
    u = g + mu * (m2 - g) if nesterov else m2
    o = iterate(u, torch.float64)
    scale = hip_ops.muon_scale(p.shape[-2], p.shape[-1], adjust)
    return (1.0 - lr * wd) * p.double() - lr * scale * o, m2, lr * scale * o, u


def check_step(p, m, want, dtype):
    wp, wm, update, u = want
    # the momentum: float32's half step for each of its three operations
    assert rel(m, wm) <= 3 * 2.0 ** -24
    # the weights: their own rounding (and that of 1 - lr wd) plus the update's error
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    tol = 2.0 ** -8 if dtype == torch.bfloat16 else tolerance(u.float(), iterate(u, torch.float64))
    assert float((p.double() - wp).norm()) <= half * float(wp.norm()) + tol * float(update.norm())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("nesterov,wd,adjust", [(True, 0.1, None), (False, 0.0, "match_rms_adamw")])
def test_step(dev, gen, dtype, nesterov, wd, adjust):
    from multimodalstudio_amd import hip_ops
    shapes = [(256, 71), (257, 256), (3, 64), (1, 9), (4, 100, 30), (13, 1024, 1000)]
    ps = [torch.randn(s, device="cuda", generator=gen).to(dtype) for s in shapes]
    ms = [torch.zeros(s, device="cuda") for s in shapes]
    for t in range(3):
        gs = [gradient(s, gen, dtype) for s in shapes]
        want = [reference_step(p, g, m, 0.02, 0.95, nesterov, wd, adjust) for p, g, m in zip(ps, gs, ms)]
        keep = [g.clone() for g in gs]
        hip_ops.muon_step(ps, gs, ms, lr=0.02, momentum=0.95, nesterov=nesterov, weight_decay=wd, adjust=adjust)
        for p, g, m, w, k in zip(ps, gs, ms, want, keep):
            check_step(p, m, w, dtype)
            assert torch.equal(g, k)


def test_step_clips(dev, gen):
    """The gradient is scaled by min(1, max_norm / (norm + 1e-6)) with the norm of the whole group, read on the device."""
    from multimodalstudio_amd import hip_ops
    for norm, clip in ((0.5, 1.0), (8.0, 2.0 / (8.0 + 1e-6))):
        p, g = torch.randn(60, 50, device="cuda", generator=gen), gradient((60, 50), gen, torch.float32)
        m = gradient((60, 50), gen, torch.float32)
        want = reference_step(p, g, m, 0.02, 0.95, True, 0.1, None, clip)
        sumsq = torch.tensor([norm * norm], device="cuda")
        hip_ops.muon_step([p], [g], [m], lr=0.02, sumsq=sumsq, max_norm=2.0)
        check_step(p, m, want, torch.float32)


def test_step_writes_only_its_weights(dev, gen):
    """Weights that are columns of a wider buffer: what lies beside them stays."""
    from multimodalstudio_amd import hip_ops
    for shape in ((60, 100), (100, 60)):
        buf = torch.randn(shape[0] + 2, shape[1] + 7, device="cuda", generator=gen)
        keep = buf.clone()
        p = buf[1:-1, 3:-4]
        g, m = gradient(shape, gen, torch.float32), torch.zeros(shape, device="cuda")
        want = reference_step(p, g, m, 0.02, 0.95, True, 0.1)
        hip_ops.muon_step([p], [g], [m], lr=0.02)
        check_step(p, m, want, torch.float32)
        keep[1:-1, 3:-4] = p
        assert torch.equal(buf, keep)


def test_step_in_a_graph(dev, gen):
    """Captured with device scalars and replayed between eager steps of other weights: the same bits as eager steps."""
    from multimodalstudio_amd import hip_ops
    shapes = [(256, 71), (90, 300), (5, 128, 128)]
    p0 = [torch.randn(s, device="cuda", generator=gen) for s in shapes]
    grads = [[gradient(s, gen, torch.float32) for s in shapes] for _ in range(4)]
    lrs = [0.02, 0.01, 0.03, 0.005]
    eager, em = [p.clone() for p in p0], [torch.zeros_like(p) for p in p0]
    seen = []
    for gs, lr in zip(grads, lrs):
        hip_ops.muon_step(eager, gs, em, lr=lr, weight_decay=0.1,
                          hyper=torch.tensor([1.0 - lr * 0.1, -lr], device="cuda"))
        seen.append([p.clone() for p in eager])
    ps, ms, gs = [p.clone() for p in p0], [torch.zeros_like(p) for p in p0], [torch.zeros_like(p) for p in p0]
    hyper = torch.zeros(2, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        hip_ops.muon_step(ps, gs, ms, lr=1.0, hyper=hyper)
    for t in range(4):
        for a, b in zip(gs, grads[t]):
            a.copy_(b)
        hyper.copy_(torch.tensor([1.0 - lrs[t] * 0.1, -lrs[t]]))
        graph.replay()
        hip_ops.muon_step([p.clone() for p in p0], grads[0], [torch.zeros_like(p) for p in p0], lr=0.1)
        torch.cuda.synchronize()
        for a, b in zip(ps, seen[t]):
            assert torch.equal(a, b)


def test_another_stream(dev, gen):
    from multimodalstudio_amd import hip_ops
    g = gradient((300, 400), gen, torch.float32)
    want = hip_ops.newton_schulz(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [hip_ops.newton_schulz(g) for _ in range(3)]
    here = [hip_ops.newton_schulz(g) for _ in range(3)]
    torch.cuda.synchronize()
    for o in outs + here:
        assert torch.equal(o, want)


def test_offsets_past_32_bits(dev, gen):
    """A stack of more than 2^31 elements: its first, middle and last matrix."""
    from multimodalstudio_amd import hip_ops
    few = gradient((3, 1024, 1100), gen, torch.bfloat16)
    n = 2 ** 31 // (1024 * 1100) + 2
    stack = few[1].expand(n, -1, -1).contiguous()
    stack[0], stack[n - 1] = few[0], few[2]
    out = hip_ops.newton_schulz(stack)
    for k, g in ((0, few[0]), (n // 2, few[1]), (n - 1, few[2])):
        want = iterate(g, torch.float64)
        assert rel(out[k], want) <= tolerance(g, want), k


def test_two_calls_at_once(dev, gen):
    """Calls on two streams that run together, their sums over long rows split: each gives its own bits."""
    from multimodalstudio_amd import hip_ops
    calls = [[gradient((40, 5000), gen, torch.float32), gradient((300, 4096), gen, torch.float32)],
             [gradient((700, 8192), gen, torch.bfloat16), gradient((9, 3000), gen, torch.bfloat16)]]
    want = [hip_ops.newton_schulz(c) for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(hip_ops.newton_schulz(c))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))


def test_refusals(dev):
    from multimodalstudio_amd import hip_ops
    p, m = torch.zeros(6, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    for bad in (lambda: hip_ops.newton_schulz(p.half()), lambda: hip_ops.newton_schulz([p, p.double()]),
                lambda: hip_ops.muon_step([p.half()], [p.half()], [m], lr=0.1)):
        with pytest.raises(TypeError):
            bad()
    s = torch.ones(1, device="cuda")
    for bad in (lambda: hip_ops.newton_schulz(p[0]), lambda: hip_ops.muon_step([p], [p[:5]], [m], lr=0.1),
                lambda: hip_ops.muon_step([p], [p], [m[:, :4]], lr=0.1),
                lambda: hip_ops.muon_step([p], [p.bfloat16()], [m], lr=0.1),
                lambda: hip_ops.muon_step([p], [p], [m.bfloat16()], lr=0.1),
                lambda: hip_ops.muon_step([p], [p], [torch.zeros(8, 6, device="cuda").mT], lr=0.1),
                lambda: hip_ops.muon_step([torch.zeros(8, 6, device="cuda").mT], [p], [m], lr=0.1),
                lambda: hip_ops.muon_step([p[:1].expand(6, 8)], [p], [m], lr=0.1),
                lambda: hip_ops.muon_step([p, p], [p, p], [m, m.clone()], lr=0.1),
                lambda: hip_ops.muon_step([p, p.clone()], [p, p], [m, m], lr=0.1),
                lambda: hip_ops.muon_step([p], [p], [m], lr=0.1, sumsq=s),
                lambda: hip_ops.muon_step([p], [p], [m], lr=0.1, sumsq=s.double(), max_norm=1.0),
                lambda: hip_ops.muon_step([p], [p], [m], lr=0.1, hyper=s),
                lambda: hip_ops.muon_step([p], [p], [m], lr=0.1, adjust="none")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: hip_ops.newton_schulz(p, steps=0), lambda: hip_ops.newton_schulz(p, eps=0.0),
                lambda: hip_ops.newton_schulz(p, prec=3), lambda: hip_ops.newton_schulz(p.cpu()),
                lambda: hip_ops.muon_step([p], [p], [m], lr=0.1, momentum=1.0)):
        with pytest.raises(RuntimeError):
            bad()
    assert (p == 0).all() and (m == 0).all()

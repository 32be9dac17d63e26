"""Calls of muon_step on memory that its matrices share: refused with nothing changed, or right."""
import pytest
import torch

from test_gpu_muon import check_step, gradient, reference_step

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gen(dev):
    return torch.Generator(device="cuda").manual_seed(51)


def test_overlapping_matrices(dev, gen):
    from multimodalstudio_amd import hip_ops
    w, g, m = torch.randn(6, 8, device="cuda", generator=gen), torch.randn(6, 8, device="cuda", generator=gen), \
        torch.zeros(6, 8, device="cuda")
    stack = torch.randn(3, 4, 8, device="cuda", generator=gen)
    keep = [t.clone() for t in (w, g, m, stack)]

    def zeros(t):
        return torch.zeros_like(t, memory_format=torch.contiguous_format)
    for ps, gs, ms in (([w[:4], w[2:]], [g[:4], g[2:]], None), ([stack, stack[1]], [stack.clone(), g[:4]], None),
                       ([w[:, :5], w[:, 4:]], [g[:, :5], g[:, 4:]], None), ([w[:3], w[3:]], [g[:3], g[3:]], [m[:3], m[1:4]]),
                       ([w], [g], [w]), ([w], [m], [m]), ([w, stack[0]], [g, w[:4]], None)):
        with pytest.raises(RuntimeError, match="overlap"):
            hip_ops.muon_step(ps, gs, ms or [zeros(p) for p in ps], lr=0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((w, g, m, stack), keep))


def test_backward_passes_notice_the_step(dev, gen):
    """A backward pass that saved the weights or a momentum from before the step raises instead of using the new ones."""
    from multimodalstudio_amd import hip_ops
    from multimodalstudio_amd import pipeline as pl
    x = torch.randn(5, 8, device="cuda", generator=gen, requires_grad=True)
    p, g = torch.nn.Parameter(torch.randn(6, 8, device="cuda", generator=gen)), torch.randn(6, 8, device="cuda", generator=gen)
    m = torch.zeros(6, 8, device="cuda")
    for saved in (p, m):
        loss = (x @ saved.mT).sum()
        hip_ops.muon_step([p], [g], [m], lr=0.1)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    group = pl.MuonGroup([p], lr=0.1, weight_decay=0.0)
    p.grad.copy_(g)
    loss = (x @ p.mT).sum()
    group.step(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    assert p.grad.data_ptr() == group.grad.data_ptr() and p.data_ptr() == group.flat.data_ptr()


def test_columns_side_by_side(dev, gen):
    """Weights that are columns of one buffer, as fused projections are, each stepped by itself."""
    from multimodalstudio_amd import hip_ops
    buf, g = torch.randn(90, 150, device="cuda", generator=gen), gradient((90, 150), gen, torch.float32)
    cuts = [(0, 50), (50, 120), (120, 147)]
    ps = [buf[:, a:b] for a, b in cuts]
    gs = [g[:, a:b] for a, b in cuts]
    ms = [torch.zeros(90, b - a, device="cuda") for a, b in cuts]
    keep = buf[:, 147:].clone()
    want = [reference_step(p, x, m, 0.02, 0.95, True, 0.1) for p, x, m in zip(ps, gs, ms)]
    hip_ops.muon_step(ps, gs, ms, lr=0.02)
    for p, m, w in zip(ps, ms, want):
        check_step(p, m, w, torch.float32)
    assert torch.equal(buf[:, 147:], keep)

"""Muon in the trainer: one clip over all of the fields' gradients, and replayed steps that move the matrices as eager
ones do."""
import pytest
import torch

from test_gpu_muon import check_step, reference_step

pytestmark = pytest.mark.gpu


def _groups(dev, together):
    from multimodalstudio_amd import pipeline as pl
    gen = torch.Generator().manual_seed(6)
    mats = [torch.nn.Parameter((0.1 * torch.randn(s, generator=gen)).to(dev)) for s in ((60, 71), (33, 60))]
    vec = torch.nn.Parameter(torch.randn(500, generator=gen).to(dev))
    ad = pl.FlatGroup([vec], lr=1e-3, weight_decay=0.01, eps=1e-15)
    mu = pl.MuonGroup(mats, lr=1e-2, weight_decay=0.1)
    if together:
        pl.clip_together([ad, mu])
    return ad, mu, vec, mats


@pytest.mark.parametrize("form", ["eager", "captured", "bank"])
@pytest.mark.parametrize("together", [True, False])
def test_clip_of_several_groups(dev, form, together):
    """Gradients of norms 4 and 3: clipped at 2 together by 2 / 5, each by itself by 2 / 4 and 2 / 3."""
    from multimodalstudio_amd import pipeline as pl
    ad, mu, vec, mats = _groups(dev, together)
    bank = pl.OptimBank([ad, mu]) if form == "bank" else None
    gen = torch.Generator(device="cuda").manual_seed(1)
    ref = vec.detach().clone().requires_grad_()
    adamw = torch.optim.AdamW([ref], lr=1e-3, weight_decay=0.01, eps=1e-15)
    for t in range(2):
        if bank:
            bank.zero_grads()
        else:
            ad.zero_grad()
            mu.zero_grad()
        for group, norm in ((ad, 4.0), (mu, 3.0)):
            group.grad[:group.n].normal_(generator=gen)
            group.grad.mul_(norm / group.grad.norm())
        clip = {True: (0.4, 0.4), False: (0.5, 2.0 / 3.0)}[together]
        want = [reference_step(p.detach(), p.grad, m, 1e-2, 0.95, True, 0.1, "match_rms_adamw", clip[1])
                for p, m in zip(mats, mu.momenta)]
        ref.grad = vec.grad * clip[0]
        adamw.step()
        if bank:
            bank.load_hyper(1.0)
            bank.step_captured()
        else:
            for g in (ad, mu):
                if form == "captured":
                    g.load_hyper(1.0)
                    g.step_captured()
                else:
                    g.step(1.0)
        for p, m, w in zip(mats, mu.momenta, want):
            # the norm is a float32 sum of 6743 squares by atomics and a quotient: some half steps on the momentum
            assert float((m.double() - w[1]).norm()) <= 64 * 2.0 ** -24 * float(w[1].norm())
            check_step(p.detach(), w[1].float(), w, torch.float32)
        assert (vec - ref).abs().max() <= 2e-6 * ref.abs().max()


def test_no_clip_and_a_torn_bank(dev):
    """max_norm 0 does not clip, as with AdamW; a bank needs every group that the clip goes by."""
    from multimodalstudio_amd import pipeline as pl
    ad, mu, vec, mats = _groups(dev, True)
    mu.grad.fill_(1.0)
    want = [reference_step(p.detach(), p.grad, m, 1e-2, 0.95, True, 0.1, "match_rms_adamw") for p, m in zip(mats, mu.momenta)]
    mu.step(1.0, max_norm=0.0)
    for p, m, w in zip(mats, mu.momenta, want):
        check_step(p.detach(), m, w, torch.float32)
    with pytest.raises(ValueError, match="bank"):
        pl.OptimBank([mu])
    pl.OptimBank([ad, mu])
    with pytest.raises(ValueError, match="OptimBank"):
        pl.clip_together([ad, mu])


def test_the_trainer_clips_as_with_adamw(dev):
    from multimodalstudio_amd import pipeline as pl
    cfg = pl.TrainConfig(num_rays_per_modality=64, log2T=12, width=64, height=48, n_views=20, optimizer="muon")
    t = pl.Trainer(cfg, dev)
    assert t.fields.norm_groups == [t.fields, t.matrices] == t.matrices.norm_groups and t.poses.norm_groups is None
    assert t.fields.sumsq is t.matrices.sumsq and t.poses.sumsq is not t.fields.sumsq
    t.set_step(9500)
    t.train_step()
    total = sum(float(g.grad.double().square().sum()) for g in (t.fields, t.matrices))
    # a float32 sum of 10^5 .. 10^6 squares, by blocks and atomics
    assert abs(float(t.fields.sumsq) - total) <= 1e-4 * total


def test_replayed_steps_move_the_matrices_as_eager_ones(dev):
    """Each step of a GraphTrainer, its eager first one and the replays, moves the matrices as the definition does on the
    gradients that the step left, clipped by the fields' norm; and the losses follow those of eager steps from the same
    state (within the 1e-3 that test_gpu_graph.py has for float-atomic gradients)."""
    from multimodalstudio_amd import graphs
    from multimodalstudio_amd import pipeline as pl
    cfg = pl.TrainConfig(method="grid", modalities=("rgb",), num_rays_per_modality=512, log2T=14, n_views=10, width=160,
                         height=128, optimizer="muon")

    def make():
        t = pl.Trainer(cfg, dev)
        t.set_step(95000)
        t.model.eval()       # no sampler jitter: both see the same samples
        return t
    eager, t = make(), make()
    runner = graphs.GraphTrainer(t, granule=64)
    losses = []
    for k in range(6):
        before = [p.detach().clone() for p in t.matrices.params]
        momenta = [m.clone() for m in t.matrices.momenta]
        lr = 1e-3 * pl.lr_factor(t.step, cfg.max_iters)
        replays = runner.stats["replays"]
        losses.append((float(eager.train_step()[1]), float(runner.step()[1])))
        torch.cuda.synchronize()
        assert k < 2 or runner.stats["replays"] == replays + 1, (k, runner.stats)
        total = sum(float(g.grad.double().square().sum()) for g in (t.fields, t.matrices))
        clip = min(1.0, 2.0 / (total ** 0.5 + 1e-6))
        moved = 0.0
        for p, q, m, n in zip(before, t.matrices.params, momenta, t.matrices.momenta):
            want = reference_step(p, q.grad, m, lr, 0.95, True, 0.01, "match_rms_adamw", clip)
            # the clip goes by a float32 sum of 10^5 .. 10^6 squares
            assert float((n.double() - want[1]).norm()) <= 1e-4 * float(want[1].norm())
            check_step(q.detach(), want[1].float(), want, torch.float32)
            moved += float((q.detach() - p).norm())
        assert moved > 0.0
    assert runner.disabled is None and runner.stats["replays"] >= 4
    assert t.matrices.step_count == t.fields.step_count == eager.fields.step_count
    for a, b in losses:
        assert abs(a - b) <= 1e-3 * abs(a), losses


@pytest.mark.parametrize("graphed", [False, True])
def test_data_parallel_steps_exchange_every_group(dev, monkeypatch, graphed):
    """Data-parallel steps with Muon, the other rank's part of a sum taken to be half of this one's: every value of every
    group's gradients is summed once a step, its mean is what the matrices are moved by."""
    from multimodalstudio_amd import ddp as mddp
    from multimodalstudio_amd import graphs
    from multimodalstudio_amd import pipeline as pl
    cfg = pl.TrainConfig(method="grid", modalities=("rgb",), num_rays_per_modality=256, log2T=12, n_views=10, width=64,
                         height=48, optimizer="muon")
    t = pl.Trainer(cfg, dev)
    t.set_step(95000)
    summed, done = [], []

    class Work:
        def wait(self):
            done.append(1)

    def all_reduce(buf, op=None, async_op=False):
        assert async_op and buf.is_contiguous()
        summed.append((buf.data_ptr(), buf.numel()))
        buf.mul_(1.5)
        return Work()
    monkeypatch.setattr(mddp.dist, "all_reduce", all_reduce)
    ddp = mddp.DDP(2, bucket_bytes=1 << 16)
    means = []
    finish = ddp.finish_step

    def spy(groups):
        before = {id(g): g.grad.clone() for g in groups}
        n = len(summed)
        finish(groups)
        late = {id(g): [(p, k) for p, k in summed[n:]] for g in groups}
        for g in groups:
            want = 0.5 * before[id(g)]     # summed while the backward ran: the mean is left
            for p, k in late[id(g)]:
                off = (p - g.grad.data_ptr()) // 4
                if 0 <= off < g.grad.numel():
                    want[off:off + k] = 0.75 * before[id(g)][off:off + k]
            assert (g.grad - want).abs().max() <= 2.0 ** -22 * want.abs().max()
        means.append([g.grad.clone() for g in groups])
    monkeypatch.setattr(ddp, "finish_step", spy)
    runner = graphs.GraphTrainer(t, granule=64, neighbours=0, ddp=ddp) if graphed else None
    for k in range(5):
        summed.clear()
        done.clear()
        before = [p.detach().clone() for p in t.matrices.params]
        momenta = [m.clone() for m in t.matrices.momenta]
        lr = 1e-3 * pl.lr_factor(t.step, cfg.max_iters)
        if graphed:
            runner.step()
        else:
            t.train_step(ddp=ddp)
        torch.cuda.synchronize()
        assert len(means[-1]) == 3 and len(done) == len(summed)
        covered = sorted(summed)
        for g in t.groups:
            at = g.grad.data_ptr()
            for p, n in covered:
                if at <= p < g.grad.data_ptr() + 4 * g.grad.numel():
                    assert p == at
                    at = p + 4 * n
            assert at == g.grad.data_ptr() + 4 * g.grad.numel()
        assert all(torch.equal(g.grad, m) for g, m in zip(t.groups, means[-1]))
        clip = min(1.0, 2.0 / (sum(float(g.grad.double().square().sum()) for g in (t.fields, t.matrices)) ** 0.5 + 1e-6))
        for p, q, m, n in zip(before, t.matrices.params, momenta, t.matrices.momenta):
            want = reference_step(p, q.grad, m, lr, 0.95, True, 0.01, "match_rms_adamw", clip)
            assert float((n.double() - want[1]).norm()) <= 1e-4 * float(want[1].norm())
            check_step(q.detach(), want[1].float(), want, torch.float32)
    if graphed:
        assert runner.disabled is None and runner.stats["replays"] >= 2, (runner.disabled, runner.stats)

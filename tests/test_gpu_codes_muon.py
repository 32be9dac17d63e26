"""The parameter operators where the framework uses them: per-view codes into a radiance field, its matrices stepped by
Muon and its tables by AdamW (pipeline.MuonGroup beside FlatGroup), the trainer with ``optimizer="muon"``."""
import pytest
import torch

from test_gpu_muon import check_step, reference_step

pytestmark = pytest.mark.gpu


def _field_and_codes(dev, views=45, dim=32):
    from multimodalstudio_amd import plugins as pg
    torch.manual_seed(3)
    codes = pg.EmbeddingEncodingConfig(num_embeddings=views, embedding_dim=dim, init_scale=0.1, scale=2.0,
                                       padding_index=0).setup().to(dev)
    grid = pg.FeatureGridConfig(encoding=pg.HashEncodingConfig(log2_hashmap_size=12))
    mlp = pg.mm.MLPConfig(num_layers=3, hidden_dim=64, out_activation="Sigmoid")
    cfg = pg.RadianceFieldConfig(base_field=pg.FeatureGridAndMLPConfig(feature_grid=grid, mlp_head=mlp))
    field = pg.RadianceField(cfg, 3, 3, dim, 3).to(dev)
    return field, codes


def _batch(dev, n=700, views=45, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.rand(n, 3, device=dev, generator=g) - 0.5
    d = torch.nn.functional.normalize(torch.randn(n, 3, device=dev, generator=g), dim=-1)
    cams = torch.randint(0, views, (n, 3), device=dev, generator=g, dtype=torch.int32)[:, :1]
    return x, d, cams, torch.rand(n, 3, device=dev, generator=g)


def test_codes_in_a_radiance_field(dev):
    """The codes' gradient through the field against torch's own lookup in the same field; the padding code has none."""
    field, codes = _field_and_codes(dev)
    assert codes.get_out_dim() == 32 and (codes.table[0] == 0).all()
    x, d, cams, target = _batch(dev)
    out = field(x, d, codes(cams))
    ((out - target) ** 2).mean().backward()
    own = codes.table.grad.clone()
    plain = codes.table.detach().clone().requires_grad_()
    other = field(x, d, 2.0 * plain[cams[:, 0].long()])
    assert torch.equal(out, other)
    (rows,) = torch.autograd.grad(((other - target) ** 2).mean(), plain)
    rows[0] = 0.0
    # two float32 sums of the same values in different orders, at most 40 of them a row: 40 half steps of their size
    assert (own - rows).abs().max() <= 40 * 2.0 ** -24 * 40 * rows.abs().max()
    assert (own[0] == 0).all() and own[1:].abs().sum() > 0
    for bad in (cams[:, 0], cams.expand(-1, 2)):
        with pytest.raises(ValueError):
            codes(bad)


def test_codes_field_and_both_optimizers(dev):
    """Three steps of codes + field: the matrices as Muon's definition moves them on the step's gradients, clipped by
    their group's norm; the tables, biases and norms by AdamW as torch does."""
    from multimodalstudio_amd import pipeline as pl
    field, codes = _field_and_codes(dev)
    model = torch.nn.ModuleDict({"field": field, "codes": codes})
    mats = pl.muon_matrices(model)
    assert [tuple(p.shape) for p in mats] == [(64, 38 + 32), (64, 64), (3, 64)]
    rest = [p for p in model.parameters() if not any(p is q for q in mats)]
    assert any(p is codes.table for p in rest)
    groups = [pl.FlatGroup(rest, lr=1e-3, weight_decay=0.01, eps=1e-15),
              pl.MuonGroup(mats, lr=1e-3, weight_decay=0.01)]
    ref = [p.detach().clone().requires_grad_() for p in rest]
    adamw = torch.optim.AdamW(ref, lr=1e-3, weight_decay=0.01, eps=1e-15)
    for t in range(3):
        for g in groups:
            g.zero_grad()
        x, d, cams, target = _batch(dev, seed=t)
        # the second step's gradients are large: the clip is active
        (((field(x, d, codes(cams)) - target) ** 2).mean() * (1.0 if t != 1 else 1e4)).backward()
        for g in groups:
            g.check_grads_attached()
        norm = float(torch.stack([p.grad.double().square().sum() for p in mats]).sum().sqrt())
        clip = min(1.0, 2.0 / (norm + 1e-6))
        assert (clip < 1.0) == (t == 1)
        want = [reference_step(p.detach(), p.grad, m, 1e-3, 0.95, True, 0.01, "match_rms_adamw", clip)
                for p, m in zip(mats, groups[1].momenta)]
        for a, b in zip(ref, rest):
            a.grad = b.grad.clone()
        torch.nn.utils.clip_grad_norm_(ref, 2.0)
        adamw.step()
        for g in groups:
            g.step(1.0)
        for p, m, w in zip(mats, groups[1].momenta, want):
            # the clip's own scale is a float32 quotient of a float32 norm: a few half steps more on the momentum
            wp, wm, update, u = w
            assert float((m.double() - wm).norm()) <= 8 * 2.0 ** -24 * float(wm.norm())
            check_step(p.detach(), wm.float(), w, torch.float32)
        for a, b in zip(ref, rest):
            assert (a - b).abs().max() <= 2e-6 * a.abs().max()


@pytest.mark.parametrize("banked", [False, True])
def test_muon_group_captured_equals_eager(dev, banked):
    """MuonGroup's captured form (device scalars; alone and in an OptimBank beside an AdamW group) against its eager
    step: the same weights and momenta, within two half steps of the scalars' rounding."""
    from multimodalstudio_amd import pipeline as pl
    gen = torch.Generator().manual_seed(2)
    shapes = [(256, 71), (257, 256), (3, 64)]
    p0 = [torch.randn(s, generator=gen) * 0.1 for s in shapes]
    v0 = torch.randn(130, generator=gen)
    grads = [[torch.randn(s, generator=gen) for s in shapes] for _ in range(3)]
    runs = []
    for captured in (False, True):
        ps = [torch.nn.Parameter(p.clone().to(dev)) for p in p0]
        vec = torch.nn.Parameter(v0.clone().to(dev))
        mu = pl.MuonGroup(ps, lr=1e-2, weight_decay=0.1)
        ad = pl.FlatGroup([vec], lr=1e-3, weight_decay=0.01, eps=1e-15)
        bank = pl.OptimBank([ad, mu]) if captured and banked else None
        for t, gs in enumerate(grads):
            if bank is not None:
                bank.zero_grads()
            else:
                mu.zero_grad()
                ad.zero_grad()
            for p, g in zip(ps, gs):
                p.grad.copy_(g.to(dev))
            vec.grad.fill_(0.5)
            f = 1.0 / (t + 1)
            if bank is not None:
                bank.load_hyper(f)
                bank.step_captured()
            elif captured:
                for g in (mu, ad):
                    g.load_hyper(f)
                    g.step_captured()
            else:
                for g in (mu, ad):
                    g.step(f)
        torch.cuda.synchronize()
        assert mu.step_count == 3 and mu.v is None
        runs.append([mu.flat.clone(), mu.m.clone(), ad.flat.clone()])
    for a, b in zip(*runs):
        # sums of squares by float atomics: the clip may differ by some half steps
        assert (a - b).abs().max() <= 16 * 2.0 ** -24 * a.abs().max()


def test_trainer_with_muon(dev):
    """The trainer's eager and graph-replayed steps with Muon: the grouping, the step counts and a finite loss; the
    replayed steps move the matrices as eager ones do."""
    from multimodalstudio_amd import pipeline as pl
    from multimodalstudio_amd.graphs import GraphTrainer
    cfg = pl.TrainConfig(num_rays_per_modality=256, log2T=12, width=64, height=48, n_views=20, optimizer="muon",
                         gpu_sampler=True)
    t = pl.Trainer(cfg, dev)
    assert len(t.matrices.params) == 18 and t.groups == [t.fields, t.matrices, t.poses]
    names = {id(p): n for n, p in t.model.named_parameters()}
    assert all(names[id(p)].endswith("original1") for p in t.matrices.params)
    assert sum(p.numel() for p in t.model.parameters()) == t.fields.n + t.matrices.n
    t.set_step(9500)
    before = t.matrices.flat.clone()
    _, total, _ = t.train_step()
    assert torch.isfinite(total).all() and t.matrices.step_count == 1
    moved = (t.matrices.flat - before).norm()
    assert moved > 0
    g = GraphTrainer(t, neighbours=0)
    t.set_step(95000)
    for _ in range(4):
        _, total = g.step()
        torch.cuda.synchronize()
        assert torch.isfinite(total).all()
    assert g.disabled is None and g.stats["replays"] >= 2, (g.disabled, g.stats)
    # a step is queued ahead of the replays: its scalars count
    assert t.matrices.step_count == t.fields.step_count and t.matrices.step_count >= 5
    assert torch.isfinite(t.matrices.flat).all()
    with pytest.raises(ValueError):
        pl.Trainer(pl.TrainConfig(num_rays_per_modality=16, log2T=12, width=64, height=48, n_views=20,
                                  optimizer="sgd"), dev)

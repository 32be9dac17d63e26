"""Calls of the row tables' operators beside the plain ones of test_gpu_embedding.py: what they write, and what they
refuse to."""
import pytest
import torch

from test_gpu_embedding import check

pytestmark = pytest.mark.gpu


@pytest.fixture()
def gen(dev):
    return torch.Generator(device="cuda").manual_seed(61)


@pytest.mark.parametrize("n", [100, 1000])
def test_backward_passes_notice_the_gradient_written_into_a_tensor(dev, gen, n):
    from multimodalstudio_amd import hip_ops
    ids = torch.randint(0, 300, (n,), device="cuda", generator=gen)
    dout, out = torch.randn(n, 16, device="cuda", generator=gen), torch.randn(300, 16, device="cuda", generator=gen)
    w = torch.randn(300, 16, device="cuda", generator=gen, requires_grad=True)
    loss = (out * w).sum()
    hip_ops.embedding_backward(ids, dout, 300, out=out)
    check(out, ids, dout, 300)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


@pytest.mark.parametrize("n,dim", [(9000, 1025), (20000, 1024), (70000, 1024), (70001, 1027)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_lookups_through_the_caches_and_past_them(dev, gen, n, dim, dtype):
    """Outputs below 33 MB, between that and 128 MB, and larger ones, rows of whole pieces and others."""
    from multimodalstudio_amd import hip_ops
    table = torch.randn(700, dim, device="cuda", generator=gen).to(dtype)
    ids = torch.randint(-2, 703, (n,), device="cuda", generator=gen)
    want = (table[ids.clamp(0, 699)].float() * 0.3).to(dtype)
    want[(ids < 0) | (ids >= 700)] = 0
    assert torch.equal(hip_ops.embedding(ids, table, 0.3), want)


@pytest.mark.parametrize("column", [False, True])
def test_lookups_of_more_than_2_to_24_indices(dev, gen, column):
    from multimodalstudio_amd import hip_ops
    n = 2 ** 24 + 77
    coords = torch.randint(-1, 60, (n, 2), device="cuda", generator=gen, dtype=torch.int32)
    ids = coords[:, 1] if column else coords[:, 1].contiguous()
    table = torch.randn(59, 3, device="cuda", generator=gen).half()
    out = hip_ops.embedding(ids, table, 1.5)
    want = (table[ids.clamp(0, 58).long()].float() * 1.5).half()
    want[(ids < 0) | (ids >= 59)] = 0
    assert torch.equal(out, want)
    # the gradient sorts at most 2^24 - 1 positions: refused before the forward pass, not after it
    with pytest.raises(ValueError, match="indices"):
        hip_ops.EmbeddingFunction.apply(ids, table.requires_grad_())
    assert hip_ops.EmbeddingFunction.apply(ids, table.detach()).shape == (n, 3)
    with pytest.raises(RuntimeError, match="indices"):
        hip_ops.embedding_backward(ids, out, 59)

"""Calls of the row tables' operators beside the plain ones of test_gpu_embedding.py: what they write, and what they
refuse to."""
import pytest
import torch

from test_gpu_embedding import check, draw_ids

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


# A sort by one block (129 .. 4096 positions) in one, two and three digits of the row: 1023 rows are one digit's last,
# 2^20 - 1 two digits'; its ends, one position more (several blocks), some positions beside its 64-lane rounds
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n,rows,dim", [
    (129, 1023, 40), (129, 50257, 33), (1024, 1024, 40), (1025, 32000, 130), (2047, 32000, 7), (2500, 1048575, 3),
    (2500, 1048576, 3), (3000, 2097153, 2), (4095, 131072, 8), (4096, 131072, 8), (4097, 131072, 8), (4096, 1025, 771),
])
@pytest.mark.parametrize("kind", ["uniform", "skewed", "outside", "same", "reversed"])
def test_one_block_sort(dev, gen, n, rows, dim, dtype, kind):
    from multimodalstudio_amd import hip_ops
    ids = draw_ids(kind, n, rows, gen)
    dout = torch.randn(n, dim, device="cuda", generator=gen).to(dtype)
    got = hip_ops.embedding_backward(ids, dout, rows, 0.6)
    check(got, ids, dout, rows, 0.6)
    assert torch.equal(got, hip_ops.embedding_backward(ids.int(), dout, rows, 0.6))
    # padding that holds what must reach nothing, into columns of a wider buffer
    pad = int(ids[n // 3].clamp(0, rows - 1))
    dirty = torch.where((ids == pad)[:, None], torch.full((), float("nan"), dtype=dtype, device="cuda"), dout)
    buf = torch.full((rows, dim + 5), 7.0, dtype=dtype, device="cuda")
    hip_ops.embedding_backward(ids, dirty, rows, 0.6, padding_idx=pad, out=buf[:, 2:2 + dim])
    check(buf[:, 2:2 + dim], ids, torch.nan_to_num(dirty, 0.0), rows, 0.6, pad)
    assert (buf[:, :2] == 7).all() and (buf[:, 2 + dim:] == 7).all()


@pytest.mark.parametrize("n", [100, 600])
def test_gradient_written_where_it_is_read(dev, gen, n):
    """Refused; into other columns of the same buffer it is right."""
    from multimodalstudio_amd import hip_ops
    buf = torch.randn(n, 48, device="cuda", generator=gen)
    ids = torch.randint(0, n, (n,), device="cuda", generator=gen)
    keep = buf.clone()
    for dout, out in ((buf, buf), (buf[:, :20], buf[:, 19:39])):
        for accumulate in (False, True):
            with pytest.raises(ValueError, match="share"):
                hip_ops.embedding_backward(ids, dout, n, out=out, accumulate=accumulate)
    assert torch.equal(buf, keep)
    hip_ops.embedding_backward(ids, buf[:, :20], n, out=buf[:, 20:40])
    check(buf[:, 20:40], ids, keep[:, :20], n)
    assert torch.equal(buf[:, :20], keep[:, :20]) and torch.equal(buf[:, 40:], keep[:, 40:])

"""Which outputs of embedding_backward share memory with the gradient that it reads (decided on the host)."""
import pytest
import torch

from multimodalstudio_amd import hip_ops


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_that_share_memory(dtype):
    buf = torch.zeros(20, 16, dtype=dtype)
    flat = buf.view(-1)
    for a, b in ((buf, buf), (buf[:10], buf[9:]), (buf[:, :9], buf[:, 8:]), (buf, flat[300:310].view(2, 5)),
                 (buf[::2], buf[:4]), (buf[:, :8].reshape(2, 10, 8), buf), (buf, buf[:1].expand(20, 16)),
                 (buf[:, 4:12], flat[12:12 + 320 - 16].view(19, 16)[:, :9])):
        assert hip_ops._rows_overlap(a, b) == hip_ops._rows_overlap(b, a)
    for a, b in ((buf, buf), (buf[:10], buf[9:]), (buf[:, :9], buf[:, 8:]), (buf, flat[300:310].view(2, 5)),
                 (buf, buf[:1].expand(20, 16)), (buf[::2], buf[:4])):
        assert hip_ops._rows_overlap(a, b)
    for a, b in ((buf, torch.zeros_like(buf)), (buf[:10], buf[10:]), (buf[:, :8], buf[:, 8:]), (buf[:, 8:], buf[:, :8]),
                 (buf[3:, 2:5], buf[:7, 5:]), (buf, buf[:0])):
        assert not hip_ops._rows_overlap(a, b) and not hip_ops._rows_overlap(b, a)

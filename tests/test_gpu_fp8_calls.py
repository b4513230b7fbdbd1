"""Calls of the 8-bit operators at the edges of what they take: addresses, strides,
numbers of rows and outputs, scales far from one."""
import pytest
import torch

from conftest import announce
from test_gpu_fp8 import BF16, F32, rnd

pytestmark = pytest.mark.gpu


def flat(t, offset):
    """The same values as a contiguous view into a flat buffer, `offset` elements in."""
    buf = torch.empty(t.numel() + offset, device="cuda", dtype=t.dtype)
    buf[offset:] = t.flatten()
    return buf[offset:].view(t.shape)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_of_views_into_flat_buffers(gpu, dtype):
    from mogt_amd import ops
    announce(f"add_rmsnorm_fp8 at odd addresses {dtype}")
    x, z, w = rnd(5, 260, seed=1), rnd(5, 260, seed=2, dtype=dtype), 1 + 0.1 * rnd(260, seed=3)
    want = ops.add_rmsnorm_fp8(x, z, 0.7, w)
    for i, j, k in ((1, 0, 0), (0, 1, 0), (0, 0, 3), (2, 3, 1)):
        got = ops.add_rmsnorm_fp8(flat(x, i), flat(z, j), 0.7, flat(w, k))
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))

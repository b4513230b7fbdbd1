"""Calls of the 8-bit operators at the edges of what they take: addresses, strides,
numbers of rows and outputs, scales far from one."""
import pytest
import torch

from conftest import announce
from test_gpu_fp8 import BF16, F32, product, rnd

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


def test_product_of_one_row_of_each_long_sequence(gpu):
    """Rows further apart than a tile's offsets reach, for few rows and for many,
    and a single row, whose stride is any number."""
    from mogt_amd import ops
    announce("linear_fp8 of the last rows of long sequences")
    L, K = 2304, 2048
    x, xs, w, ws = product(40, 130, K, seed=1)
    wide, scales = torch.zeros(40, L, K, device="cuda", dtype=x.dtype), torch.zeros(40, L, K // 128, device="cuda")
    wide[:, -1], scales[:, -1] = x, xs
    for M in (1, 2, 32, 33, 40):
        assert wide[:M, -1].stride(0) == L * K > 1 << 22
        for out in (F32, BF16):
            got = ops.linear_fp8(wide[:M, -1], scales[:M, -1], w, ws, out_dtype=out)
            assert torch.equal(got, ops.linear_fp8(x[:M].contiguous(), xs[:M].contiguous(), w, ws, out_dtype=out))

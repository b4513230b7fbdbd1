"""Calls of the 8-bit operators at the edges of what they take: addresses, strides,
numbers of rows and outputs, scales far from one."""
import pytest
import torch

from conftest import announce
from test_gpu_fp8 import BF16, F32, F8, check_product, product, rnd

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


def check_whole_range(y, x, xs, w, ws):
    """As check_product, with no more slack than the output's least step."""
    K, N = x.shape[-1], w.shape[0]
    xd = x.double() * xs.double().repeat_interleave(128, -1)[..., :K]
    wd = w.double() * ws.double().repeat_interleave(128, 1)[:, :K].repeat_interleave(128, 0)[:N]
    want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    lim = (K + 4) * 2.0 ** -24 * mag
    if y.dtype == BF16:
        lim = lim + 2.0 ** -13 * mag
        lim = lim + 2.0 ** -8 * (want.abs() + lim)
    least = 2.0 ** -149 if y.dtype == F32 else 2.0 ** -133
    err = (y.double() - want).abs()
    assert bool((err <= lim + least).all()), f"{float((err / (lim + least)).max()):.3g} of the bound"
    return want


@pytest.mark.parametrize("M", [5, 30, 40, 700, 4100])
@pytest.mark.parametrize("out", [F32, BF16])
def test_scales_far_from_one(gpu, M, out):
    """The scales' product below fp32's normal numbers, or above its largest, where
    the result is an ordinary number."""
    from mogt_amd import ops
    announce(f"linear_fp8 far scales {M} {out}")
    N, K = 1300, 400
    x, xs, w, ws = product(M, N, K, seed=3)
    # rows of 1e-36 (scales of 2^-126) and weights of 0.02 (4.5e-5)
    small, small_s = ops.quantize_fp8(rnd(M, K, seed=1) * 1e-36)
    light, light_s = ops.quantize_fp8(rnd(N, K, seed=2) * 0.02, block_rows=128)
    assert float((small_s.max().double() * light_s.max().double()).item()) < 2.0 ** -126
    want = check_whole_range(ops.linear_fp8(small, small_s, light, light_s, out_dtype=out), small, small_s, light, light_s)
    assert float(want.abs().median()) > 2.0 ** -124
    # scales up to 2^+-110 that cancel
    g = torch.Generator(device="cuda").manual_seed(5)
    e = torch.randint(-110, 111, (xs.shape[1],), generator=g, device="cuda")
    r = torch.randint(-9, 10, (M, 1), generator=g, device="cuda")
    xe, we = torch.exp2((r - e).float()), torch.exp2(e.float()).expand_as(ws)
    check_whole_range(ops.linear_fp8(x, xe, w, we.contiguous(), out_dtype=out), x, xe, w, we)
    # a block whose scales' product is beyond fp32 and whose sums are zero for some outputs
    zero = w.clone().view(torch.uint8)
    zero[::3, 128:256] = 0
    zero = zero.view(w.dtype)
    rest = [i for i in range(K) if not 128 <= i < 256]
    xd = x.double() * xs.double().repeat_interleave(128, -1)[..., :K]
    wd = zero.double() * ws.double().repeat_interleave(128, 1)[:, :K].repeat_interleave(128, 0)[:N]
    want, mag = xd[:, rest] @ wd[::3, rest].t(), xd[:, rest].abs() @ wd[::3, rest].abs().t()
    lim = (K + 4) * 2.0 ** -24 * mag + (2.0 ** -12 * mag + 2.0 ** -8 * want.abs() if out == BF16 else 0.0)
    for far in (2.0 ** 20, 2.0 ** 103):
        xl, wl = xs.clone(), ws.clone()
        xl[:, 1], wl[:, 1] = 2.0 ** 119, far
        y = ops.linear_fp8(x, xl, zero, wl, out_dtype=out)
        assert bool(((y[:, ::3].double() - want).abs() <= lim + 1e-30).all())
        wl[:, 1] = float("inf")   # as the definition: infinity times nothing
        assert bool(ops.linear_fp8(x, xl, zero, wl, out_dtype=out)[:, ::3].isnan().all())
    # the quantiser's largest and least scales: nothing times them is nothing
    for a, b in ((torch.finfo(F32).max / 448, 2.0 ** 103), (2.0 ** 110, torch.finfo(F32).max / 448), (2.0 ** -126, 2.0 ** -126)):
        assert not ops.linear_fp8(torch.zeros_like(x), torch.full_like(xs, a), w, torch.full_like(ws, b), out_dtype=out).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_rows_than_a_launch_has_threads_along_x(gpu, dtype):
    from mogt_amd import ops
    for rows in ((1 << 26) + 5, (1 << 27) + 19):
        announce(f"8 bits, {rows} rows of 4 {dtype}")
        x, z, w = rnd(rows, 4, seed=1), rnd(rows, 4, seed=2, dtype=dtype), 1 + 0.1 * rnd(4, seed=3)
        for got, want in ((ops.add_rmsnorm_fp8(x, z, 0.5, w), lambda at: ops.add_rmsnorm_fp8(x[at], z[at], 0.5, w)),
                          (ops.quantize_fp8(z), lambda at: ops.quantize_fp8(z[at]))):
            for at in (slice(0, 300), slice(rows // 2, rows // 2 + 300), slice(rows - 300, rows)):
                assert all(torch.equal(a[at].float(), b.float()) for a, b in zip(got, want(at)))
        del x, z, got
        torch.cuda.empty_cache()


@pytest.mark.parametrize("M", [1, 17])
def test_more_outputs_than_a_launch_has_threads_along_x(gpu, M):
    from mogt_amd import ops
    N, K = (1 << 28) + 272, 16
    announce(f"linear_fp8 {M} rows by {N} outputs")
    x, xs = ops.quantize_fp8(rnd(M, K, seed=1))
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randint(0, 0x70, (N, K), generator=g, device="cuda", dtype=torch.uint8).view(F8)
    ws = torch.rand(-(-N // 128), 1, generator=g, device="cuda") + 0.5
    y = ops.linear_fp8(x, xs, w, ws)
    for a in (0, N // 256 * 128, N - 272):
        b = min(a + 384, N)
        assert torch.equal(y[:, a:b], ops.linear_fp8(x, xs, w[a:b], ws[a // 128:-(-b // 128)]))


@pytest.mark.parametrize("dtype,scale", [(F32, 0.3), (F32, 0.5), (BF16, 0.3)])
def test_norm_and_its_scales_are_the_definition_s(gpu, dtype, scale):
    """The norm is in 64 bits: a block's scale is off by its rounding to fp32, 2^-24 of
    it, and no value falls on the other side of a border (one in 2^45 might).  bf16 z is
    scaled in fp32 and rounded, fp32 z enters unrounded."""
    from mogt_amd import ops
    announce(f"add_rmsnorm_fp8 against 64 bits {dtype} {scale}")
    M, D = 2048, 4096
    x, z, w = rnd(M, D, seed=11), rnd(M, D, seed=12, dtype=dtype), 1 + 0.2 * rnd(D, seed=13)
    _, q, s = ops.add_rmsnorm_fp8(x, z, scale, w, 1e-6)
    factor = torch.tensor(scale, device="cuda")
    added = factor.double() * z.double() if dtype == F32 else (factor * z.float()).bfloat16().double()
    v = x.double() + added
    n = (v * w.double()).view(M, 32, 128)
    most = n.abs().amax(2)
    want = most / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) / 448
    assert bool(((s.double() - want).abs() <= 2.0 ** -24 * (1 + 1e-6) * want).all())
    u = (448 * n / most.unsqueeze(2)).view(M, D)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    assert int((q.double() != torch.round(u / step) * step).sum()) == 0


@pytest.mark.parametrize("out", [F32, BF16])
def test_product_of_many_tiles_and_stages(gpu, out):
    from mogt_amd import ops
    announce(f"linear_fp8 4100 3500 2048 {out}")
    p = product(4100, 3500, 2048, seed=9)
    check_product(ops.linear_fp8(*p, out_dtype=out), *p)


@pytest.mark.parametrize("out", [F32, BF16])
def test_product_past_2_32_bytes(gpu, out):
    """Operand and output of more than 2^31 elements and 2^32 bytes, against the same
    products of a tile's rows."""
    from mogt_amd import ops
    M, N, K = 2_200_003, 1100, 2048
    announce(f"linear_fp8 {M} {N} {K} {out}")
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(0, 0x78, (M, K), generator=g, device="cuda", dtype=torch.uint8).view(F8)
    xs = torch.rand(M, K // 128, generator=g, device="cuda") + 0.5
    _, _, w, ws = product(1, N, K, seed=4)
    y = ops.linear_fp8(x, xs, w, ws, out_dtype=out)
    for a in (0, (1 << 31) // N - 50, (1 << 32) // K - 50, M - 99):
        assert torch.equal(y[a:a + 99], ops.linear_fp8(x[a:a + 99], xs[a:a + 99], w, ws, out_dtype=out))
    del x, xs, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,out", [(1, F32), (1, BF16), (16, BF16), (17, F32), (32, BF16), (40, F32), (700, F32), (4100, F32)])
def test_products_that_cancel_add_in_fp32(gpu, M, out):
    """Whole numbers whose sums stay below 2^24 are exact in fp32 in any order: 32 pairs
    of 2^16 to 448 * 448 that cancel, and between them 64 products of up to 9 that are
    left.  (The 8-bit instruction drops what lies below 2^-14 of the largest product.)"""
    from mogt_amd import ops
    announce(f"linear_fp8 products that cancel {M} {out}")
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g, device="cuda").float()  # noqa: E731
    N, K = 300, 384
    x, w = r(-3, 3, M, K // 128, 128), r(-3, 3, N, K // 128, 128)
    x[..., ::4], w[..., ::4] = 32 * r(8, 14, M, K // 128, 32), 32 * r(8, 14, N, K // 128, 32)
    x[..., 1::4], w[..., 1::4] = x[..., ::4], -w[..., ::4]
    x, w = x.view(M, K).to(F8), w.view(N, K).to(F8)
    y = ops.linear_fp8(x, torch.ones(M, 3, device="cuda"), w, torch.ones(3, 3, device="cuda"), out_dtype=out)
    assert torch.equal(y.double(), (x.double() @ w.double().t()).to(out).double())

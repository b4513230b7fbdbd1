"""8-bit rows and weights (``ops.add_rmsnorm_fp8``, ``ops.quantize_fp8``) and
their product (``ops.linear_fp8``) against the definitions in 64 bits.

Tolerances, derived: a scale is a quotient of an fp32 value, one rounding, 2^-24
of it, and in the norm that value's own: the residual's 1, the statistics' D / 2 + 4
(a squared sum of D terms under a root, the reciprocal root's 2 ulp) and 2
products: (D / 2 + 8) 2^-24.  A value x / scale carries those and its quotient's,
and is rounded to e4m3: half a step, 2^-4 of it, or 2^-10 where steps are 2^-9; where
the 64-bit value lies within its own error of a border the other neighbour is as
right, so a value may be off by half a step and twice that error.  A product in
fp32 adds K + 4 roundings of the sum S of its terms' absolute values, and with the
8-bit instruction 2^-13 S: an instruction aligns the products that it adds to the
largest and drops what lies below 2^-14 or so of it, from each of them at most."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu
F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24


def rnd(*s, seed=0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*s, generator=g, device="cuda").to(dtype)


def check_eight(n, q, scale, rows, rel):
    """q, scale against the float64 values n [M, D], known to `rel`, in blocks of
    `rows` by 128."""
    M, D = n.shape
    q, scale = q.double().cpu(), scale.double().cpu()
    for i, r in enumerate(n.split(rows)):
        for j, b in enumerate(r.split(128, 1)):
            s = max(float(b.abs().max()) / 448, 2.0 ** -126)
            got = float(scale[i, j])
            assert abs(got - s) <= (rel + U) * s
            u = b / got
            v = q[i * rows:i * rows + b.shape[0], j * 128:j * 128 + b.shape[1]]
            half = torch.maximum(u.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64))
            assert bool(((v - u).abs() <= half + 2 * (rel + 2 * U) * u.abs()).all())


@pytest.mark.parametrize("M,D", [(1, 4), (3, 128), (5, 132), (7, 256), (2, 260), (65, 768), (4, 1028), (9, 2048),
                                 (2, 2052), (3, 4096)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm(gpu, M, D, dtype):
    from mogt_amd import ops
    announce(f"add_rmsnorm_fp8 {M} {D} {dtype}")
    x, z, w = rnd(M, D, seed=1) * 3, rnd(M, D, seed=2, dtype=dtype), 1 + 0.2 * rnd(D, seed=3)
    x_out, q, s = ops.add_rmsnorm_fp8(x, z, 0.3, w, 1e-5)
    assert q.dtype == F8 and s.shape == (M, -(-D // 128))
    assert torch.equal(x_out, ops.add_rmsnorm(x, z, 0.3, w, 1e-5)[0])
    xd = x_out.double().cpu()
    n = xd / torch.sqrt((xd * xd).mean(1, keepdim=True) + 1e-5) * w.double().cpu()
    check_eight(n, q, s, 1, (D / 2 + 8) * U)


def test_norm_borders(gpu):
    """Values next to a border of two 8-bit values fall where the definition in 64
    bits puts them: of 8 million none elsewhere (in fp32 some 6 do; 64 bits are off by
    a few 2^-53 and a border is within that of one value in 2^45)."""
    from mogt_amd import ops
    announce("add_rmsnorm_fp8 borders")
    x, z, w = rnd(4096, 2048, seed=11), rnd(4096, 2048, seed=12, dtype=BF16), 1 + 0.2 * rnd(2048, seed=13)
    q = ops.add_rmsnorm_fp8(x, z, 0.5, w, 1e-6)[1].double()
    n = (x.double() + 0.5 * z.double()) * w.double()   # the root mean square cancels in a block
    u = (448 * n.view(4096, 16, 128) / n.view(4096, 16, 128).abs().amax(2, keepdim=True)).view(4096, 2048)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    assert int((q != torch.round(u / step) * step).sum()) == 0


@pytest.mark.parametrize("shape", [(1, 4), (3, 5, 128), (7, 132), (130, 4096), (3, 5124)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows(gpu, shape, dtype):
    from mogt_amd import ops
    announce(f"quantize_fp8 rows {shape} {dtype}")
    x = rnd(*shape, seed=4, dtype=dtype) * 50
    q, s = ops.quantize_fp8(x)
    assert q.shape == x.shape and s.shape == (*shape[:-1], -(-shape[-1] // 128))
    check_eight(x.double().cpu().reshape(-1, shape[-1]), q.reshape(-1, shape[-1]), s.reshape(-1, s.shape[-1]), 1, 0.0)
    wide = rnd(shape[0], shape[-1] + 3, seed=5, dtype=dtype)[:, 1:shape[-1] + 1]   # unaligned rows
    a, b = ops.quantize_fp8(wide), ops.quantize_fp8(wide.contiguous())
    assert torch.equal(a[0].float(), b[0].float()) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("M,D", [(1, 4), (127, 128), (129, 132), (300, 768), (128, 5120)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_blocks(gpu, M, D, dtype):
    from mogt_amd import ops
    announce(f"quantize_fp8 blocks {M} {D} {dtype}")
    x = rnd(M, D, seed=6, dtype=dtype) * torch.exp(rnd(M, 1, seed=7)).to(dtype)
    q, s = ops.quantize_fp8(x, block_rows=128)
    assert s.shape == (-(-M // 128), -(-D // 128))
    check_eight(x.double().cpu(), q, s, 128, 0.0)


def test_zeros_and_tiny_rows(gpu):
    """A block of zeros is zeros at the least scale, values below it do not divide
    by zero; what is not finite stays in its block."""
    from mogt_amd import ops
    x = torch.zeros(4, 256, device="cuda")
    x[1, :128] = 1e-38
    x[2, 5] = float("nan")
    x[3, 200] = float("inf")
    for rows in (1, 128):
        announce(f"quantize_fp8 special values, blocks of {rows}")
        q, s = ops.quantize_fp8(x, block_rows=rows)
        q = q.float()
        assert not q[0].any() and float(s[0, 0]) > 0
        assert bool(torch.isnan(q[2, 5])) and bool(torch.isnan(q[3, 200]))
        assert int(torch.isnan(q).sum()) == 2
    q, s = ops.quantize_fp8(x)
    assert float(s[1, 0]) == 2.0 ** -126 and bool((q[1, :128].float() - 1e-38 * 2.0 ** 126).abs().max() <= 2.0 ** -10 + 0.06)


def test_norm_special_values(gpu):
    """Rows below the least scale, of zeros, and with what is not finite: the last
    leave their own row only, a row with an infinity is zeros but for it (its norm is
    over an infinite root mean square), as the definition's."""
    from mogt_amd import ops
    announce("add_rmsnorm_fp8 special values")
    x, z, w = rnd(7, 516, seed=21), torch.zeros(7, 516, device="cuda"), 1 + 0.2 * rnd(516, seed=22)
    want = ops.add_rmsnorm_fp8(x, z, 1.0, w)
    bad = x.clone()
    bad[1] = 0.0
    bad[3, 130] = float("nan")
    bad[5, 200] = float("-inf")
    x_out, q, s = ops.add_rmsnorm_fp8(bad, z, 1.0, w)
    q = q.float()
    assert torch.equal(q[[0, 2, 4, 6]], want[1].float()[[0, 2, 4, 6]]) and torch.equal(s[[0, 2, 4, 6]], want[2][[0, 2, 4, 6]])
    assert not q[1].any() and bool((s[1] == 2.0 ** -126).all())
    assert bool(q[3].isnan().all())
    assert bool(q[5, 200].isnan()) and not q[5, [i for i in range(516) if i != 200]].any()
    # normalised values up to 3e-36: the scale is 2^-126 and steps are its e4m3 steps
    xo, q, s = ops.add_rmsnorm_fp8(x, z, 1.0, w * 1e-36)
    xd = xo.double()
    u = xd / torch.sqrt((xd * xd).mean(1, keepdim=True) + 1e-6) * (w * 1e-36).double() * 2.0 ** 126
    assert bool((s == 2.0 ** -126).all())
    assert bool(((q.double() - u).abs() <= torch.clamp(u.abs() * 2.0 ** -4, min=2.0 ** -10) * (1 + 1e-6)).all())


def product(M, N, K, seed=0):
    from mogt_amd import ops
    x, xs = ops.quantize_fp8(rnd(M, K, seed=seed) * torch.exp(rnd(M, 1, seed=seed + 1)))
    w, ws = ops.quantize_fp8(rnd(N, K, seed=seed + 2) / K ** 0.5, block_rows=128)
    return x, xs, w, ws


def check_product(y, x, xs, w, ws):
    K, N = x.shape[-1], w.shape[0]
    xd = x.double() * xs.double().repeat_interleave(128, -1)[..., :K]
    wd = w.double() * ws.double().repeat_interleave(128, 1)[:, :K].repeat_interleave(128, 0)[:N]
    want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    lim = (K + 4) * U * mag
    if y.dtype == BF16:
        lim = lim + 2.0 ** -13 * mag
        lim = lim + 2.0 ** -8 * (want.abs() + lim)
    err = (y.double() - want).abs()
    assert bool((err <= lim + 1e-30).all()), f"{float((err / (lim + 1e-30)).max()):.3g} of the bound"


@pytest.mark.parametrize("M,N,K", [
    (1, 1, 16), (1, 17, 128), (2, 130, 144), (15, 64, 768), (16, 129, 1024), (17, 16, 2048), (33, 300, 112),
    (64, 128, 640), (65, 128, 128), (66, 1, 16), (100, 131, 272), (129, 257, 384), (501, 300, 768), (1000, 5, 1040),
])
@pytest.mark.parametrize("out", [F32, BF16])
def test_product(gpu, M, N, K, out):
    from mogt_amd import ops
    announce(f"linear_fp8 {M} {N} {K} {out}")
    p = product(M, N, K)
    y = ops.linear_fp8(*p, out_dtype=out)
    assert y.dtype == out and y.shape == (M, N)
    check_product(y, *p)


@pytest.mark.parametrize("M,N,K", [(4100, 3500, 400), (3841, 4097, 256)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_product_of_many_tiles(gpu, M, N, K, out):
    from mogt_amd import ops
    announce(f"linear_fp8 {M} {N} {K} {out}")
    p = product(M, N, K, seed=9)
    check_product(ops.linear_fp8(*p, out_dtype=out), *p)


def test_product_layouts(gpu):
    """Leading dimensions, rows of a wider matrix, unaligned and transposed operands."""
    from mogt_amd import ops
    announce("linear_fp8 layouts")
    x, xs, w, ws = product(70, 96, 160)
    want = ops.linear_fp8(x, xs, w, ws)
    got = ops.linear_fp8(x.view(7, 10, 160), xs.view(7, 10, 2), w, ws)
    assert got.shape == (7, 10, 96) and torch.equal(got.view(70, 96), want)
    for pad in (16, 3):
        wide = torch.zeros(70, 160 + 2 * pad, device="cuda").to(F8)
        wide[:, pad:pad + 160] = x
        assert torch.equal(ops.linear_fp8(wide[:, pad:pad + 160], xs, w, ws), want)
    wt = torch.empty(160, 96, device="cuda", dtype=F8).copy_(w.t()).t()
    assert torch.equal(ops.linear_fp8(x, xs, wt, ws), want)
    assert ops.linear_fp8(x[:0], xs[:0], w, ws).shape == (0, 96)


def test_norm_feeds_the_product(gpu):
    """A projection after a residual norm, for a batch and for one token."""
    from mogt_amd import ops
    for M in (1, 200):
        announce(f"add_rmsnorm_fp8 into linear_fp8, {M} rows")
        x, z, weight = rnd(M, 768, seed=1), rnd(M, 768, seed=2, dtype=BF16), 1 + 0.1 * rnd(768, seed=3)
        w, ws = ops.quantize_fp8(rnd(320, 768, seed=4) / 768 ** 0.5, block_rows=128)
        _, q, s = ops.add_rmsnorm_fp8(x, z, 0.5, weight)
        check_product(ops.linear_fp8(q, s, w, ws), q, s, w, ws)


@pytest.mark.parametrize("M,N,K", [(4100, 3520, 400), (700, 2304, 272), (2600, 1032, 144), (33, 64, 1040), (16, 40, 16)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_product_of_whole_rows(gpu, M, N, K, out):
    """Outputs whose rows are whole 16 bytes leave through LDS: several tiles a
    work-group, edges inside a tile, blocks of K that are not full."""
    from mogt_amd import ops
    announce(f"linear_fp8 {M} {N} {K} {out}")
    p = product(M, N, K, seed=5)
    check_product(ops.linear_fp8(*p, out_dtype=out), *p)


@pytest.mark.parametrize("M,N,K", [(9000, 8200, 128), (20000, 4096, 256)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_product_of_several_tiles_a_work_group(gpu, M, N, K, out):
    """Against the same product of its rows in pieces small enough for one tile a
    work-group, whose blocks are added in the same order."""
    from mogt_amd import ops
    announce(f"linear_fp8 {M} {N} {K} {out}")
    x, xs, w, ws = product(M, N, K, seed=6)
    y = ops.linear_fp8(x, xs, w, ws, out_dtype=out)
    for lo in range(0, M, 4000):
        part = ops.linear_fp8(x[lo:lo + 100], xs[lo:lo + 100], w, ws, out_dtype=out)
        check_product(part, x[lo:lo + 100], xs[lo:lo + 100], w, ws)
        assert torch.equal(part, y[lo:lo + 100])
    check_product(y[-300:], x[-300:], xs[-300:], w, ws)


def test_product_neighbours_are_left_alone(gpu):
    """Rows behind the last and columns past the end of the output's memory."""
    from mogt_amd import _lib
    from mogt_amd import ops
    for M, N, K, out in ((70, 130, 144, BF16), (300, 520, 128, BF16), (129, 132, 128, F32), (5, 24, 32, F32), (4000, 3500, 128, BF16)):
        announce(f"mogt_linear_fp8 {M} {N} {K} {out}")
        x, xs, w, ws = product(M, N, K, seed=7)
        y = torch.full((M + 3, N), 7.0, device="cuda", dtype=out)
        rc = _lib.load().mogt_linear_fp8(x.data_ptr(), K, xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), M, N, K,
                                         1 if out == BF16 else 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(y[:M], ops.linear_fp8(x, xs, w, ws, out_dtype=out)) and bool((y[M:] == 7).all())


@pytest.mark.parametrize("N", [3502, 3501, 523, 262])
@pytest.mark.parametrize("out", [F32, BF16])
def test_product_of_rows_in_pieces(gpu, N, out):
    """Outputs whose rows are whole 2, 4 or 8 bytes: each tile's size, and rows behind the last."""
    from mogt_amd import _lib
    announce(f"linear_fp8 rows of {N} {out}")
    for M in (70, 700, 4100):
        p = product(M, N, 272, seed=9)
        x, xs, w, ws = p
        y = torch.full((M + 3, N), 7.0, device="cuda", dtype=out)
        rc = _lib.load().mogt_linear_fp8(x.data_ptr(), 272, xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), M, N, 272,
                                         1 if out == BF16 else 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and bool((y[M:] == 7).all())
        check_product(y[:M], *p)


def test_product_of_very_long_rows(gpu):
    """A tile's rows of the output more than 2^31 bytes apart in all."""
    from mogt_amd import ops
    announce("linear_fp8 long rows")
    N = 1 << 22
    x, xs, w, ws = product(40, N, 16, seed=10)
    y = ops.linear_fp8(x, xs, w, ws)
    for a, b in ((0, 384), (N - 384, N), (N // 2 - 128, N // 2 + 128)):
        assert torch.equal(y[:, a:b], ops.linear_fp8(x, xs, w[a:b], ws[a // 128:b // 128]))


def test_what_is_not_finite_stays_in_its_row(gpu):
    from mogt_amd import ops
    announce("linear_fp8 special values")
    for M in (5, 200):
        x, xs, w, ws = product(M, 96, 272, seed=8)
        want = ops.linear_fp8(x, xs, w, ws)
        bad = x.float()
        bad[3, 7] = float("nan")
        s = xs.clone()
        s[2, 1] = float("inf")
        got = ops.linear_fp8(bad.to(F8), s, w, ws)
        rest = [i for i in range(M) if i not in (2, 3)]
        assert torch.equal(got[rest], want[rest]) and not got[2:4].isfinite().any()


def test_empty(gpu):
    from mogt_amd import ops
    announce("8-bit operators, empty")
    w, ws = ops.quantize_fp8(torch.randn(40, 32, device="cuda"), block_rows=128)
    z = torch.zeros(0, 32, device="cuda")
    x, q, s = ops.add_rmsnorm_fp8(z, z, 1.0, torch.ones(32, device="cuda"))
    assert x.shape == q.shape == (0, 32) and s.shape == (0, 1)
    assert ops.linear_fp8(q, s, w, ws).shape == (0, 40)
    assert ops.linear_fp8(q, s, w[:0], ws[:0]).shape == (0, 0)
    assert [t.shape for t in ops.quantize_fp8(z, block_rows=128)] == [(0, 32), (0, 1)]
    assert [t.shape for t in ops.quantize_fp8(z.view(0, 4, 8))] == [(0, 4, 8), (0, 4, 1)]


def test_strides_of_the_norm_and_one_row(gpu):
    from mogt_amd import ops
    announce("add_rmsnorm_fp8 strides")
    x, z, w = rnd(4, 6, 256, seed=1), rnd(4, 6, 256, seed=2, dtype=BF16), rnd(256, seed=3)
    want = ops.add_rmsnorm_fp8(x, z, 0.7, w)
    far = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, z)]
    wide = torch.zeros(4, 6, 513, device="cuda", dtype=BF16)
    wide[..., 1:257] = z
    for a in (ops.add_rmsnorm_fp8(*far, 0.7, w), ops.add_rmsnorm_fp8(x, wide[..., 1:257], 0.7, w.double())):
        assert all(torch.equal(p.float(), r.float()) for p, r in zip(a, want))
    one = ops.add_rmsnorm_fp8(x[1, 2], z[1, 2], 0.7, w)
    assert one[2].shape == (2,) and all(torch.equal(p.float(), r[1, 2].float()) for p, r in zip(one, want))


def test_streams_and_captured_graphs(gpu):
    """Two streams at once, and a norm and its products captured and replayed on
    changing inputs with eager work between."""
    from mogt_amd import ops
    announce("8-bit operators captured")
    shapes = [(1, 768), (300, 768), (4200, 768)]
    w, ws = ops.quantize_fp8(rnd(3504, 768, seed=1) / 28, block_rows=128)
    weight = rnd(768, seed=2)

    def work(x, z):
        res, q, s = ops.add_rmsnorm_fp8(x, z, 0.5, weight)
        return res, q, s, ops.linear_fp8(q, s, w, ws), ops.linear_fp8(q, s, w, ws, out_dtype=F32)

    held = [(rnd(*s, seed=3), rnd(*s, seed=4, dtype=BF16)) for s in shapes]
    want = [work(*h) for h in held]
    streams = [torch.cuda.Stream() for _ in held]
    torch.cuda.synchronize()
    got = []
    for s, h in zip(streams, held):
        with torch.cuda.stream(s):
            got.append(work(*h))
    torch.cuda.synchronize()
    same = lambda a, b: all(torch.equal(p.float(), r.float()) for p, r in zip(a, b))  # noqa: E731
    assert all(same(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [work(*h) for h in held]
    for seed in range(10, 13):
        for x, z in held:
            x.copy_(rnd(*x.shape, seed=seed))
            z.copy_(rnd(*x.shape, seed=seed + 50, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, work(*h)) for a, h in zip(out, held))

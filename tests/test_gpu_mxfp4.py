"""MXFP4 on the GPU: quantisation against the definition in 64 bits, code for
code."""

import pytest
import torch

import lowbit

pytestmark = pytest.mark.gpu

BF, F16, F32, U8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8


def _x(M, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-9, 9, (M, 1), generator=g).float())
    x = x.to(dtype)
    # ties of the element grid, a block of zeros, one huge element
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.0])
    x[0, :16] = ties.to(dtype)
    x[0, 16:32] = (ties / 2).to(dtype)
    if K > 32:
        x[0, 32:64] = 0
        x[M - 1, K - 1] = 30000.0
    return x


def _check(x, got):
    out, scales, codes = got
    code, sc, val = lowbit.mxfp4(x)
    assert torch.equal(scales.cpu().long(), sc.long())
    assert torch.equal(codes.cpu(), lowbit.pack_nibbles(code))
    if out is not None:
        # the values are exact in fp32 and bf16 down to their smallest normal
        # numbers, in fp16 after one rounding
        want = val.to(x.dtype)
        assert torch.equal(out.cpu().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0)) and out.dtype == x.dtype


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,K", [(1, 32), (3, 64), (64, 4096), (7, 2080), (1025, 96), (300, 1056)])
def test_quant_matches_the_definition(cuda_dev, dtype, M, K):
    from dsv4attn import ops
    x = _x(M, K, dtype, M + K)
    _check(x, ops.mxfp4_quant(x.to(cuda_dev), out=True))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quant_range_ends(cuda_dev, dtype):
    """Maxima at every power of two of the type, denormal blocks, the largest
    number, NaN and infinities."""
    from dsv4attn import ops
    e = torch.arange(-133 if dtype == BF else -149, 128).double()
    x = torch.exp2(e).unsqueeze(1) * torch.linspace(-1, 1, 32, dtype=torch.float64)
    x = torch.cat([x, x * 1.99]).to(dtype)
    x[0] = torch.finfo(dtype).max
    x[1, 3] = float("nan")
    x[2, 31] = float("inf")
    x[3, 0] = float("-inf")
    x[4] = -0.0
    _check(x, ops.mxfp4_quant(x.to(cuda_dev), out=True))


def test_quant_strides_in_place_and_leading_dims(cuda_dev):
    from dsv4attn import ops
    big = _x(24, 640, BF, 5).to(cuda_dev)
    x = big[:, 64:64 + 256]                                   # a column slice
    code, sc, val = lowbit.mxfp4(x)
    wide = torch.full((24, 400), 7.0, dtype=BF, device=cuda_dev)
    _check(x.cpu(), ops.mxfp4_quant(x, out=wide[:, 8:264]))
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 264:] == 7).all())
    x3 = big.view(2, 3, 4, 640)
    out, scales, codes = ops.mxfp4_quant(x3)
    assert out is None and scales.shape == (2, 3, 4, 20) and codes.shape == (2, 3, 4, 320)
    _check(x3.cpu(), (None, scales, codes))
    ops.mxfp4_quant(x, out=x)                                 # in place, the columns beside it untouched
    torch.cuda.synchronize()
    assert torch.equal(x.cpu().double(), val)
    empty = ops.mxfp4_quant(torch.empty(0, 64, dtype=BF, device=cuda_dev), out=True)
    assert empty[0].shape == (0, 64) and empty[2].shape == (0, 32)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,K", [(1, 32), (65, 96), (4000, 4096)])
def test_quant_in_place_is_quant(cuda_dev, dtype, M, K):
    """out = x, whole rows and a column slice, gives what a separate out does."""
    from dsv4attn import ops
    x = _x(M, K, dtype, 3 * M + K).to(cuda_dev)
    out, scales, codes = ops.mxfp4_quant(x, out=True)
    wide = torch.full((M, K + 64), 7.0, dtype=dtype, device=cuda_dev)
    wide[:, 32:32 + K] = x
    for buf in (x.clone(), wide[:, 32:32 + K]):
        got, s, c = ops.mxfp4_quant(buf, out=buf)
        torch.cuda.synchronize()
        assert got.data_ptr() == buf.data_ptr()
        assert torch.equal(buf, out) and torch.equal(s, scales) and torch.equal(c, codes)
    assert bool((wide[:, :32] == 7).all()) and bool((wide[:, 32 + K:] == 7).all())


def test_quant_refusals(cuda_dev):
    from dsv4attn import ops
    d = cuda_dev
    with pytest.raises(ValueError, match="32"):
        ops.mxfp4_quant(torch.zeros(2, 48, dtype=BF, device=d))
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        ops.mxfp4_quant(torch.zeros(2, 64, dtype=torch.float64, device=d))
    with pytest.raises(ValueError, match="unit stride"):
        ops.mxfp4_quant(torch.zeros(64, 64, dtype=BF, device=d).t()[:, :32])
    with pytest.raises(ValueError, match="rows"):
        ops.mxfp4_quant(torch.zeros(3, 4, 64, dtype=BF, device=d).transpose(0, 1))
    with pytest.raises(ValueError, match="alignment"):
        ops.mxfp4_quant(torch.zeros(2, 72, dtype=BF, device=d)[:, 4:36])
    with pytest.raises(ValueError, match="codes"):
        ops.mxfp4_quant(torch.zeros(2, 64, dtype=BF, device=d), codes=torch.zeros(2, 64, dtype=U8, device=d))
    with pytest.raises(ValueError, match="shape"):
        ops.mxfp4_quant(torch.zeros(2, 64, dtype=BF, device=d), out=torch.zeros(2, 32, dtype=BF, device=d))


# --------------------------------------------------------------- projection

def _w(N, K, seed):
    """(codes, scales) of an MXFP4 weight whose rows differ in size."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(N, K, generator=g) * K ** -0.5 * torch.exp2(torch.randint(-4, 4, (N, 1), generator=g).float())
    code, sc, _ = lowbit.mxfp4(w)
    return lowbit.pack_nibbles(code), sc.to(U8)


def _check_linear(y, x, codes, scales):
    """Products of E2M1 values and power-of-two scales are exact; a sum of K
    of them in fp32, in any order and with truncation, is off by at most
    K 2^-23 of the sum of magnitudes; bf16 rounds by 2^-8."""
    xv = lowbit.mxfp4(x)[2]
    wv = lowbit.mxfp4_values(codes, scales)
    exact, mag = xv @ wv.T, xv.abs() @ wv.abs().T
    tol = mag * x.shape[1] * 2.0 ** -23 + (exact.abs() * 2.0 ** -8 if y.dtype == BF else 0.0) + 1e-30
    err = (y.cpu().double() - exact).abs()
    assert bool((err <= tol).all()), f"max err/tol {float((err / tol).max()):.3f}"


SIZES = [(1, 1, 32), (1, 128, 256), (2, 7, 64), (1, 1024, 4096), (31, 200, 96), (32, 129, 288), (33, 64, 4096),
         (64, 2048, 1024), (64, 512, 4096), (100, 2001, 512), (128, 256, 8192), (192, 384, 256), (193, 130, 544),
         (333, 2001, 4128), (400, 64, 32), (1000, 300, 2080), (2, 24000, 1024), (700, 8200, 512), (5, 1, 8192),
         (3, 8, 64), (40, 16, 512), (200, 40, 320), (65, 72, 2048), (17, 136, 8192), (1, 32768, 1024)]


@pytest.mark.parametrize("B,N,K", SIZES)
@pytest.mark.parametrize("f32", [False, True])
def test_linear_matches_the_definition(cuda_dev, B, N, K, f32):
    from dsv4attn import ops
    g = torch.Generator().manual_seed(B + N + K)
    x = torch.randn(B, K, generator=g).to(BF)
    codes, scales = _w(N, K, B * 7 + N)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    y = ops.linear_mxfp4(x.to(cuda_dev), w, out_f32=f32, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0 and y.shape == (B, N) and y.dtype == (F32 if f32 else BF)
    _check_linear(y, x, codes, scales)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_input_types(cuda_dev, dtype):
    from dsv4attn import ops
    x = torch.randn(37, 1056, generator=torch.Generator().manual_seed(1)).to(dtype)
    codes, scales = _w(300, 1056, 2)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    _check_linear(ops.linear_mxfp4(x.to(cuda_dev), w), x, codes, scales)


@pytest.mark.parametrize("B", [3, 70, 250])
@pytest.mark.parametrize("f32", [False, True])
def test_linear_strided_rows_and_out(cuda_dev, B, f32):
    """x a column slice, y into a wider buffer with and without 16-byte rows;
    columns past N and the rows behind it untouched."""
    from dsv4attn import ops
    g = torch.Generator().manual_seed(4)
    big = torch.randn(B, 640, generator=g).to(BF)
    codes, scales = _w(320, 256, 3)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    xd = big.to(cuda_dev)[:, 64:320]
    want = ops.linear_mxfp4(xd, w, out_f32=f32)
    _check_linear(want, big[:, 64:320], codes, scales)
    for width in (400, 403):
        buf = torch.full((B + 1, width), 7.0, dtype=F32 if f32 else BF, device=cuda_dev)
        got = ops.linear_mxfp4(xd, w, out=buf[:B], out_f32=f32)
        torch.cuda.synchronize()
        assert got.data_ptr() == buf.data_ptr() and torch.equal(buf[:B, :320], want)
        assert bool((buf[:B, 320:] == 7.0).all()) and bool((buf[B] == 7.0).all())


def test_linear_rows_do_not_depend_on_the_batch_around_them(cuda_dev):
    """Rows split from a batch give the same values up to the sum's order."""
    from dsv4attn import ops
    x = torch.randn(290, 2048, generator=torch.Generator().manual_seed(9)).to(BF).to(cuda_dev)
    codes, scales = _w(640, 2048, 5)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    whole = ops.linear_mxfp4(x, w, out_f32=True)
    for n in (1, 40, 200):
        _check_linear(ops.linear_mxfp4(x[:n], w, out_f32=True), x[:n].cpu(), codes, scales)
    again = ops.linear_mxfp4(x, w, out_f32=True)
    torch.cuda.synchronize()
    assert torch.equal(whole, again)                       # a fixed order: the same bits every time


@pytest.mark.parametrize("B", [4, 200])
def test_linear_nan_blocks(cuda_dev, B):
    """A NaN or an infinity in x makes its token's row NaN and no other; a NaN
    scale in W its column."""
    from dsv4attn import ops
    x = torch.randn(B, 512, generator=torch.Generator().manual_seed(9)).to(BF)
    x[1, 300] = float("nan")
    x[3, 511] = float("inf")
    codes, scales = _w(200, 512, 6)
    scales[150, 3] = 255
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    y = ops.linear_mxfp4(x.to(cuda_dev), w).cpu()
    nan = torch.zeros(B, 200, dtype=torch.bool)
    nan[[1, 3]] = True
    nan[:, 150] = True
    assert torch.equal(y.isnan(), nan)


def test_linear_scale_range(cuda_dev):
    """Weight blocks of very different size in one row, and zero rows."""
    from dsv4attn import ops
    x = torch.randn(20, 256, generator=torch.Generator().manual_seed(2))
    x[:, 64:128] *= 2.0 ** 40
    x[5] = 0
    x = x.to(BF)
    codes, scales = _w(130, 256, 8)
    scales[:, 1] = 200
    scales[:, 5] = 60
    codes[7] = 0
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    y = ops.linear_mxfp4(x.to(cuda_dev), w, out_f32=True)
    _check_linear(y, x, codes, scales)
    assert bool((y[5] == 0).all()) and bool((y[:, 7] == 0).all())


def test_pack_from_floats_and_typed_views(cuda_dev):
    from dsv4attn import ops
    g = torch.Generator().manual_seed(3)
    w = (torch.randn(130, 288, generator=g) * 0.1).to(BF)
    code, sc, _ = lowbit.mxfp4(w)
    codes, scales = lowbit.pack_nibbles(code).to(cuda_dev), sc.to(U8).to(cuda_dev)
    a = ops.pack_linear_weight_mxfp4(codes, scales)
    b = ops.pack_linear_weight_mxfp4(w.to(cuda_dev))
    c = ops.pack_linear_weight_mxfp4(codes.view(torch.float4_e2m1fn_x2), scales.view(torch.float8_e8m0fnu))
    assert a.shape == (130, 288) and torch.equal(a.packed, b.packed) and torch.equal(a.packed, c.packed)


def test_linear_refusals(cuda_dev):
    from dsv4attn import ops
    d = cuda_dev
    codes, scales = _w(64, 128, 1)
    codes, scales = codes.to(d), scales.to(d)
    w = ops.pack_linear_weight_mxfp4(codes, scales)
    x = torch.zeros(4, 128, dtype=BF, device=d)
    with pytest.raises(ValueError, match="scales"):
        ops.pack_linear_weight_mxfp4(codes, scales[:, :3].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        ops.pack_linear_weight_mxfp4(codes[:, :32], scales[:, :2].contiguous())
    with pytest.raises(ValueError, match="without scales"):
        ops.pack_linear_weight_mxfp4(codes)
    with pytest.raises(ValueError, match="uint8"):
        ops.pack_linear_weight_mxfp4(codes, scales.float())
    with pytest.raises(TypeError, match="MXFP4Weight"):
        ops.linear_mxfp4(x, codes)
    with pytest.raises(ValueError, match="128"):
        ops.linear_mxfp4(x[:, :64], w)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.linear_mxfp4(x.double(), w)
    with pytest.raises(ValueError, match="alignment"):
        ops.linear_mxfp4(torch.zeros(4, 132, dtype=BF, device=d)[:, 4:], w)
    with pytest.raises(ValueError, match="out"):
        ops.linear_mxfp4(x, w, out=torch.zeros(3, 64, dtype=BF, device=d))
    with pytest.raises(ValueError, match="out must be"):
        ops.linear_mxfp4(x, w, out=torch.zeros(4, 64, dtype=F32, device=d))
    assert ops.linear_mxfp4(x[:0], w).shape == (0, 64)


def test_linear_captured_and_on_two_streams(cuda_dev):
    """Two captured graphs and eager calls on a third stream, at once: each
    keeps its own scratch."""
    from dsv4attn import ops
    g = torch.Generator().manual_seed(12)
    codes, scales = _w(1024, 2048, 4)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    xs = [torch.randn(b, 2048, generator=g).to(BF).to(cuda_dev) for b in (9, 120, 300)]
    want = [ops.linear_mxfp4(x, w) for x in xs]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    for x, s in zip(xs[:2], streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs.append(ops.linear_mxfp4(x, w))
        graphs.append(gr)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        with torch.cuda.stream(streams[2]):
            eager = [ops.linear_mxfp4(xs[2], w) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, wt) for o, wt in zip(outs, want))
        assert all(torch.equal(e, want[2]) for e in eager)


def test_workspace_of_another_device(cuda_dev):
    from dsv4attn import ops
    w = ops.pack_linear_weight_mxfp4(_x(256, 4096, BF, 1).to(cuda_dev))
    x = _x(512, 4096, BF, 2).to(cuda_dev)
    with pytest.raises(ValueError, match="workspace on cpu"):
        ops.linear_mxfp4(x, w, ws=ops.Workspace("cpu"))
    ws = ops.Workspace(cuda_dev)
    assert torch.equal(ops.linear_mxfp4(x, w, ws=ws), ops.linear_mxfp4(x, w))
    assert ws.nbytes > 16


@pytest.mark.parametrize("B,N,K", [(1024, 9600, 65536), (8, 128, 1 << 21)])
@pytest.mark.parametrize("f32", [False, True])
def test_waits_that_run_out_end_the_call_once(cuda_dev, B, N, K, f32):
    """A wait limit far below the sums' time, whole items and items split over a
    cluster: the first wait to run out ends the others of its CTA, nothing wrong
    is stored, the status says so, and the next call is right."""
    import time

    from dsv4attn import ops
    g = torch.Generator(device=cuda_dev).manual_seed(B)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=U8, device=cuda_dev)
    w = ops.pack_linear_weight_mxfp4(codes, torch.full((N, K // 32), 127, dtype=U8, device=cuda_dev))
    del codes
    x = torch.randn(B, K, generator=g, device=cuda_dev).to(BF)
    want = ops.linear_mxfp4(x, w, out_f32=f32)
    for width in (N, N + 1):                                # stored by tiles, and by elements
        out = torch.full((B, width), 12345.0, dtype=want.dtype, device=cuda_dev)
        blank = out[0, 0].clone()
        status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
        torch.cuda.synchronize()
        prev = ops.set_wait_limit(1)
        try:
            t0 = time.time()
            ops.linear_mxfp4(x, w, out=out, out_f32=f32, status=status)
            torch.cuda.synchronize()
            dt = time.time() - t0
        finally:
            ops.set_wait_limit(prev)
        assert dt < 0.5, f"{dt:.3f} s"
        with pytest.raises(TimeoutError):
            ops.raise_for_status(status, "linear_mxfp4")
        y = out[:, :N]
        fine = (y == want) | (y == blank) | (y.isnan() if N == 128 else torch.zeros_like(y, dtype=torch.bool))
        assert bool(fine.all()) and not torch.equal(y, want)
        status.zero_()
        again = ops.linear_mxfp4(x, w, out_f32=f32, status=status)
        torch.cuda.synchronize()
        assert torch.equal(again, want) and int(status) == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,N,K", [(1, 1024, 4096), (3, 200, 96), (5, 300, 512), (5, 512, 32768), (48, 130, 256)])
@pytest.mark.parametrize("f32", [False, True])
def test_linear_input_types_of_a_few_tokens(cuda_dev, dtype, B, N, K, f32):
    """The product quantises x itself, of each type, whole and split over K (with
    owners that have no row)."""
    from dsv4attn import ops
    x = torch.randn(B, K, generator=torch.Generator().manual_seed(B + K)).to(dtype)
    codes, scales = _w(N, K, N)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    _check_linear(ops.linear_mxfp4(x.to(cuda_dev), w, out_f32=f32), x, codes, scales)


@pytest.mark.parametrize("B,N,K", [(33, 128, 16384), (40, 130, 16384), (59, 290, 7072), (143, 22, 7424),
                                   (47, 200, 65536), (100, 130, 29984), (97, 24, 8192)])
@pytest.mark.parametrize("f32", [False, True])
def test_linear_split_over_several_token_tiles(cuda_dev, B, N, K, f32):
    """Splits over K of several token tiles, most of which do not divide the
    tile: owners with fewer rows or none, no row of the next tile touched."""
    from dsv4attn import ops
    x = torch.randn(B, K, generator=torch.Generator().manual_seed(B)).to(BF)
    codes, scales = _w(N, K, K)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    buf = torch.full((B + 1, N + 8), 7.0, dtype=F32 if f32 else BF, device=cuda_dev)
    y = ops.linear_mxfp4(x.to(cuda_dev), w, out=buf[:B], out_f32=f32)
    torch.cuda.synchronize()
    _check_linear(y[:, :N], x, codes, scales)
    assert bool((buf[B] == 7.0).all()) and bool((buf[:, N:] == 7.0).all())
    status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    assert torch.equal(ops.linear_mxfp4(x.to(cuda_dev), w, out_f32=f32, status=status), y[:, :N]) and int(status) == 0


def test_quant_of_more_blocks_than_the_grid_holds(cuda_dev):
    """Every CTA takes a second step (148 SMs x 64 CTAs x 128 blocks)."""
    from dsv4attn import ops
    M, K = 10300, 4096
    x = torch.randn(M, K, generator=torch.Generator(device=cuda_dev).manual_seed(5), device=cuda_dev).to(BF)
    assert M * K // 32 > 148 * 64 * 128
    out, scales, codes = ops.mxfp4_quant(x, out=True)
    pick = [0, 1, M // 2, 9471, 9472, 9473, M - 2, M - 1]  # 148 * 64 * 128 blocks = 9472 rows
    _check(x[pick].cpu(), (out[pick], scales[pick], codes[pick]))
    half = M // 2
    lo, hi = ops.mxfp4_quant(x[:half], out=True), ops.mxfp4_quant(x[half:], out=True)
    for whole, a, b in zip((out, scales, codes), lo, hi):
        assert torch.equal(whole[:half], a) and torch.equal(whole[half:], b)


@pytest.mark.parametrize("B,N,K", [(40001, 8, 32), (20003, 64, 1056)])
def test_linear_of_more_tokens_than_the_grid_holds(cuda_dev, B, N, K):
    """x's quantisation takes a second step a warp (148 SMs x 32 CTAs x 8)."""
    from dsv4attn import ops
    assert B * -(-K // 1024) > 148 * 32 * 8
    x = torch.randn(B, K, generator=torch.Generator().manual_seed(2)).to(BF)
    codes, scales = _w(N, K, 11)
    w = ops.pack_linear_weight_mxfp4(codes.to(cuda_dev), scales.to(cuda_dev))
    y = ops.linear_mxfp4(x.to(cuda_dev), w)
    pick = torch.cat([torch.arange(40), torch.arange(B // 2, B // 2 + 40), torch.arange(B - 3000, B)])
    _check_linear(y[pick.to(cuda_dev)], x[pick], codes, scales)


def test_quant_into_columns_beside_its_own(cuda_dev):
    """x and out as column blocks of one buffer, touching and apart, and as rows
    one behind the other."""
    from dsv4attn import ops
    M, K = 300, 96
    x = _x(M, K, BF, 9).to(cuda_dev)
    want = ops.mxfp4_quant(x, out=True)
    for a, b in ((0, K), (K, 0), (8, 2 * K + 16), (160, 0)):
        buf = torch.full((2 * M, 400), 7.0, dtype=BF, device=cuda_dev)
        buf[:M, a:a + K] = x
        got = ops.mxfp4_quant(buf[:M, a:a + K], out=buf[:M, b:b + K])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and torch.equal(buf[:M, a:a + K], x)
        got = ops.mxfp4_quant(buf[:M, a:a + K], out=buf[M:, a:a + K])
        assert torch.equal(got[0], want[0])
    with pytest.raises(ValueError, match="overlap"):
        ops.mxfp4_quant(buf[:M, 0:K], out=buf[1:M + 1, 0:K])
    one = torch.full((1, 400), 7.0, dtype=BF, device=cuda_dev)
    one[:, :K] = x[:1]
    assert torch.equal(ops.mxfp4_quant(one[:, :K], out=one[:, :K])[0], want[0][:1])

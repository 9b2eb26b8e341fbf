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

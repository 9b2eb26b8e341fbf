"""The low-bit operators as a decode step uses them, one after the other:
MXFP4 projections around the FP8 latent cache that the sparse attention reads.
Each stage is checked against its 64-bit form on the inputs it really had."""

import pytest
import torch

import lowbit
import oracle as O
from test_gpu_kv_quant import _bits
from test_gpu_mxfp4 import _check_linear

pytestmark = pytest.mark.gpu

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


class _Fp4Linear:
    """A checkpoint's Linear: int8 codes with a float8_e8m0fnu scale."""

    def __init__(self, n, k, seed):
        w = torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) * k ** -0.5
        code, sc, _ = lowbit.mxfp4(w)
        self.weight = lowbit.pack_nibbles(code).view(torch.int8)
        self.scale = sc.to(torch.uint8).view(torch.float8_e8m0fnu)

    @property
    def parts(self):
        return self.weight.view(torch.uint8), self.scale.view(torch.uint8)


def test_decode_steps_over_the_low_bit_layer(cuda_dev):
    """x -> wkv -> ring write, x -> q -> attention over ring and older rows ->
    wo, five steps that wrap the ring, replayed from one captured graph."""
    from dsv4attn import modules as M
    from dsv4attn import ops
    B, dim, win, older, K = 5, 512, 8, 40, 30
    g = torch.Generator().manual_seed(7)
    wkv, wq, wo = _Fp4Linear(512, dim, 1), _Fp4Linear(64 * 512, dim, 2), _Fp4Linear(dim, 64 * 512, 3)
    d_kv, d_q, d_o = (M.DeviceLinear(cuda_dev, w) for w in (wkv, wq, wo))
    sa = M.DeviceSparseAttn(cuda_dev, torch.randn(64, generator=g), 1.0)
    cache = ops.kv_quant_cache(B, win + older, device=cuda_dev)
    old = torch.randn(B, older, 512, generator=g).to(BF)
    ops.kv_quant_write(old.to(cuda_dev), cache, torch.zeros(B, dtype=I32, device=cuda_dev), older, offset=win)
    idx = torch.empty(B, win + K, dtype=I32, device=cuda_dev)
    idx[:, win:] = torch.randint(win, win + older, (B, K), generator=g, dtype=I32).to(cuda_dev)
    pos = torch.full((B,), 4, dtype=I32, device=cuda_dev)
    x = torch.empty(B, dim, dtype=BF, device=cuda_dev)
    cos, sin = (t.to(cuda_dev) for t in O.rope_tables(64, 64, compressed=True))

    def step():
        kv = d_kv(x, rope=(cos, sin, pos, 512, 64))
        ops.kv_quant_write(kv, cache, pos, win)
        ops.window_indices(pos, win, out=idx)
        q = d_q(x)
        o = sa.forward_device(q.view(B, 1, 64, 512) * 512 ** -0.5, cache, idx, None, 1, win + K)
        return kv, q, o, d_o(o.view(B, -1)), ops.kv_quant_read(cache, idx)

    x.copy_(torch.randn(B, dim, generator=g).to(BF))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv, q, o, y, rows = step()
    for p in range(5, 10):
        x.copy_(torch.randn(B, dim, generator=g).to(BF))
        pos.fill_(p)
        graph.replay()
        torch.cuda.synchronize()
        _check_linear(q, x.cpu(), *wq.parts)
        _check_linear(y, o.cpu().view(B, -1), *wo.parts)
        # kv: the projection, then the oracle's rotary of the kernel's own result
        plain = ops.linear_mxfp4(x, d_kv.weight)
        _check_linear(plain, x.cpu(), *wkv.parts)
        c, s = cos.cpu()[p].expand(B, -1), sin.cpu()[p].expand(B, -1)
        assert torch.equal(_bits(kv).cpu(), _bits(O.head_norm_rope(plain.cpu(), 1, 512, c, s, rope_dim=64, norm=False)))
        # the ring's newest row reads back as act_quant's round trip
        want = torch.cat([O.act_quant_block(kv.cpu()[:, :448].contiguous())[0], kv.cpu()[:, 448:]], 1)
        whole = ops.kv_quant_read(cache)
        assert torch.equal(_bits(whole[:, p % win]).cpu(), _bits(want))
        # window places past the position are masked and read as zero rows
        assert int((idx[0] >= 0).sum()) == K + min(p + 1, win)
        sel = torch.stack([whole[b][idx[b].long().clamp(min=0)] for b in range(B)])
        assert torch.equal(rows, sel.masked_fill((idx < 0).unsqueeze(-1), 0))
        # attention of the scaled q over those rows
        qs = q.view(B, 1, 64, 512) * 512 ** -0.5
        want_o, A, dmax, _ = lowbit.attention(qs, whole, idx.view(B, 1, -1), sa.sink, 1.0)
        slack = (dmax * 512 * 2.0 ** -23 + 2.0 ** -20).unsqueeze(-1)
        tol = A * (2 * 2.0 ** -8 + 2 * slack) + want_o.abs() * 2.0 ** -8 + 1e-30
        assert bool(((o.cpu().double() - want_o).abs() <= tol).all())
        assert int(sa.status) == 0


def test_prefill_chunk_then_decode_reads_the_same_cache(cuda_dev):
    """A padded chunk written behind the ring in one call gives the records
    that writing its tokens one by one gives."""
    from dsv4attn import ops
    B, S, win, rows = 3, 21, 16, 16 + 64
    kv = torch.randn(B, S, 512, generator=torch.Generator().manual_seed(3)).to(BF).to(cuda_dev)
    n = torch.tensor([21, 0, 13], dtype=I32, device=cuda_dev)
    pos = torch.tensor([40, 5, 60], dtype=I32, device=cuda_dev)
    once, each = ops.kv_quant_cache(B, rows, device=cuda_dev), ops.kv_quant_cache(B, rows, device=cuda_dev)
    ops.kv_quant_write(kv, once, pos, rows - win, offset=win, n_valid=n)
    for s in range(S):
        ops.kv_quant_write(kv[:, s], each, pos + s, rows - win, offset=win, n_valid=(n > s).int())
    torch.cuda.synchronize()
    assert torch.equal(once, each) and bool((once[1] == 0).all())


def test_device_linear_with_mxfp4_weights(cuda_dev):
    from dsv4attn import modules as M
    from dsv4attn import ops
    a, b = _Fp4Linear(96, 256, 4), _Fp4Linear(160, 256, 5)
    x = torch.randn(2, 3, 256, generator=torch.Generator().manual_seed(1)).to(BF)
    y = M.DeviceLinear(cuda_dev, a, out_dtype=F32)(x.to(cuda_dev))
    assert y.shape == (2, 3, 96) and y.dtype == F32
    _check_linear(y.view(6, 96), x.view(6, 256), *a.parts)
    lin = M.DeviceLinear.fused(cuda_dev, [a, b])
    assert (lin._fused_kv_out, lin._fused_gate_out, lin.out_dim) == (96, 160, 256)
    both = lin(x.to(cuda_dev))
    assert torch.equal(both[..., :96], M.DeviceLinear(cuda_dev, a)(x.to(cuda_dev)))
    with pytest.raises(ValueError, match="scale"):
        M.DeviceLinear(cuda_dev, a, scale=0.5)
    with pytest.raises(ValueError, match="rotary"):
        lin(x.to(cuda_dev), rope=(None, None, None, 96, 64))
    with pytest.raises(ValueError, match="dtype"):
        M.DeviceLinear(cuda_dev, torch.zeros(32, 32, dtype=torch.int8))   # no scale: not MXFP4
    assert isinstance(lin.weight, ops.MXFP4Weight)


def test_device_linear_mxfp4_has_a_status_word(cuda_dev, monkeypatch):
    """A call that brings no status word still reports into one."""
    from dsv4attn import modules as M
    from dsv4attn import ops
    seen = []
    real = ops.linear_mxfp4
    monkeypatch.setattr(ops, "linear_mxfp4", lambda *a, **k: (seen.append(k["status"]), real(*a, **k))[1])
    a, b = _Fp4Linear(96, 256, 4), _Fp4Linear(160, 256, 5)
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1)).to(BF).to(cuda_dev)
    own = torch.zeros(1, dtype=I32, device=cuda_dev)
    for lin in (M.DeviceLinear(cuda_dev, a), M.DeviceLinear.fused(cuda_dev, [a, b])):
        lin(x)
        lin(x, status=own)
        assert seen[-2] is lin.status and seen[-1] is own
        ops.raise_for_status(lin.status, "linear_mxfp4")

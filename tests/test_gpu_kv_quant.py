"""The FP8 latent cache on the GPU: rows quantised as they are written (against
the oracle's act_quant, bit for bit, and the definition in 64 bits), read
back, and attended where they lie (against sparse_attn over the rows read back,
bit for bit, and sink attention in 64 bits)."""

import pytest
import torch

import lowbit
import oracle as O

pytestmark = pytest.mark.gpu

BF, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
SCALE = 512 ** -0.5


def _kv(B, S, D, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, D, generator=g) * torch.exp(torch.randn(B, S, 1, generator=g))
    if S > 1:
        x[0, 1, :64] = 0.0                     # a block of zeros: the smallest scale
    return x.to(BF)


def _want_rows(kv, rope):
    """(codes, scales, row values) of kv [B, S, D] by the oracle's act_quant."""
    nope = kv.shape[-1] - rope
    val, s, codes = O.act_quant_block(kv[..., :nope].reshape(-1, nope).contiguous())
    return codes, s, torch.cat([val.reshape(*kv.shape[:-1], nope), kv[..., nope:]], -1)


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32 if t.element_size() == 4 else U8)


def _expected_cache(before, kv, pos, win, offset, rope, n_valid):
    """The cache bytes after a write, token by token."""
    after = before.clone()
    B, S, D = kv.shape
    nope = D - rope
    codes, s, _ = _want_rows(kv, rope)
    codes, s = codes.view(B, S, nope), s.view(B, S, nope // 64)
    for b in range(B):
        n = S if n_valid is None else min(int(n_valid[b]), S)
        for t in range(max(0, n - win), n):
            p = int(pos[b]) + t
            if p < 0:
                continue
            rec = after[b, offset + p % win]
            rec.zero_()
            rec[:nope] = codes[b, t].contiguous().view(U8)
            rec[nope:nope + 2 * rope] = kv[b, t, nope:].contiguous().view(U8)
            rec[nope + 2 * rope:nope + 2 * rope + nope // 16] = s[b, t].contiguous().view(U8)
    return after


@pytest.mark.parametrize("B,S,D,rope,win,offset,extra,pos0,ragged", [
    (1, 1, 512, 64, 128, 0, 0, 0, False),
    (3, 1, 512, 64, 128, 0, 7, 32767, False),
    (2, 5, 512, 64, 8, 3, 2, 6, False),          # wraps inside the call
    (2, 40, 512, 64, 16, 0, 1, 9, False),        # more tokens than rows
    (4, 33, 512, 64, 64, 128, 0, 60, True),      # padded batch
    (3, 6, 512, 64, 8, 0, 0, -4, False),         # tokens before position 0
    (2, 3, 512, 64, 1, 0, 1, 5, False),          # a ring of one row
    (2, 9, 128, 0, 12, 0, 0, 2, False),
    (2, 9, 96, 32, 12, 1, 0, 2, True),
    (1, 4, 576, 64, 50, 0, 0, 2 ** 31 - 3, False),   # positions past 2^31 inside the call
    (1, 3, 2112, 64, 4, 0, 0, 1, False),
    (0, 3, 512, 64, 4, 0, 0, 0, False),
])
def test_write_is_the_oracles_act_quant(cuda_dev, B, S, D, rope, win, offset, extra, pos0, ragged):
    from dsv4attn import ops
    kv = _kv(max(B, 1), S, D, seed=B * 100 + S)[:B]
    g = torch.Generator().manual_seed(1)
    before = torch.randint(0, 256, (B, offset + win + extra, ops.kv_quant_row_bytes(D, rope)), generator=g, dtype=U8)
    pos = torch.arange(B, dtype=I32) + pos0 if pos0 < 2 ** 30 else torch.full((B,), pos0, dtype=I32)
    n_valid = torch.tensor([0, S, S // 2, S + 5][:B], dtype=I32) if ragged else None
    cache = before.to(cuda_dev)
    ops.kv_quant_write(kv.to(cuda_dev), cache, pos.to(cuda_dev), win, offset=offset, rope_dim=rope,
                       n_valid=n_valid.to(cuda_dev) if ragged else None)
    torch.cuda.synchronize()
    want = _expected_cache(before, kv, pos, win, offset, rope, n_valid)
    assert torch.equal(cache.cpu(), want)


@pytest.mark.parametrize("amax", [448.0, 447.0, 1.0, 3.0, 1e-4, 5e-5, 0.7109375, 3.3e38, 1.1e-38, 2.0 ** -100, 96.5])
def test_write_of_every_bf16_value(cuda_dev, amax):
    """Every bf16 number up to amax, in blocks of that maximum: the quotient
    is the correctly rounded one, so the codes are the oracle's."""
    from dsv4attn import ops
    x = torch.arange(0x7f80, dtype=torch.int32).to(torch.int16).view(BF)
    top = torch.tensor([amax]).to(BF)
    x = torch.cat([x[x < top], -x[x < top]])
    x = torch.cat([x, torch.zeros(-x.numel() % 63, dtype=BF)]).view(-1, 63)
    x = torch.cat([x, top.expand(x.shape[0], 1)], 1)
    x = torch.cat([x, torch.zeros(-x.shape[0] % 8, 64, dtype=BF)])
    kv = x.view(1, -1, 512)
    n = kv.shape[1]
    cache = ops.kv_quant_cache(1, n, 512, 0, device=cuda_dev)
    ops.kv_quant_write(kv.to(cuda_dev), cache, torch.zeros(1, dtype=I32, device=cuda_dev), n, rope_dim=0)
    codes, s, _ = _want_rows(kv, 0)
    got, _, gs = ops.kv_quant_views(cache, 512, 0)
    assert torch.equal(gs.cpu().view(-1), s.view(-1))
    assert torch.equal(got.cpu().view(U8).view(-1), codes.view(U8).view(-1))


def test_write_error_is_half_a_step(cuda_dev):
    """|value - x| <= |x| 2^-4 (half an e4m3 step) or half of the smallest
    step, s 2^-10, then bf16's 2^-8; s and the quotient are fp32: 3 roundings
    of 2^-24 each, which can only move a value over a tie (both neighbours
    are then half a step away)."""
    from dsv4attn import ops
    kv = _kv(4, 50, 512, seed=3)
    cache = ops.kv_quant_cache(4, 50, device=cuda_dev)
    ops.kv_quant_write(kv.to(cuda_dev), cache, torch.zeros(4, dtype=I32, device=cuda_dev), 50)
    got = ops.kv_quant_read(cache, dtype=F32).cpu().double()
    x = kv.double()
    s = ops.kv_quant_views(cache)[2].cpu().double().repeat_interleave(64, -1)
    n = x[..., :448]
    tol = torch.maximum(n.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20)
    assert bool(((got[..., :448] - n).abs() <= tol).all())
    assert torch.equal(got[..., 448:], x[..., 448:])
    amax = n.unflatten(-1, (7, 64)).abs().amax(-1).clamp(min=1e-4)
    assert bool(((s[..., ::64] * 448 / amax - 1).abs() <= 3 * 2.0 ** -24).all())


def test_write_matches_kv_window_write(cuda_dev):
    """The records read back as the bf16 rows kv_window_write stores."""
    from dsv4attn import ops
    B, win = 37, 128
    kv = _kv(B, 1, 512, seed=8)[:, 0].to(cuda_dev)
    pos = torch.randint(0, 4000, (B,), generator=torch.Generator().manual_seed(2), dtype=I32).to(cuda_dev)
    plain = torch.zeros(B, win, 512, dtype=BF, device=cuda_dev)
    cache = ops.kv_quant_cache(B, win, device=cuda_dev)
    ops.kv_window_write(kv, plain, pos, win)
    ops.kv_quant_write(kv, cache, pos, win)
    torch.cuda.synchronize()
    assert torch.equal(_bits(ops.kv_quant_read(cache)).cpu(), _bits(plain).cpu())


def test_non_finite_blocks_read_nan(cuda_dev):
    from dsv4attn import ops
    kv = _kv(1, 3, 512, seed=4)
    kv[0, 0, 5] = float("nan")
    kv[0, 1, 447] = float("-inf")
    kv[0, 2, 500] = float("inf")               # a rotary dim: kept as it is
    cache = ops.kv_quant_cache(1, 3, device=cuda_dev)
    ops.kv_quant_write(kv.to(cuda_dev), cache, torch.zeros(1, dtype=I32, device=cuda_dev), 3)
    got = ops.kv_quant_read(cache).cpu()
    nan = torch.zeros(3, 512, dtype=torch.bool)
    nan[0, :64] = True
    nan[1, 384:448] = True
    assert torch.equal(got[0].isnan(), nan)
    assert got[0, 2, 500] == float("inf")
    _, _, want = _want_rows(torch.where(torch.isfinite(kv), kv, torch.zeros_like(kv)), 64)
    want[0, 2, 500] = float("inf")
    assert torch.equal(got[0][~nan], want[0][~nan])


def test_more_sequences_than_a_grid_dimension(cuda_dev):
    from dsv4attn import ops
    B = 66_000
    kv = _kv(B, 1, 128, seed=2).to(cuda_dev)
    cache = ops.kv_quant_cache(B, 2, 128, 0, device=cuda_dev)
    pos = (torch.arange(B, dtype=I32) % 5).to(cuda_dev)
    ops.kv_quant_write(kv, cache, pos, 2, rope_dim=0)
    got = ops.kv_quant_read(cache, (pos % 2).view(B, 1), D=128, rope_dim=0)
    other = ops.kv_quant_read(cache, (1 - pos % 2).view(B, 1), D=128, rope_dim=0)
    assert torch.equal(_bits(got).cpu(), _bits(_want_rows(kv.cpu(), 0)[2])) and bool((other == 0).all())


def test_write_strided_kv_and_a_wider_cache(cuda_dev):
    """kv as a column slice of a wider projection output, batch and token
    strides swapped; a cache of more sequences than the call writes."""
    from dsv4attn import ops
    big = _kv(6, 3, 768, seed=9).to(cuda_dev)                  # [S=6, B=3, wide]
    kv = big.transpose(0, 1)[:, :, 128:640]
    cache = torch.full((5, 20, 608), 7, dtype=U8, device=cuda_dev)
    pos = torch.tensor([0, 3, 18], dtype=I32, device=cuda_dev)
    ops.kv_quant_write(kv, cache, pos, 20)
    torch.cuda.synchronize()
    want = _expected_cache(torch.full((5, 20, 608), 7, dtype=U8)[:3], kv.cpu().contiguous(), pos.cpu(), 20, 0, 64, None)
    assert torch.equal(cache[:3].cpu(), want) and bool((cache[3:] == 7).all())


@pytest.mark.parametrize("D,rope", [(512, 64), (128, 0), (96, 32), (576, 64)])
def test_read_by_index_and_whole(cuda_dev, D, rope):
    from dsv4attn import ops
    B, rows = 3, 41
    kv = _kv(B, rows, D, seed=D)
    cache = ops.kv_quant_cache(B, rows, D, rope, device=cuda_dev)
    ops.kv_quant_write(kv.to(cuda_dev), cache, torch.zeros(B, dtype=I32, device=cuda_dev), rows, rope_dim=rope)
    _, _, want = _want_rows(kv, rope)
    got = ops.kv_quant_read(cache, D=D, rope_dim=rope)
    assert got.dtype == BF and torch.equal(_bits(got).cpu(), _bits(want))
    # a column slice of a wider index buffer, the same row twice, masked places
    wide = torch.randint(-1, rows, (B, 90), generator=torch.Generator().manual_seed(3), dtype=I32)
    wide[:, 7] = wide[:, 6]
    wide[1, :] = -1
    idx = wide.to(cuda_dev)[:, 5:82]
    status = torch.zeros(1, dtype=I32, device=cuda_dev)
    sel = ops.kv_quant_read(cache, idx, D=D, rope_dim=rope, status=status).cpu()
    i = idx.cpu().long()
    ref = torch.stack([want[b][i[b].clamp(min=0)] for b in range(B)])
    ref[i < 0] = 0
    assert torch.equal(_bits(sel), _bits(ref)) and int(status) == 0
    # fp32: the products themselves
    f = ops.kv_quant_read(cache, idx, D=D, rope_dim=rope, dtype=F32).cpu()
    codes, _, scales = ops.kv_quant_views(cache, D, rope)
    prod = codes.cpu().float() * scales.cpu().repeat_interleave(64, -1)
    ref = torch.cat([prod, want[..., D - rope:].float()], -1)
    ref = torch.stack([ref[b][i[b].clamp(min=0)] for b in range(B)])
    ref[i < 0] = 0
    assert torch.equal(f, ref)


def test_read_clamps_and_reports_bad_rows(cuda_dev):
    from dsv4attn import ops
    cache = ops.kv_quant_cache(1, 4, device=cuda_dev)
    kv = _kv(1, 4, 512, seed=1)
    ops.kv_quant_write(kv.to(cuda_dev), cache, torch.zeros(1, dtype=I32, device=cuda_dev), 4)
    status = torch.zeros(1, dtype=I32, device=cuda_dev)
    idx = torch.tensor([[0, 4, 2 ** 31 - 1, -2 ** 31]], dtype=I32, device=cuda_dev)
    got = ops.kv_quant_read(cache, idx, status=status).cpu()
    _, _, want = _want_rows(kv, 64)
    assert torch.equal(got[0, 1], want[0, 3]) and torch.equal(got[0, 2], want[0, 3]) and bool((got[0, 3] == 0).all())
    assert int(status) & ops.STATUS_BAD_INDEX


# ---------------------------------------------------------------- attention

def _attn_case(B, S, rows, K, seed, dev, masked=0.1):
    from dsv4attn import ops
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, S, 64, 512, generator=g).to(BF).to(dev)
    cache = ops.kv_quant_cache(B, rows, device=dev)
    ops.kv_quant_write(_kv(B, rows, 512, seed + 1).to(dev), cache, torch.zeros(B, dtype=I32, device=dev), rows)
    idx = torch.randint(0, rows, (B, S, K), generator=g, dtype=I32)
    idx[torch.rand(B, S, K, generator=g) < masked] = -1
    sink = torch.randn(64, generator=g).to(dev)
    return q, cache, idx, sink


def _check_attention(out, lse, q, rows, idx, sink):
    """Roundings on the way to an output o = sum_k p_k v_k, with A = sum_k p_k
    |v_k|: P in bf16 (2^-8 A), a split's O in bf16 where splits are joined
    (2^-8 A), o in bf16 (2^-8 |o|); a score is a sum of 512 products in fp32,
    off by at most d 512 2^-23 for d = sum |q k| scale (any summation order,
    truncation included), plus 2^-20 for the exponential and the rescaled
    sums, on p and on the denominator."""
    o, A, d, want_lse = lowbit.attention(q, rows, idx, sink, SCALE)
    slack = (d * 512 * 2.0 ** -23 + 2.0 ** -20).unsqueeze(-1)
    tol = A * (2 * 2.0 ** -8 + 2 * slack) + o.abs() * 2.0 ** -8 + 1e-30
    err = (out.cpu().double() - o).abs()
    assert bool((err <= tol).all()), f"max err/tol {float((err / tol).max()):.3f}"
    assert bool(((lse.cpu().double().view_as(want_lse) - want_lse).abs() <= slack.squeeze(-1) + want_lse.abs() * 2.0 ** -22 + 1e-6).all())


@pytest.mark.parametrize("B,S,rows,K", [(1, 1, 5, 1), (2, 1, 9, 3), (1, 1, 200, 63), (1, 1, 200, 64), (1, 1, 200, 65),
                                        (3, 1, 300, 129), (1, 1, 3000, 2176), (5, 1, 900, 701), (64, 1, 700, 320),
                                        (70, 1, 300, 200), (149, 1, 70, 70), (2, 7, 400, 450), (1, 1, 4000, 2304),
                                        (1, 150, 300, 2400), (40, 1, 2500, 2304)])
def test_attention_over_the_records(cuda_dev, B, S, rows, K):
    from dsv4attn import ops
    q, cache, idx, sink = _attn_case(B, S, rows, K, seed=B * 1000 + S * 10 + K, dev=cuda_dev)
    status = torch.zeros(1, dtype=I32, device=cuda_dev)
    lse = torch.empty(B * S, 64, device=cuda_dev)
    out = ops.sparse_attn_quant(q, cache, idx.to(cuda_dev), sink, SCALE, lse=lse, status=status)
    rows_bf = ops.kv_quant_read(cache)
    lse2 = torch.empty_like(lse)
    same = ops.sparse_attn(q, rows_bf, idx.to(cuda_dev), sink, SCALE, lse=lse2)
    torch.cuda.synchronize()
    assert int(status) == 0
    # same tiles, same order, same splits: the same bits as over the bf16 rows
    assert torch.equal(_bits(out), _bits(same)) and torch.equal(lse, lse2)
    pick = list(range(min(B, 3))) + ([B - 1] if B > 3 else [])
    sp = [0, S - 1] if S > 1 else [0]
    sub = lambda t: t.view(B, S, *t.shape[2:])[pick][:, sp]  # noqa: E731
    _check_attention(sub(out), lse.view(B, S, 64)[pick][:, sp], sub(q), rows_bf[pick], idx[pick][:, sp], sink)


def test_attention_rows_without_keys(cuda_dev):
    """A row whose mask leaves nothing, K = 0, and tiles masked throughout
    before, between and after live ones: zero output, lse = sink."""
    from dsv4attn import ops
    q, cache, idx, sink = _attn_case(4, 1, 300, 640, seed=5, dev=cuda_dev, masked=0.0)
    idx[0] = -1
    idx[1, :, :300] = -1
    idx[2, :, 64:512] = -1
    idx[3, :, 1:] = -7                         # any negative number masks
    lse = torch.empty(4, 64, device=cuda_dev)
    out = ops.sparse_attn_quant(q, cache, idx.to(cuda_dev), sink, SCALE, lse=lse)
    assert bool((out[0] == 0).all()) and torch.allclose(lse[0], sink, rtol=0, atol=1e-6)
    _check_attention(out, lse, q, ops.kv_quant_read(cache), idx, sink)
    none = ops.sparse_attn_quant(q, cache, idx[..., :0].to(cuda_dev), sink, SCALE, lse=lse)
    torch.cuda.synchronize()
    assert bool((none == 0).all()) and torch.allclose(lse, sink.expand(4, 64), rtol=0, atol=1e-6)


def test_attention_extreme_scores_and_nan_rows(cuda_dev):
    """Scores far over the running maximum in a late tile, a sink that takes
    everything, and a NaN row that only one sequence selects."""
    from dsv4attn import ops
    q, cache, idx, sink = _attn_case(3, 1, 260, 256, seed=6, dev=cuda_dev, masked=0.0)
    idx[:] = torch.arange(256, dtype=I32)
    kv = _kv(3, 260, 512, 7).to(cuda_dev)
    kv[:, 200] *= 30                           # the largest scores in the last tile
    kv[2, 259, 3] = float("nan")
    ops.kv_quant_write(kv, cache, torch.zeros(3, dtype=I32, device=cuda_dev), 260)
    sink[0] = 500.0
    lse = torch.empty(3, 64, device=cuda_dev)
    out = ops.sparse_attn_quant(q, cache, idx.to(cuda_dev), sink, SCALE, lse=lse)
    _check_attention(out, lse, q, torch.nan_to_num(ops.kv_quant_read(cache)), idx, sink)
    idx[2, 0, 0] = 259
    out = ops.sparse_attn_quant(q, cache, idx.to(cuda_dev), sink, SCALE, lse=lse)
    torch.cuda.synchronize()
    assert bool(out[2].isnan().any()) and not bool(out[:2].isnan().any())


def test_attention_bad_index_is_clamped(cuda_dev):
    from dsv4attn import ops
    q, cache, idx, sink = _attn_case(1, 1, 30, 8, seed=3, dev=cuda_dev, masked=0.0)
    status = torch.zeros(1, dtype=I32, device=cuda_dev)
    bad = idx.clone()
    bad[0, 0, 3], idx[0, 0, 3] = 30, 29
    got = ops.sparse_attn_quant(q, cache, bad.to(cuda_dev), sink, SCALE, status=status)
    want = ops.sparse_attn_quant(q, cache, idx.to(cuda_dev), sink, SCALE)
    torch.cuda.synchronize()
    assert int(status) & ops.STATUS_BAD_INDEX and torch.equal(got, want)


def test_rows_past_2_to_31_bytes(cuda_dev):
    """One sequence whose cache is larger than 2^31 bytes, written, read and
    attended at its far end."""
    from dsv4attn import ops
    rows = 3_700_000                            # 2.25e9 bytes
    cache = ops.kv_quant_cache(1, rows, device=cuda_dev)
    kv = _kv(1, 70, 512, seed=12)
    far = rows - 70
    pos = torch.tensor([far], dtype=I32, device=cuda_dev)
    ops.kv_quant_write(kv.to(cuda_dev), cache, pos, rows)
    _, _, want = _want_rows(kv, 64)
    idx = torch.arange(far, rows, dtype=I32, device=cuda_dev).view(1, 70)
    assert torch.equal(_bits(ops.kv_quant_read(cache, idx)).cpu(), _bits(want))
    q = torch.randn(1, 64, 512, generator=torch.Generator().manual_seed(0)).to(BF).to(cuda_dev)
    sink = torch.zeros(64, device=cuda_dev)
    out = ops.sparse_attn_quant(q, cache, idx, sink, SCALE)
    same = ops.sparse_attn(q, want.to(cuda_dev), torch.arange(70, dtype=I32, device=cuda_dev).view(1, 70), sink, SCALE)
    torch.cuda.synchronize()
    assert torch.equal(out, same)


def test_refusals_on_the_device(cuda_dev):
    from dsv4attn import ops
    d = cuda_dev
    cache = ops.kv_quant_cache(2, 8, device=d)
    pos = torch.zeros(2, dtype=I32, device=d)
    kv = torch.zeros(2, 1, 512, dtype=BF, device=d)
    with pytest.raises(ValueError, match="ring"):
        ops.kv_quant_write(kv, cache, pos, 9)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.kv_quant_write(kv.float(), cache, pos, 8)
    with pytest.raises(ValueError, match="pos"):
        ops.kv_quant_write(kv, cache, pos[:1], 8)
    with pytest.raises(ValueError, match="int32"):
        ops.kv_quant_write(kv, cache, pos.long(), 8)
    with pytest.raises(ValueError, match="cache"):
        ops.kv_quant_write(torch.zeros(3, 1, 512, dtype=BF, device=d), cache, torch.zeros(3, dtype=I32, device=d), 8)
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.kv_quant_write(kv, torch.zeros(2, 8, 640, dtype=U8, device=d)[..., :608], pos, 8)
    with pytest.raises(ValueError, match="kv needs"):
        ops.kv_quant_write(torch.zeros(2, 1, 516, dtype=BF, device=d)[..., 4:], cache, pos, 8)
    with pytest.raises(ValueError, match="dtype"):
        ops.kv_quant_read(cache, dtype=torch.float16)
    with pytest.raises(ValueError, match="idx"):
        ops.kv_quant_read(cache, torch.zeros(3, 4, dtype=I32, device=d))
    with pytest.raises(ValueError, match="out"):
        ops.kv_quant_read(cache, out=torch.zeros(2, 7, 512, dtype=BF, device=d))
    q = torch.zeros(2, 64, 512, dtype=BF, device=d)
    idx = torch.zeros(2, 4, dtype=I32, device=d)
    sink = torch.zeros(64, device=d)
    with pytest.raises(ValueError, match="64 heads"):
        ops.sparse_attn_quant(q[:, :32].contiguous(), cache, idx, sink[:32].clone(), SCALE)
    with pytest.raises(ValueError, match="idx"):
        ops.sparse_attn_quant(q, cache, idx[:1], sink, SCALE)
    with pytest.raises(ValueError, match="cache"):
        ops.sparse_attn_quant(q, cache[:1], idx, sink, SCALE)
    with pytest.raises(ValueError, match="out"):
        ops.sparse_attn_quant(q, cache, idx, sink, SCALE, out=torch.empty(1, 64, 512, dtype=BF, device=d))


def test_captured_steps_and_a_second_stream(cuda_dev):
    """A decode step (write, attend, read) captured once and replayed with new
    inputs and positions in place, while an eager call of other sizes runs on
    a second stream."""
    from dsv4attn import ops
    B, W, K = 6, 16, 700
    rows = W + 800
    q, cache, idx, sink = _attn_case(B, 1, rows, K, seed=21, dev=cuda_dev)
    q2, cache2, idx2, sink2 = _attn_case(3, 1, 500, 1500, seed=22, dev=cuda_dev)
    idx, idx2 = idx.to(cuda_dev), idx2.to(cuda_dev)
    idx[..., :W] = torch.arange(W, dtype=I32, device=cuda_dev)
    kv = _kv(B, 1, 512, 30).to(cuda_dev)
    pos = torch.full((B,), 13, dtype=I32, device=cuda_dev)
    ref = cache.clone()
    want2 = ops.sparse_attn_quant(q2, cache2, idx2, sink2, SCALE)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        ops.sparse_attn_quant(q, cache, idx, sink, SCALE)     # set-up outside the capture
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            ops.kv_quant_write(kv, cache, pos, W)
            out = ops.sparse_attn_quant(q, cache, idx, sink, SCALE)
            back = ops.kv_quant_read(cache, idx[:, 0])
    other = torch.cuda.Stream()
    for step in range(4):
        kv.copy_(_kv(B, 1, 512, 40 + step))
        pos.add_(1)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            eager = [ops.sparse_attn_quant(q2, cache2, idx2, sink2, SCALE) for _ in range(3)]
        graph.replay()
        torch.cuda.synchronize()
        ops.kv_quant_write(kv, ref, pos, W)
        assert torch.equal(cache, ref)
        rows_bf = ops.kv_quant_read(ref)
        assert torch.equal(out, ops.sparse_attn(q, rows_bf, idx, sink, SCALE))
        assert torch.equal(_bits(back), _bits(ops.kv_quant_read(ref, idx[:, 0].contiguous())))
        assert all(torch.equal(e, want2) for e in eager)


def test_refusals_of_sizes_and_types_that_do_not_fit(cuda_dev):
    from dsv4attn import ops
    d = cuda_dev
    cache = ops.kv_quant_cache(2, 8, device=d)
    kv = torch.zeros(2, 512, dtype=BF, device=d)
    pos = torch.zeros(2, dtype=I32, device=d)
    for win in (2**32 + 8, -2**32 + 8):                    # 8 in 32 bits
        with pytest.raises(ValueError, match="too large"):
            ops.kv_quant_write(kv, cache, pos, win)
    with pytest.raises(ValueError, match="status must be torch.int32"):
        ops.kv_quant_read(cache, status=torch.zeros(1, dtype=torch.int64, device=d))
    with pytest.raises(ValueError, match="tensors on cuda:0 and cpu"):
        ops.kv_quant_read(cache, status=torch.zeros(1, dtype=I32))
    with pytest.raises(TypeError, match="out"):
        ops.mxfp4_quant(kv, out=False)
    assert not cache.any()


def test_strides_that_nothing_steps_by(cuda_dev):
    """One token, one sequence: the strides of those dims are not looked at."""
    from dsv4attn import ops
    d = cuda_dev
    flat = _kv(1, 2, 512, seed=31).to(d).view(-1)
    cache = torch.zeros(2, 4, 608, dtype=U8, device=d)
    pos = torch.zeros(2, dtype=I32, device=d)
    ops.kv_quant_write(flat.as_strided((2, 1, 512), (512, 3, 1)), cache, pos, 4)
    want = torch.zeros_like(cache)
    ops.kv_quant_write(flat.view(2, 512), want, pos, 4)
    torch.cuda.synchronize()
    assert torch.equal(cache, want) and bool(want.any())
    one = want[1].clone().view(-1).as_strided((1, 4, 608), (5, 608, 1))
    ops.kv_quant_write(flat.as_strided((1, 1, 512), (5, 3, 1)), one, pos[:1], 4, offset=0)
    idx = torch.tensor([[0, 1, -1]], dtype=I32, device=d)
    q = torch.randn(1, 64, 512, generator=torch.Generator().manual_seed(1)).to(BF).to(d)
    sink = torch.zeros(64, device=d)
    torch.cuda.synchronize()
    assert torch.equal(one[0], want[0])
    assert torch.equal(ops.kv_quant_read(one, idx), ops.kv_quant_read(want[:1], idx))
    assert torch.equal(ops.sparse_attn_quant(q, one, idx, sink, SCALE),
                       ops.sparse_attn_quant(q, want[:1], idx, sink, SCALE))


def test_write_over_every_pair_of_significands(cuda_dev):
    """Every bf16 significand over the scale of every maximum's, from the
    maximum down to a code of zero, both signs."""
    from dsv4attn import ops
    sig = 1 + torch.arange(128, dtype=torch.float64) / 128
    x = (sig.view(1, -1) * torch.exp2(-torch.arange(21).double()).view(-1, 1)).flatten()     # 2^0 .. 2^-20 of it
    x = torch.cat([x, -x, torch.zeros(-2 * x.numel() % 63, dtype=torch.float64)]).view(1, -1, 63)
    top = (2 * sig).view(-1, 1, 1).expand(-1, x.shape[1], 1)
    rows = torch.cat([x.expand(128, -1, -1), top], -1).reshape(-1, 64)
    rows = torch.cat([rows, torch.zeros(-rows.shape[0] % 8, 64, dtype=torch.float64)])
    for scale in (1.0, 2.0 ** -10, 2.0 ** 90):
        kv = (rows * scale).to(BF).view(1, -1, 512)
        assert torch.equal(kv.double().view(-1, 64), rows * scale)
        n = kv.shape[1]
        cache = ops.kv_quant_cache(1, n, 512, 0, device=cuda_dev)
        ops.kv_quant_write(kv.to(cuda_dev), cache, torch.zeros(1, dtype=I32, device=cuda_dev), n, rope_dim=0)
        codes, s, _ = _want_rows(kv, 0)
        got, _, gs = ops.kv_quant_views(cache, 512, 0)
        assert torch.equal(gs.cpu().view(-1), s.view(-1))
        assert torch.equal(got.cpu().view(U8).view(-1), codes.view(U8).view(-1))

"""The low-bit operators without a GPU: the 64-bit forms the GPU tests compare
with, sizes that are host arithmetic, and every refusal - none of these calls
reaches a launch."""

import pytest
import torch

import lowbit

BF, I32 = torch.bfloat16, torch.int32


def test_mxfp4_reference_values():
    x = torch.zeros(1, 64)
    x[0, :8] = torch.tensor([7.9, 0.25, 0.75, 2.5, -3.5, 5.0, 1.0, -0.1])
    x[0, 32] = 1e-40
    code, sc, val = lowbit.mxfp4(x)
    assert sc.tolist() == [[127, 0]]                       # floor(log2 7.9) - 2 = 0; below 2^-124: code 0
    # 7.9 saturates; ties 0.25, 0.75, 2.5, 3.5, 5 go to the even code
    assert val[0, :8].tolist() == [6.0, 0.0, 1.0, 2.0, -4.0, 4.0, 1.0, -0.0]
    assert code[0, :8].tolist() == [7, 0, 2, 4, 14, 6, 2, 8]
    assert torch.equal(lowbit.mxfp4_values(lowbit.pack_nibbles(code), sc), val)


def test_mxfp4_reference_non_finite_block():
    x = torch.ones(1, 64)
    x[0, 3] = float("inf")
    code, sc, val = lowbit.mxfp4(x)
    assert sc.tolist() == [[255, 125]] and bool(val[0, :32].isnan().all()) and not bool(val[0, 32:].isnan().any())


def test_record_bytes():
    from dsv4attn import ops
    from dsv4attn import _lib
    assert ops.kv_quant_row_bytes(512, 64) == 608          # 448 + 128 + 28, up to a multiple of 32
    assert ops.kv_quant_row_bytes(128, 0) == 160
    assert ops.kv_quant_row_bytes(96, 32) == 160
    for D, r in ((512, 60), (512, 512), (500, 64), (0, 0), (8256, 64), (64, -8)):
        assert _lib.lib().dsa_kv_quant_row_bytes(D, r) == 0
        with pytest.raises(ValueError, match="multiple"):
            ops.kv_quant_row_bytes(D, r)


def test_cache_views():
    from dsv4attn import ops
    cache = ops.kv_quant_cache(2, 5, device="cpu")
    codes, rope, scales = ops.kv_quant_views(cache)
    assert codes.shape == (2, 5, 448) and rope.shape == (2, 5, 64) and scales.shape == (2, 5, 7)
    scales[1, 4, 6] = 1.0
    rope[1, 4, 0] = 1.0
    assert cache[1, 4, 448:450].view(BF).item() == 1.0 and cache[1, 4, 600:604].view(torch.float32).item() == 1.0
    with pytest.raises(ValueError, match="608"):
        ops.kv_quant_views(torch.zeros(2, 5, 600, dtype=torch.uint8))


def test_ops_refuse_cpu_tensors():
    from dsv4attn import ops
    cache = ops.kv_quant_cache(1, 8, device="cpu")
    pos = torch.zeros(1, dtype=I32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.mxfp4_quant(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_quant_write(torch.zeros(1, 512, dtype=BF), cache, pos, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_quant_read(cache)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sparse_attn_quant(torch.zeros(1, 64, 512, dtype=BF), cache, torch.zeros(1, 4, dtype=I32), torch.zeros(64), 0.1)


# --------------------------------------------------- refusals of the C entries
# pointers are 16-byte-aligned numbers that nothing reads: every call returns
# before it touches the GPU

def _refused(rc, *words):
    from dsv4attn import _lib
    assert rc == _lib.DSA_ERR_ARG, rc
    msg = _lib.last_error()
    assert all(w in msg for w in words), msg


def test_mxfp4_quant_refusals():
    from dsv4attn import _lib
    f = _lib.lib().dsa_mxfp4_quant
    _refused(f(None, 0, 64, None, 0, 16, 16, 1, 64, None), "null")
    _refused(f(16, 0, 64, None, 0, None, 16, 1, 64, None), "null")
    _refused(f(16, 3, 64, None, 0, 16, 16, 1, 64, None), "x_type")
    _refused(f(16, 0, 48, None, 0, 16, 16, 1, 48, None), "32")
    _refused(f(16, 0, 64, None, 0, 16, 16, -1, 64, None), "M/K")
    _refused(f(16, 0, 32, None, 0, 16, 16, 1, 64, None), "stride")
    _refused(f(16, 0, 68, None, 0, 16, 16, 2, 64, None), "16 bytes")
    _refused(f(8, 0, 64, None, 0, 16, 16, 1, 64, None), "alignment")
    _refused(f(16, 0, 64, 8, 64, 16, 16, 1, 64, None), "out")
    _refused(f(16, 0, 64, None, 0, 18, 16, 1, 64, None), "codes")
    assert f(16, 0, 64, None, 0, 16, 16, 0, 64, None) == _lib.DSA_OK


def test_kv_quant_write_refusals():
    from dsv4attn import _lib
    f = _lib.lib().dsa_kv_quant_write
    ok = dict(kv=16, ld_b=512, ld_s=512, cache=16, bs=608 * 8, rows=8, pos=16, n=None, B=2, S=1, D=512, r=64, win=8,
              off=0, st=None)

    def call(**kw):
        return f(*{**ok, **kw}.values())
    _refused(call(kv=None), "null")
    _refused(call(pos=None), "null")
    _refused(call(r=60), "multiple of 64")
    _refused(call(D=8256), "8192")
    _refused(call(rows=0), "rows")
    _refused(call(bs=608 * 7), "batch stride")
    _refused(call(bs=608 * 8 + 8), "16-byte")
    _refused(call(cache=24), "16-byte")
    _refused(call(win=0), "ring")
    _refused(call(off=1), "ring")
    _refused(call(off=-1), "ring")
    _refused(call(kv=18), "kv needs")
    _refused(call(ld_s=516), "kv needs")
    _refused(call(B=-1), "B/rows")
    assert call(B=0) == _lib.DSA_OK and call(S=0) == _lib.DSA_OK


def test_kv_quant_read_refusals():
    from dsv4attn import _lib
    f = _lib.lib().dsa_kv_quant_read
    ok = dict(cache=16, bs=608 * 8, rows=8, idx=16, ld=4, out=16, f32=0, B=2, K=4, D=512, r=64, status=None, st=None)

    def call(**kw):
        return f(*{**ok, **kw}.values())
    _refused(call(cache=None), "null")
    _refused(call(out=None), "null")
    _refused(call(ld=3), "ld_idx")
    _refused(call(idx=None, K=9), "more rows")
    _refused(call(out=24), "aligned")
    _refused(call(D=500), "multiple of 64")
    _refused(call(K=-1), "K")
    assert call(B=0) == _lib.DSA_OK and call(K=0) == _lib.DSA_OK


def test_sparse_attn_quant_refusals():
    from dsv4attn import _lib
    f = _lib.lib().dsa_sparse_attn_quant
    ok = dict(q=16, cache=16, bs=608 * 8, rows=8, idx=16, ld=4, sink=16, out=16, lse=None, B=2, S=1, H=64, D=512, K=4,
              scale=1.0, ws=None, wsb=0, status=None, st=None)

    def call(**kw):
        return f(*{**ok, **kw}.values())
    _refused(call(q=None), "null")
    _refused(call(sink=None), "null")
    _refused(call(H=32), "H=64")
    _refused(call(D=576), "D=512")
    _refused(call(bs=608 * 7), "stride")
    _refused(call(bs=608 * 8 + 8), "stride")
    _refused(call(ld=3), "ld_idx")
    _refused(call(q=24), "aligned")
    _refused(call(B=32768, S=2), "65535")
    assert call(B=0) == _lib.DSA_OK


def test_linear_mxfp4_refusals():
    from dsv4attn import _lib
    L = _lib.lib()
    assert L.dsa_linear_mxfp4_packed_bytes(128, 256) == 17408
    assert L.dsa_linear_mxfp4_packed_bytes(129, 288) == 2 * 2 * 17408
    assert L.dsa_linear_mxfp4_packed_bytes(128, 48) == 0 and L.dsa_linear_mxfp4_packed_bytes(0, 64) == 0
    assert L.dsa_linear_mxfp4_packed_bytes(1 << 25, 64) == 0
    assert L.dsa_linear_mxfp4_workspace_size(0, 64, 64) == 0 and L.dsa_linear_mxfp4_workspace_size(4, 64, 48) == 0
    # a few tokens are quantised by the product itself; many need room for their codes and scales
    assert L.dsa_linear_mxfp4_workspace_size(4, 64, 64) == 0
    assert L.dsa_linear_mxfp4_workspace_size(100, 64, 1536) >= 100 * 1536 * 17 // 32
    p = L.dsa_linear_mxfp4_pack
    _refused(p(None, 16, 128, 256, 16, 17408, None), "null")
    _refused(p(16, 16, 128, 250, 16, 17408, None), "multiple of 32")
    _refused(p(8, 16, 128, 256, 16, 17408, None), "aligned")
    _refused(p(16, 16, 128, 256, 16, 17407, None), "packed buffer")
    f = L.dsa_linear_mxfp4
    ok = dict(x=16, xt=0, ld_x=256, w=16, y=16, ld_y=128, B=2, N=128, K=256, f32=0, ws=16, wsb=1 << 20, status=None,
              st=None)

    def call(**kw):
        return f(*{**ok, **kw}.values())
    _refused(call(x=None), "null")
    _refused(call(w=None), "null")
    _refused(call(xt=7), "x_type")
    _refused(call(K=250), "multiple of 32")
    _refused(call(B=-1), "B/N/K")
    _refused(call(N=1 << 25), "2^24")
    _refused(call(ld_x=255), "row stride")
    _refused(call(ld_x=260), "16 bytes")
    _refused(call(x=8), "alignment")
    _refused(call(ld_y=127), "ld_y")
    _refused(call(y=17), "aligned")
    big = dict(B=100, K=1536, ld_x=1536)
    assert call(wsb=100, **big) == _lib.DSA_ERR_WORKSPACE and "workspace" in _lib.last_error()
    assert call(ws=None, **big) == _lib.DSA_ERR_WORKSPACE
    assert call(B=0) == _lib.DSA_OK


def test_a_missing_module_is_an_error(monkeypatch):
    import sys
    from dsv4attn import _lib
    monkeypatch.setitem(sys.modules, "dsv4attn._torch_ops", None)
    monkeypatch.delattr("dsv4attn._torch_ops", raising=False)
    with pytest.raises(_lib.NativeLibraryError, match="build.py"):
        _lib.torch_ops()


def test_a_ring_behind_the_cache_is_refused_at_any_offset():
    """offset + win past 2^63 must not come round to a small number."""
    from dsv4attn import _lib
    f = _lib.lib().dsa_kv_quant_write
    for offset in (2**63 - 8, 2**63 - 1, 2**62, 1):
        _refused(f(16, 512, 512, 16, 608 * 8, 8, 16, None, 2, 0, 512, 64, 8, offset, None), "ring")
    assert f(16, 512, 512, 16, 608 * 8, 8, 16, None, 2, 0, 512, 64, 8, 0, None) == _lib.DSA_OK


def test_a_packed_weight_smaller_than_its_sizes_is_refused():
    """The kernel streams ceil(N/128) x ceil(K/256) tiles of 17,408 bytes."""
    from dsv4attn import ops
    x = torch.zeros(2, 512, dtype=BF)
    tiles = 2 * 2 * 17408                                  # N = 129, K = 512
    bad = [(torch.zeros(tiles - 1, dtype=torch.uint8), 129, 512), (torch.zeros(tiles, dtype=torch.uint8), 257, 512),
           (torch.zeros(tiles, dtype=torch.int8), 129, 512), (torch.zeros(2 * tiles, dtype=torch.uint8)[::2], 129, 512),
           (torch.zeros(tiles, dtype=torch.uint8), 129, 500), (torch.zeros(tiles, dtype=torch.uint8), 0, 512),
           (torch.zeros(tiles, dtype=torch.uint8), 2**32 + 129, 512)]
    for packed, N, K in bad:
        with pytest.raises(ValueError, match="packed"):
            ops.linear_mxfp4(x, ops.MXFP4Weight(packed, N, K))
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_mxfp4(x, ops.MXFP4Weight(torch.zeros(tiles, dtype=torch.uint8), 129, 512))


def test_attention_refuses_an_index_list_whose_tiles_wrap():
    """K + 63 must stay below 2^31: a wrapped tile count attended the first 64
    entries only.  (A list this long is 8 GB of indices for one query row.)"""
    from dsv4attn import _lib
    L = _lib.lib()
    for K in (2**31 - 1, 2**31 - 64, 2**31 - 4096):
        assert L.dsa_sparse_attn_workspace_size(1, 1, 64, 512, K) == 0
        _refused(L.dsa_sparse_attn_quant(16, 16, 608 * 8, 8, 16, K, 16, 16, None, 1, 1, 64, 512, K, 1.0, None, 0, None,
                                         None), "K")
        _refused(L.dsa_sparse_attn(16, 16, 512 * 8, 8, 16, K, 16, 16, None, 1, 1, 64, 512, K, 1.0, None, 0, None, None),
                 "K")
    assert L.dsa_sparse_attn_workspace_size(1, 1, 64, 512, 2**31 - 8192) > 2**31


def test_the_package_imports_on_a_torch_without_cuda():
    import os
    import subprocess
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-deepseek-v4_b200")
    code = ("import sys, torch; del torch._C._cuda_getCurrentRawStream; sys.path.insert(0, sys.argv[1]); "
            "import dsv4attn; from dsv4attn import modules, ops")
    subprocess.run([sys.executable, "-c", code, pkg], check=True, timeout=300)


def test_the_module_is_rebuilt_for_another_torch_or_python(monkeypatch, tmp_path):
    """The compiled module links torch's C++ internals, so file times alone do
    not say that it is up to date."""
    from types import SimpleNamespace

    import build
    ran = []

    def run(cmd, check):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "_torch_ops.so"))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "subprocess", SimpleNamespace(run=run))
    assert build.build_torch_ops() == build.TORCH_LIB and len(ran) == 1
    build.build_torch_ops()
    assert len(ran) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build_torch_ops()
    build.build_torch_ops()
    assert len(ran) == 2
    monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    build.build_torch_ops()
    assert len(ran) == 3
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "another python")
    build.build_torch_ops()
    build.build_torch_ops()
    assert len(ran) == 4


def _fl32(v):
    """The fp32 number nearest to a Fraction, ties to even (no range ends)."""
    from fractions import Fraction
    if v == 0:
        return v
    a, e = abs(v), 0
    e = a.numerator.bit_length() - a.denominator.bit_length()
    if Fraction(2) ** e > a:
        e -= 1
    step = Fraction(2) ** (e - 23)
    n = round(a / step)                                    # (Fraction's round: half to even)
    return n * step if v > 0 else -n * step


def test_the_cache_writes_quotient_is_correctly_rounded():
    """q = fl(x r), e = fl(q s - x), fl(q - e r) with r = fl(1 / s) is fl(x / s)
    for every bf16 significand x over every scale s = fl(m fl(1/448)) of a bf16
    maximum m, and over the smallest scale.  (e is not always exact: q can be
    more than an ulp off.)"""
    from fractions import Fraction
    inv = _fl32(Fraction(1, 448))
    eps = _fl32(Fraction(1, 10000))
    scales = [_fl32(Fraction(128 + i, 128) * inv) for i in range(128)] + [_fl32(eps * inv)]
    inexact = 0
    for s in scales:
        r = _fl32(1 / s)
        for j in range(128):
            x = Fraction(128 + j, 128)
            q = _fl32(x * r)
            e = _fl32(q * s - x)
            inexact += e != q * s - x
            assert _fl32(q - e * r) == _fl32(x / s), (x, s)
    assert inexact == 21                                   # of 129 x 128


def test_mxfp4_quant_refuses_an_out_that_partly_covers_x():
    """out is x itself, a block of columns beside x's, or elsewhere: anything
    else would overwrite elements that other CTAs have still to read."""
    from dsv4attn import _lib
    f = _lib.lib().dsa_mxfp4_quant
    at, M, K, ld = 1 << 20, 4, 64, 256                     # bf16: rows of 512 B, 128 B of them used
    for out, ld_out in ((at, ld + 8), (at + 64, ld), (at - 64, ld), (at + 3 * 512 + 112, ld), (at - 3 * 512 - 112, ld),
                        (at + 512, ld), (at + 400, ld), (at + 128, 64), (at + 1664 - 16, ld)):
        _refused(f(at, 0, ld, out, ld_out, 16, 16, M, K, None), "overlap")
    _refused(f(at, 2, 256, at + 256, 256, 16, 16, 2, 128, None), "overlap")   # fp32

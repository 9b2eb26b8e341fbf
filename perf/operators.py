"""The low-bit operators of a decode layer, for measurement: MXFP4 quantisation, the MXFP4 projection, the FP8 latent
cache (rows quantised as they are written, read back) and the sparse attention that reads that cache.

A decode layer streams two things: its projection weights and the latent rows that its queries select.  These
operators keep both at few bits.  Sizes are the decode path's own: model width 4096, q rank 1024, 64 heads of 512
dims (448 plus 64 rotary), a 128-slot window ring before 8192 compressed rows, top-2048 plus the window selected.
"""

import math
import os
import sys

import torch

own = False

H, D, ROPE = 64, 512, 64         # heads, latent row, its rotary dims
WIN, ROWS = 128, 128 + 8192      # window ring, rows of a sequence's cache at a 32768-token context
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _ops():
    """The framework's operators (its package folder is not a Python name, so it goes on the path)."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-deepseek-v4_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from dsv4attn import ops
    return ops


# ------------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the activations of a decode batch of 64 tokens, before a projection
        {"name": "quant_batch", "op": "quant", "M": 64, "K": 4096, "dtype": "bfloat16"},
        # a master weight of the q up-projection, converted at load time
        {"name": "quant_weight", "op": "quant", "M": 32768, "K": 1024, "dtype": "float32"},
        # one token through the q down-projection: pure latency
        {"name": "linear_one", "op": "linear", "B": 1, "N": 1024, "K": 4096, "f32": False},
        # a decode batch through the q up-projection: the layer's largest weight, streamed
        {"name": "linear_batch", "op": "linear", "B": 64, "N": 32768, "K": 1024, "f32": False},
        # odd sizes all over, unrounded result
        {"name": "linear_odd", "op": "linear", "B": 333, "N": 2001, "K": 4128, "f32": True},
        # a 4096-token prefill chunk through the output projection
        {"name": "linear_chunk", "op": "linear", "B": 4096, "N": 4096, "K": 8192, "f32": False},
        # one decode step of 64 sequences: one row each into the window ring
        {"name": "write_step", "op": "write", "B": 64, "S": 1, "rows": ROWS, "win": WIN, "offset": 0, "D": D, "rope": ROPE, "ragged": False},
        # compressed rows of a padded prefill batch, behind the ring
        {"name": "write_chunk", "op": "write", "B": 8, "S": 4001, "rows": ROWS, "win": ROWS - WIN, "offset": WIN, "D": D, "rope": ROPE, "ragged": True},
        # one sequence's whole cache back as bf16 rows
        {"name": "read_one", "op": "read", "B": 1, "rows": ROWS, "K": 0, "D": D, "rope": ROPE},
        # the selected rows of 64 sequences
        {"name": "read_selected", "op": "read", "B": 64, "rows": ROWS, "K": 2176, "D": D, "rope": ROPE},
        # a single sequence decoding over its selection
        {"name": "attn_one", "op": "attn", "B": 1, "S": 1, "rows": ROWS, "K": 2176},
        # the decode batch
        {"name": "attn_batch", "op": "attn", "B": 64, "S": 1, "rows": ROWS, "K": 2176},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "linear", "write", "read", "attn"])
    if op == "quant":
        K = 32 * _log(rng, 1, 256)
        return {"op": op, "M": _log(rng, 1, min(32768, (1 << 25) // K)), "K": K, "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    if op == "linear":
        K = 32 * _log(rng, 1, 256)
        N = _log(rng, 1, min(32768, (1 << 25) // K))
        return {"op": op, "B": _log(rng, 1, min(4096, (1 << 37) // (K * N))), "N": N, "K": K, "f32": rng.random() < 0.3}
    if op == "write":
        B, S = _log(rng, 1, 64), 1 if rng.random() < 0.3 else _log(rng, 2, 4096)
        while B * S > 40000:
            B = max(1, B // 2)
        offset = rng.choice([0, WIN])
        win = rng.choice([WIN, _log(rng, 16, 4096)])
        nope, rope = rng.choice([(448, 64), (512, 64), (128, 0), (64, 32)])
        return {"op": op, "B": B, "S": S, "rows": offset + win + rng.randrange(40), "win": win, "offset": offset, "D": nope + rope, "rope": rope, "ragged": rng.random() < 0.5}
    if op == "read":
        B, rows = _log(rng, 1, 64), _log(rng, 100, ROWS)
        nope, rope = rng.choice([(448, 64), (512, 64), (128, 0), (64, 32)])
        return {"op": op, "B": B, "rows": rows, "K": 0 if B * rows < 140000 and rng.random() < 0.3 else _log(rng, 1, 2176), "D": nope + rope, "rope": rope}
    S = 1 if rng.random() < 0.6 else _log(rng, 2, 64)
    K = _log(rng, 1, 2304)
    return {"op": op, "B": _log(rng, 1, max(1, min(64, 139264 // (S * K)))), "S": S, "rows": _log(rng, 100, ROWS), "K": K}


def work(case):
    op = case["op"]
    if op == "quant":
        n, size = case["M"] * case["K"], 4 if case["dtype"] == "float32" else 2
        # values in, values out, codes and block scales
        return {"bytes": n * (2 * size + 0.5 + 1 / 32), "flops": 3 * n}
    if op == "linear":
        B, N, K = case["B"], case["N"], case["K"]
        return {"bytes": N * K * (0.5 + 1 / 32) + 2 * B * K + (4 if case["f32"] else 2) * B * N, "flops": 2 * B * N * K}
    if op in ("write", "read"):
        nope, rope = case["D"] - case["rope"], case["rope"]
        row = 2 * case["D"] + nope + 2 * rope + nope // 16  # bf16 on one side; codes, rotary dims and scales on the other
        n = case["B"] * (min(case["S"], case["win"]) if op == "write" else case["K"] or case["rows"])
        if op == "write" and case["ragged"]:
            n = n * 5 / 8  # between a quarter of the tokens and all of them
        return {"bytes": n * (row + (4 if case.get("K") else 0)), "flops": 3 * n * nope}
    M, K = case["B"] * case["S"], case["K"]
    rows = min(M * K * 0.95, case["B"] * case["rows"])  # one index in twenty is masked
    return {"bytes": rows * (D - ROPE + 2 * ROPE + (D - ROPE) // 16) + 4 * M * K + 4 * M * H * D, "flops": 4 * M * K * 0.95 * H * D}


# --------------------------------------------------------------------------------------------------- plain forms

def _mx_parts(x):
    """MXFP4 blocks of 32 along the last dim: (signed E2M1 values [.., K/32, 32], exponents [.., K/32, 1])."""
    x = x.float().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(-127, 127)  # floor(log2 amax) - 2
    a = torch.ldexp(x.abs(), -e).clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(a / step) * step * torch.sign(x), e


def _mx_values(codes, scales):
    """fp32 values of MXFP4 codes [N, K/2] (even element in the low nibble) and UE8M0 scales [N, K/32]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return torch.ldexp(table[nib].unflatten(-1, (-1, 32)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _row_bytes(nope, rope):
    return (nope + 2 * rope + nope // 16 + 31) // 32 * 32


def _records(kv, rope):
    """Cache records of bf16 rows [.., D]: e4m3 codes of the first D - rope dims, the rotary dims as they are, one
    fp32 scale for each 64 codes, zeros up to a multiple of 32 bytes."""
    nope = kv.shape[-1] - rope
    x = kv[..., :nope].float().unflatten(-1, (-1, 64))
    s = x.abs().amax(-1, keepdim=True).clamp(min=1e-4) * torch.tensor(1.0 / 448.0, device=kv.device)
    codes = (x / s).clamp(-448, 448).to(torch.float8_e4m3fn).flatten(-2).view(torch.uint8)
    parts = [codes, kv[..., nope:].contiguous().view(torch.uint8), s.squeeze(-1).contiguous().view(torch.uint8)]
    pad = _row_bytes(nope, rope) - sum(p.shape[-1] for p in parts)
    return torch.cat(parts + [codes.new_zeros(*codes.shape[:-1], pad)], -1)


def _fields(rec, nope, rope):
    """(codes, rotary dims, scales) of cache records [.., row bytes], as views."""
    a, b = nope, nope + 2 * rope
    return rec[..., :a].view(torch.float8_e4m3fn), rec[..., a:b].view(torch.bfloat16), rec[..., b:b + nope // 16].view(torch.float32)


def _row_values(rec, nope, rope):
    """bf16 rows of cache records: code times scale, rounded to bf16."""
    codes, r, s = _fields(rec, nope, rope)
    x = codes.float().unflatten(-1, (-1, 64)) * s.unsqueeze(-1)
    return torch.cat([x.flatten(-2).bfloat16(), r], -1)


def _targets(state):
    """(sequence, token, row) of every token that a write puts down."""
    case, pos, n = state["case"], state["pos"].long(), state["n_valid"]
    s = torch.arange(case["S"], device=pos.device)
    n = torch.full_like(pos, case["S"]) if n is None else n.long()
    keep = (s < n[:, None]) & (s >= n[:, None] - case["win"])
    row = case["offset"] + (pos[:, None] + s) % case["win"]
    b, t = keep.nonzero(as_tuple=True)
    return b, t, row[b, t]


def _attend(q, kv, idx, sink, scale):
    """Softmax attention over the selected rows with a sink logit in the denominator; -1 masks a place."""
    s = torch.matmul(q, kv.transpose(-1, -2)) * scale
    s = s.masked_fill((idx < 0).unsqueeze(-2), float("-inf"))
    m = torch.maximum(s.amax(-1, keepdim=True), sink[:, None])
    p = torch.exp(s - m)
    return torch.matmul(p, kv) / (p.sum(-1, keepdim=True) + torch.exp(sink[:, None] - m))


def _gather(cache, idx):
    b = torch.arange(cache.shape[0], device=idx.device).reshape(-1, *([1] * (idx.dim() - 1)))
    return cache[b, idx.long().clamp(min=0)]


# ------------------------------------------------------------------------------------------------------- inputs

def _make_cache(g, B, rows, nope, rope):
    # rows as an RMS norm leaves them, some dims larger than others
    x = torch.randn(B, rows, nope + rope, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(nope + rope, generator=g, device="cuda"))
    return _records(x.bfloat16(), rope)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, dev = case["op"], "cuda"
    state = {"case": case}
    if op == "quant":
        x = torch.randn(case["M"], case["K"], generator=g, device=dev)
        x *= torch.exp(torch.randn(case["M"], 1, generator=g, device=dev))  # tokens of different size
        state["x"] = x.to(getattr(torch, case["dtype"]))
    elif op == "linear":
        N, K = case["N"], case["K"]
        state["x"] = torch.randn(case["B"], K, generator=g, device=dev).bfloat16()
        w = torch.randn(N, K, generator=g, device=dev) * K ** -0.5
        w *= torch.exp(0.5 * torch.randn(N, 1, generator=g, device=dev))
        # a checkpoint's weight: packed E2M1 codes and UE8M0 scales
        v, e = _mx_parts(w)
        mag = torch.bucketize(v.abs(), torch.tensor(E2M1, device=dev))
        nib = (mag + 8 * (v < 0)).to(torch.uint8).flatten(-2)
        state["codes"] = nib[:, 0::2] | (nib[:, 1::2] << 4)
        state["scales"] = (e.squeeze(-1) + 127).to(torch.uint8)
        if own:  # laid out once at load time, as every projection weight of the framework is
            state["w"] = _ops().pack_linear_weight_mxfp4(state["codes"], state["scales"])
    elif op == "write":
        B, S = case["B"], case["S"]
        nope = case["D"] - case["rope"]
        state["kv"] = torch.randn(B, S, case["D"], generator=g, device=dev).bfloat16()
        state["cache"] = torch.zeros(B, case["rows"], _row_bytes(nope, case["rope"]), dtype=torch.uint8, device=dev)
        state["pos"] = torch.randint(0, 32768, (B,), generator=g, device=dev, dtype=torch.int32)
        state["n_valid"] = torch.randint(S // 4, S + 1, (B,), generator=g, device=dev, dtype=torch.int32) if case["ragged"] else None
    else:
        B, rows, K = case["B"], case["rows"], case["K"]
        rope = case.get("rope", ROPE)
        state["cache"] = _make_cache(g, B, rows, case.get("D", D) - rope, rope)
        if K:
            shape = (B, case["S"], K) if op == "attn" else (B, K)
            idx = torch.randint(0, rows, shape, generator=g, device=dev, dtype=torch.int32)
            idx[torch.rand(shape, generator=g, device=dev) < 0.05] = -1
            state["idx"] = idx.sort(-1, descending=False).values
        else:
            state["idx"] = None
        if op == "attn":
            state["q"] = torch.randn(B, case["S"], H, D, generator=g, device=dev).bfloat16()
            state["sink"] = torch.randn(H, generator=g, device=dev)
    return state


# ---------------------------------------------------------------------------------------------------------- run

def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        o = _ops()
        if op == "quant":
            out, scales, codes = o.mxfp4_quant(state["x"], out=True)
            return {"values": out, "scales": scales.view(torch.float8_e8m0fnu)}
        if op == "linear":
            return {"y": o.linear_mxfp4(state["x"], state["w"], out_f32=case["f32"])}
        if op == "write":
            o.kv_quant_write(state["kv"], state["cache"], state["pos"], case["win"], offset=case["offset"],
                             rope_dim=case["rope"], n_valid=state["n_valid"])
            codes, rope, scales = o.kv_quant_views(state["cache"], case["D"], case["rope"])
            return {"codes": codes, "rope": rope, "scales": scales}
        if op == "read":
            return {"kv": o.kv_quant_read(state["cache"], state["idx"], D=case["D"], rope_dim=case["rope"])}
        return {"o": o.sparse_attn_quant(state["q"], state["cache"], state["idx"], state["sink"], D ** -0.5)}
    if op == "quant":
        v, e = _mx_parts(state["x"])
        return {"values": torch.ldexp(v, e).flatten(-2).to(state["x"].dtype),
                "scales": (e.squeeze(-1) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)}
    if op == "linear":
        v, e = _mx_parts(state["x"])
        y = torch.matmul(torch.ldexp(v, e).flatten(-2), _mx_values(state["codes"], state["scales"]).t())
        return {"y": y if case["f32"] else y.bfloat16()}
    nope, rope = case.get("D", D) - case.get("rope", ROPE), case.get("rope", ROPE)
    if op == "write":
        b, t, row = _targets(state)
        state["cache"][b, row] = _records(state["kv"][b, t], rope)
        codes, r, scales = _fields(state["cache"], nope, rope)
        return {"codes": codes, "rope": r, "scales": scales}
    idx = state["idx"]
    if op == "read":
        if idx is None:
            return {"kv": _row_values(state["cache"], nope, rope)}
        return {"kv": _row_values(_gather(state["cache"], idx), nope, rope).masked_fill((idx < 0).unsqueeze(-1), 0)}
    kv = _row_values(_gather(state["cache"], idx), nope, rope).float()
    return {"o": _attend(state["q"].float(), kv, idx, state["sink"], D ** -0.5).bfloat16()}


# -------------------------------------------------------------------------------------------------------- exact

def _near(a, mantissa, low):
    """|a| rounded to `mantissa` bits behind the leading one, evenly spaced below 2^low; ties to even."""
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** low))).clamp(min=low)
    e = torch.where(torch.exp2(e) > a, e - 1, e).clamp(min=low)
    step = torch.exp2(e - mantissa)
    return torch.round(a / step) * step


def _mx_exact(x):
    x = x.double().reshape(*x.shape[:-1], -1, 32)
    top = x.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)))
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    scale = torch.exp2((e - 2).clamp(-127, 127))
    return _near((x.abs() / scale).clamp(max=6.0), 1, 0) * x.sign() * scale, scale.squeeze(-1)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        v, s = _mx_exact(state["x"])
        return {"values": v.reshape(state["x"].shape), "scales": s}
    if op == "linear":
        x = _mx_exact(state["x"])[0].reshape(state["x"].shape)
        mags = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
        w = torch.empty(case["N"], case["K"], dtype=torch.float64, device="cuda")
        for half in (0, 1):
            c = (state["codes"] >> (4 * half)) & 15
            w[:, half::2] = mags[(c & 7).long()] * (1 - 2 * (c >> 3).double())
        w = w.reshape(case["N"], -1, 32) * torch.exp2(state["scales"].double() - 127)[..., None]
        return {"y": x @ w.reshape(case["N"], -1).T}
    rope = case.get("rope", ROPE)
    nope = case.get("D", D) - rope
    if op == "write":
        b, t, row = _targets(state)
        kv = state["kv"].double()
        x = kv[..., :nope].reshape(*kv.shape[:2], -1, 64)
        s = x.abs().max(-1, keepdim=True).values.clamp(min=1e-4) / 448
        q = (_near((x / s).abs(), 3, -6).clamp(max=448) * x.sign()).reshape(*kv.shape[:2], nope)
        full = lambda n: torch.zeros(case["B"], case["rows"], n, dtype=torch.float64, device="cuda")  # noqa: E731
        out = {"codes": full(nope), "rope": full(rope), "scales": full(nope // 64)}
        out["codes"][b, row] = q[b, t]
        out["rope"][b, row] = kv[b, t, nope:]
        out["scales"][b, row] = s[b, t, :, 0]
        return out

    def rows_of(rec):
        codes = rec[..., :nope].contiguous().view(torch.float8_e4m3fn).double()
        r = rec[..., nope:nope + 2 * rope].contiguous().view(torch.bfloat16).double()
        s = rec[..., nope + 2 * rope:nope + 2 * rope + nope // 16].contiguous().view(torch.float32).double()
        return torch.cat([codes * s.repeat_interleave(64, -1), r], -1)

    idx = state["idx"]
    if op == "read":
        if idx is None:
            return {"kv": rows_of(state["cache"])}
        return {"kv": rows_of(_gather(state["cache"], idx)) * (idx >= 0).unsqueeze(-1)}
    out = []
    for b in range(case["B"]):  # a sequence at a time: the rows in 64 bits are large
        ids = idx[b]
        kv = rows_of(state["cache"][b][ids.long().clamp(min=0)])
        s = torch.einsum("shd,skd->shk", state["q"][b].double(), kv) * D ** -0.5
        w = torch.exp(s) * (ids >= 0).unsqueeze(1)
        z = w.sum(-1) + torch.exp(state["sink"].double())
        out.append(torch.einsum("shk,skd->shd", w, kv) / z.unsqueeze(-1))
    return {"o": torch.stack(out)}

"""The operators that serve ``ADTModel.sample`` in few bits, as measured cases: the 8-bit-integer linear layer and the 4-bit K/V cache.

Three operators, each as a user's program calls it (``own = True``) and in plain torch operations (``own = False``):

  linear_i8   bf16 / fp32 activations -> one scale per row (token), int8 products with int8 weights that carry one scale per output channel
  kv4_append  new K and V rows -> 4 bits per value with a scale and a minimum per 64 channels, placed in the cache; the rows are then read back
  attn_kv4    softmax attention of one or a few query positions per sequence over such a cache (grouped heads, ragged lengths, causal)

Sizes: the setting-1 network (768 wide, 6 heads of 128 channels, 1400 tokens, 986 frames of a 10 s clip, up to 1000 positions), and generic ones.
"""
import math
import random

import torch

own = False

TINY = 2.0 ** -100                 # smallest row magnitude / group scale: an all-zero row has this one, and codes of zero
GROUP = 64                         # channels that share a scale and a minimum in the 4-bit cache
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
TYPES = {"bf16": BF16, "f32": F32}


# --------------------------------------------------------------------------------------------------------------------- cases
def _linear(name, rows, n, k, x="bf16", out="bf16", bias=True, act=0, residual=False):
    c = dict(op="linear_i8", rows=rows, n=n, k=k, x=x, out=out, bias=bias, act=act, residual=residual)
    return dict(c, name=name) if name else c


def _append(name, batch, kv_heads, dim, keys, new, ragged):
    c = dict(op="kv4_append", batch=batch, kv_heads=kv_heads, dim=dim, keys=keys, new=new, ragged=ragged)
    return dict(c, name=name) if name else c


def _attn(name, batch, heads, kv_heads, dim, keys, q_len, causal, ragged):
    c = dict(op="attn_kv4", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, keys=keys, q_len=q_len, causal=causal, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one clip's decode step: the packed in-projection of a single token (weights only, latency)
        _linear("linear_one_token", 1, 2304, 768),
        # a decode step of 64 clips: the generator, fp32 logits
        _linear("linear_step_64", 64, 1400, 768, out="f32"),
        # the decoder over 61 whole prefixes of 127 tokens: the attention's output projection added to the fp32 residual stream, ragged rows
        _linear("linear_prefix_residual", 61 * 127, 768, 768, out="f32", residual=True),
        # the encoder over 64 clips of 10 s: the packed in-projection
        _linear("linear_encoder", 64 * 986, 2304, 768),
        # a generic square layer with GELU on fp32 activations: the matrix units' bound
        _linear("linear_square_gelu", 4096, 4096, 4096, x="f32", act=1),
        # one new position of 64 sequences, mid-cache
        _append("append_step_64", 64, 6, 128, 1000, 1, True),
        # the encoder memory of 64 clips, projected to K and V once per clip
        _append("append_memory_64", 64, 6, 128, 986, 986, False),
        # chunks of different lengths behind different prefixes, narrow heads
        _append("append_ragged_64ch", 33, 5, 64, 1500, 777, True),
        # one clip: a query per head over the 986 frames (latency)
        _attn("attn_one_clip", 1, 6, 6, 128, 986, 1, False, False),
        # 256 clips a step: the cross-attention's read of every clip's memory
        _attn("attn_step_256", 256, 6, 6, 128, 986, 1, False, False),
        # grouped heads over long, ragged contexts
        _attn("attn_grouped_long", 8, 32, 8, 128, 32000, 1, False, True),
        # a few new positions of each sequence at once behind ragged prefixes, narrow heads, causal
        _attn("attn_chunk_causal", 24, 10, 5, 64, 3001, 7, True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_i8", "kv4_append", "attn_kv4"])
    if op == "linear_i8":
        n, k = _log(rng, 33, 5000), _log(rng, 50, 5000)
        rows = _log(rng, 1, max(1, min(65000, int(6.8e10 / (n * k)))))
        return _linear(None, rows, n, k, rng.choice(["bf16", "f32"]), rng.choice(["bf16", "f32"]), rng.random() < 0.7, rng.choice([0, 0, 1]), rng.random() < 0.3)
    dim, kv_heads = rng.choice([64, 128]), rng.randint(1, 8)
    if op == "kv4_append":
        batch, keys = _log(rng, 1, 100), _log(rng, 1, 4000)
        batch = max(1, min(batch, int(4.8e7 / (keys * kv_heads * dim))))
        new = min(keys, _log(rng, 1, keys)) if rng.random() < 0.7 else 1
        return _append(None, batch, kv_heads, dim, keys, new, rng.random() < 0.6)
    q_len = rng.choice([1, 1, 1, rng.randint(2, 9)])
    batch, keys = _log(rng, 1, 256), _log(rng, 1, 32000)
    batch = max(1, min(batch, int(2.4e8 / (keys * kv_heads * dim * q_len))))
    return _attn(None, batch, kv_heads * rng.choice([1, 1, 2, 4]), kv_heads, dim, keys, q_len, rng.random() < 0.5, rng.random() < 0.6)


# --------------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _kv_rows(g, batch, n, kv_heads, dim):
    """Projected keys / values: unit rows with a per-channel offset and a few wide channels, as a trained projection's."""
    x = torch.randn((batch * n, kv_heads * dim), device="cuda", generator=g)
    off = 0.5 * torch.randn((kv_heads * dim,), device="cuda", generator=g)
    gain = 1.0 + 2.0 * (torch.rand((kv_heads * dim,), device="cuda", generator=g) > 0.97)
    return (x * gain + off).to(BF16)


def _linear_inputs(case, seed):
    """``x`` is a column slice of a wider buffer, as an activation of the network often is; the weights are quantised per channel already."""
    g = _generator(seed)
    m, n, k = case["rows"], case["n"], case["k"]
    pad = (-k) % 8 + 8
    x = torch.randn((m, k + pad), device="cuda", generator=g)
    x = (x * (1.0 + 7.0 * (torch.rand((k + pad,), device="cuda", generator=g) > 0.99)) * torch.exp(0.5 * torch.randn((m, 1), device="cuda", generator=g)))
    w = torch.randn((n, k), device="cuda", generator=g) * (0.5 + torch.rand((n, 1), device="cuda", generator=g)) / math.sqrt(k)
    top = w.abs().amax(1, keepdim=True).clamp(min=TINY).to(F64)
    ws = (top[:, 0] / 127.0).to(F32)
    wq = torch.round(w.to(F64) * 127.0 / top).to(torch.int8)
    w8 = torch.zeros((n, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    w8[:, :k] = wq
    bias = 0.1 * torch.randn((n,), device="cuda", generator=g) if case["bias"] else None
    residual = torch.randn((m, n), device="cuda", generator=g) if case["residual"] else None
    return dict(x=x.to(TYPES[case["x"]])[:, :k], w8=w8, ws=ws, bias=bias, residual=residual)


def _lengths(case, seed):
    """Positions each sequence holds after the call, and how many of them are new: one sequence of a ragged batch holds nothing."""
    rng = random.Random(seed * 7919 + 13)
    b, keys = case["batch"], case["keys"]
    if not case["ragged"]:
        end = [keys] * b
    else:
        end = [rng.randint(1, keys) for _ in range(b)]
        end[rng.randrange(b)] = keys
        if b > 2:
            end[rng.randrange(1, b)] = 0
    new = case.get("new")
    count = None if new is None else [min(new, e) if new > 1 or not case["ragged"] else min(1, e) for e in end]
    return end, count


def _cache_inputs(case, seed):
    g = _generator(seed)
    b, h, d = case["batch"], case["kv_heads"], case["dim"]
    n = case["new"] if case["op"] == "kv4_append" else case["keys"]
    packed = torch.cat([_kv_rows(g, b, n, h, d), _kv_rows(g, b, n, h, d)], dim=1)        # a packed projection: K | V columns
    end, count = _lengths(case, seed)
    s = dict(k=packed[:, :h * d], v=packed[:, h * d:], end=torch.tensor(end, dtype=torch.int32, device="cuda"))
    if count is not None:
        s["count"] = torch.tensor(count, dtype=torch.int32, device="cuda")
    else:
        q = torch.randn((b * case["q_len"], (case["heads"] + 2 * h) * d), device="cuda", generator=g)
        s["q"] = (1.5 * q).to(BF16)[:, :case["heads"] * d]
    return s


def prepare(case, seed):
    if case["op"] == "linear_i8":
        return dict(case=case, **_linear_inputs(case, seed))
    s = dict(case=case, **_cache_inputs(case, seed))
    b, keys, h, d = case["batch"], case["keys"], case["kv_heads"], case["dim"]
    if own:
        from adt_str_amd import kernels as K
        s["cache"] = K.KV4Cache(b, keys, h, d, "cuda")
        if case["op"] == "attn_kv4":
            K.kv4_append(s["cache"], s.pop("k"), s.pop("v"), torch.full((b,), keys, dtype=torch.int32, device="cuda"))
    else:
        if case["op"] == "attn_kv4":
            s["kc"] = _pack4(s.pop("k").reshape(b, keys, h, d))
            s["vc"] = _pack4(s.pop("v").reshape(b, keys, h, d))
        else:                                                   # one position more than the cache has: where rows that are not new go
            s["kc"], s["vc"] = (_pack4(torch.zeros((b, keys + 1, h, d), dtype=BF16, device="cuda")) for _ in range(2))
    return s


# --------------------------------------------------------------------------------------------------------------------- plain forms
def _pack4(x):
    """[..., d] -> (two codes per byte [..., d/2], scale, minimum [..., d/64])."""
    g = x.to(F64).unflatten(-1, (-1, GROUP))                     # 64 bits: many values lie on the border of two codes, or next to it
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 15.0).clamp(min=TINY).to(F32).to(BF16)
    c = torch.round((g - lo[..., None]) / s.to(F64)[..., None]).clamp(0, 15).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), s, lo.to(BF16)


def _unpack4(packed):
    c, s, m = packed
    c = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2).to(F32).unflatten(-1, (-1, GROUP))
    return (c * s.to(F32)[..., None] + m.to(F32)[..., None]).flatten(-2)


def _run_linear(s):
    case = s["case"]
    if own:
        from adt_str_amd import kernels as K
        return K.linear_i8(s["x"], s["w8"], s["ws"], out_dtype=TYPES[case["out"]], bias=s["bias"], act=case["act"], residual=s["residual"])
    x = s["x"].to(F64)                                           # 64 bits for the codes: many values lie on the border of two, or next to it
    top = x.abs().amax(1, keepdim=True).clamp(min=TINY)
    q, scale = torch.round(x * 127.0 / top).to(F32), (top / 127.0).to(F32)
    z = torch.matmul(q, s["w8"][:, :case["k"]].to(F32).t()) * scale * s["ws"]
    if s["bias"] is not None:
        z = z + s["bias"]
    if case["act"] == 1:
        z = 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if s["residual"] is not None:
        z = z + s["residual"]
    return z.to(TYPES[case["out"]])


def _run_append(s):
    case = s["case"]
    b, n, h, d = case["batch"], case["new"], case["kv_heads"], case["dim"]
    if own:
        from adt_str_amd import kernels as K
        K.kv4_append(s["cache"], s["k"], s["v"], s["end"], s["count"])
        return K.kv4_read(s["cache"], s["end"], s["count"], n)
    i = torch.arange(n, device="cuda")
    live = i[None, :] < s["count"][:, None]
    at = torch.where(live, (s["end"] - s["count"])[:, None] + i[None, :], case["keys"]).long()
    rows = torch.arange(b, device="cuda")[:, None]
    out = []
    for name, cache in (("k", s["kc"]), ("v", s["vc"])):
        for whole, part in zip(cache, _pack4(s[name].reshape(b, n, h, d))):
            whole[rows, at] = part
        held = _unpack4([p[rows, at] for p in cache])
        out.append(torch.where(live[:, :, None, None], held, 0.0).to(BF16).reshape(b * n, h * d))
    return out


def _run_attn(s):
    case = s["case"]
    b, keys, h, kh, d, nq = case["batch"], case["keys"], case["heads"], case["kv_heads"], case["dim"], case["q_len"]
    if own:
        from adt_str_amd import kernels as K
        return K.attn_kv4(s["q"], s["cache"], s["end"], heads=h, q_len=nq, scale=1.0 / math.sqrt(d), causal=case["causal"])
    r = h // kh
    q = s["q"].to(F32).reshape(b, nq, kh, r, d).permute(0, 2, 3, 1, 4).reshape(b, kh, r * nq, d)
    k, v = _unpack4(s["kc"]).transpose(1, 2), _unpack4(s["vc"]).transpose(1, 2)
    z = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    sees = s["end"][:, None].expand(b, nq)
    if case["causal"]:
        sees = sees - (nq - 1 - torch.arange(nq, device="cuda"))
    masked = torch.arange(keys, device="cuda") >= sees[:, :, None]                                    # [b, nq, keys]
    z = z.reshape(b, kh, r, nq, keys).masked_fill(masked[:, None, None], -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-3.0e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    o = torch.matmul(p.reshape(b, kh, r * nq, keys), v).reshape(b, kh, r, nq, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b * nq, h * d).to(BF16)


def run(state):
    op = state["case"]["op"]
    return _run_linear(state) if op == "linear_i8" else _run_append(state) if op == "kv4_append" else _run_attn(state)


# --------------------------------------------------------------------------------------------------------------------- the work
def work(case):
    if case["op"] == "linear_i8":
        m, n, k = case["rows"], case["n"], case["k"]
        b = {"bf16": 2, "f32": 4}
        return {"bytes": m * k * b[case["x"]] + n * k + 4 * n + m * n * b[case["out"]] + 4 * n * case["bias"] + 4 * m * n * case["residual"],
                "flops": 2 * m * n * k}
    d, h = case["dim"], case["kv_heads"]
    row = d // 2 + 4 * (d // GROUP)                             # one head's K or V row as it is held
    if case["op"] == "kv4_append":
        rows = 2 * h * sum(_lengths(case, 0)[1])                # K and V: read in bf16, written in 4 bits, read back, written in bf16
        return {"bytes": rows * (2 * d + 2 * row) + 2 * h * case["batch"] * case["new"] * 2 * d, "flops": rows * 6 * d}
    held = sum(_lengths(case, 0)[0])
    io = 2 * 2 * case["batch"] * case["q_len"] * case["heads"] * d
    return {"bytes": io + held * h * 2 * row, "flops": 4 * case["q_len"] * case["heads"] * d * held}


# --------------------------------------------------------------------------------------------------------------------- 64 bits
def _held64(x):
    """What the cache holds of bf16 rows [..., d], in 64 bits: nearest of 16 steps of a bf16 width from the group's minimum."""
    x = x.to(F64).unflatten(-1, (-1, GROUP))
    lo = x.min(dim=-1, keepdim=True).values
    step = torch.maximum((x.max(dim=-1, keepdim=True).values - lo) / 15.0, torch.full_like(lo, TINY)).to(F32).to(BF16).to(F64)
    return (lo + step * torch.round((x - lo) / step).clamp(0, 15)).flatten(-2)


def exact(case, seed):
    if case["op"] == "linear_i8":
        s = _linear_inputs(case, seed)
        x = s["x"].to(F64)
        step = torch.maximum(x.abs().max(dim=1, keepdim=True).values, torch.full((1, 1), TINY, dtype=F64, device=x.device)) / 127.0
        code = x / step
        code = torch.where((code * 2.0 - (code * 2.0).round()).abs() < 1e-10, (code * 2.0).round() / 2.0, code)      # a half is a half
        w = s["w8"][:, :case["k"]].to(F64) * s["ws"].to(F64)[:, None]
        y = (torch.round(code) * step) @ w.t()
        y = y if s["bias"] is None else y + s["bias"].to(F64)
        y = torch.special.ndtr(y) * y if case["act"] == 1 else y
        return y if s["residual"] is None else y + s["residual"].to(F64)
    s = _cache_inputs(case, seed)
    b, h, d = case["batch"], case["kv_heads"], case["dim"]
    end = s["end"].tolist()
    if case["op"] == "kv4_append":
        n, count = case["new"], s["count"].tolist()
        outs = []
        for x in (s["k"], s["v"]):
            held = _held64(x.reshape(b, n, h, d))
            for j, c in enumerate(count):
                held[j, c:] = 0.0
            outs.append(held.reshape(b * n, h * d))
        return outs
    nq, r = case["q_len"], case["heads"] // h
    out = torch.zeros((b, nq, case["heads"], d), dtype=F64, device="cuda")
    q, k, v = s["q"].reshape(b, nq, h, r, d), s["k"].reshape(b, -1, h, d), s["v"].reshape(b, -1, h, d)
    for j, e in enumerate(end):
        if e == 0:
            continue
        kj, vj = _held64(k[j, :e]).permute(1, 0, 2), _held64(v[j, :e]).permute(1, 0, 2)
        for i in range(nq):
            sees = e - (nq - 1 - i) if case["causal"] else e
            if sees > 0:
                z = (q[j, i].to(F64) / math.sqrt(d)) @ kj[:, :sees].transpose(1, 2)
                out[j, i] = (torch.softmax(z, dim=-1) @ vj[:, :sees]).reshape(-1, d)
    return out.reshape(b * nq, -1)

"""The few-bit operators where the framework runs them: ``precision="int8"`` and ``sample(kv_bits=4)``, against the same engine on plain torch
stand-ins of the operators, and the command line's route to them."""
import math

import pytest
import torch

from adt_str_amd import kernels as K
from oracle import adt as o_adt

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
# Two runs that differ in where a bf16 value or an 8-bit code is rounded: each is held to 3e-2 of the exact logits by the bf16 path's tests
LOGIT_TOL = 6e-2


def make_model(precision, enc=2, dec=2, nhead=2, seed=0, dropout=0.0):
    from adt_str_amd.network import ADTModel, ADTModelConfig
    cfg = ADTModelConfig(input_sec=0.5, time_res=0.01, win_length=2048, sample_rate=16000, enc_layers=enc, dec_layers=dec, nhead=nhead, d_query=128,
                         dropout=dropout, tgt_vocab_size=1400, plain=True, n_mels=128)
    model = ADTModel(cfg).set_precision(precision)
    model.load_state_dict(o_adt.seeded_state(model.state_dict(), seed))
    return model.to(DEV).eval()


def make_inputs(b=3, t=9, samples=8000):
    g = torch.Generator()
    g.manual_seed(1)
    src = (0.1 * torch.randn(b, samples, generator=g)).to(DEV)
    tok = torch.randint(4, 1400, (b, t + 1), generator=g).to(DEV)
    tok[:, 0] = 2
    pad = (torch.arange(t)[None, :] >= torch.tensor([t, t - 4, 1])[:b, None]).to(DEV)
    return src, tok, pad


# --------------------------------------------------------------------------------------------------- stand-ins
def plain_quant(x):
    x64 = x.to(F64)
    top = x64.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
    q = torch.zeros((x.shape[0], (x.shape[1] + 15) // 16 * 16), dtype=torch.int8, device=x.device)
    q[:, :x.shape[1]] = torch.round(x64 * 127.0 / top).to(torch.int8)
    return q, (top[:, 0] / 127.0).to(F32)


def plain_gemm(a, a_scale, b, b_scale, *, out=None, out_dtype=BF16, bias=None, residual=None, res_row_mod=0, act=0, aux_bf16_out=None):
    z = torch.matmul(a.to(F64), b.to(F64).t()) * a_scale.to(F64)[:, None] * b_scale.to(F64)
    z = z if bias is None else z + bias.to(F64)
    z = 0.5 * z * torch.erfc(-z / math.sqrt(2.0)) if act == 1 else z
    if residual is not None:
        z = z + (residual[torch.arange(z.shape[0], device=z.device) % res_row_mod] if res_row_mod else residual).to(F64)
    if aux_bf16_out is not None:
        aux_bf16_out.copy_(z.to(F32).to(BF16))
    z = z.to(F32).to(out_dtype)
    return z if out is None else out.copy_(z)


class PlainCache:
    def __init__(self, batch, capacity, kv_heads, head_dim, device="cuda"):
        self.batch, self.capacity, self.kv_heads, self.head_dim = batch, capacity, kv_heads, head_dim
        self.k, self.v = (torch.zeros((batch, capacity, kv_heads, head_dim), dtype=F64, device=device) for _ in range(2))


def plain_held(x):
    g = x.to(F64).unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15.0).clamp(min=2.0 ** -100).to(F32).to(BF16).to(F64)
    return (lo + s * torch.round((g - lo) / s).clamp(max=15)).flatten(-2)


def plain_append(cache, k, v, end=None, count=None):
    n = k.shape[0] // cache.batch
    for b in range(cache.batch):
        e = cache.capacity if end is None else int(end[b])
        for mine, rows in ((cache.k, k), (cache.v, v)):
            mine[b, e - n:e] = plain_held(rows[b * n:(b + 1) * n].reshape(n, cache.kv_heads, cache.head_dim))


def plain_attn(q, cache, key_len=None, *, heads, scale, q_len=1, causal=False, out=None, want_lse=False):
    o = torch.zeros((cache.batch, heads, cache.head_dim), dtype=F64, device=q.device)
    for b in range(cache.batch):
        n = cache.capacity if key_len is None else int(key_len[b])
        z = torch.matmul(cache.k[b, :n].permute(1, 0, 2), q[b].to(F64).reshape(heads, cache.head_dim, 1))[..., 0] * scale
        o[b] = torch.matmul(torch.softmax(z, -1)[:, None, :], cache.v[b, :n].permute(1, 0, 2))[:, 0]
    return o.reshape(cache.batch, -1).to(BF16)


def use_stand_ins(mp):
    for name, fn in (("quant_rows_i8", plain_quant), ("gemm_i8", plain_gemm), ("KV4Cache", PlainCache), ("kv4_append", plain_append), ("attn_kv4", plain_attn)):
        mp.setattr(K, name, fn)


# --------------------------------------------------------------------------------------------------- precision "int8"
@torch.no_grad()
def int8_logits(seed=0):
    model = make_model("int8", seed=seed)
    src, tok, pad = make_inputs()
    return model.engine.loss_and_grads(src, tok[:, :-1], pad, tok[:, 1:], want_grads=False, return_logits=True)


def test_int8_network_equals_its_plain_form_and_follows_fp32(monkeypatch):
    got = int8_logits()
    with monkeypatch.context() as mp:
        use_stand_ins(mp)
        want = int8_logits()
    assert float((got["logits"] - want["logits"]).abs().max()) <= LOGIT_TOL
    assert abs(float(got["loss"]) - float(want["loss"])) <= LOGIT_TOL
    # against fp32: an 8-bit code of a row of hundreds of numbers is off by 1 % of their root mean square (step max / 127, max about 4 of
    # it), a product of two by 1.3 %, the sixteen products of the residual stream by four times that at most; twice this is the bound
    model = make_model("fp32")
    src, tok, pad = make_inputs()
    ref = model.engine.loss_and_grads(src, tok[:, :-1], pad, tok[:, 1:], want_grads=False, return_logits=True)["logits"]
    assert float((got["logits"] - ref).norm() / ref.norm()) <= 0.1


def test_int8_weights_follow_the_parameters_and_training_is_refused():
    model = make_model("int8")
    src, tok, pad = make_inputs()
    with torch.no_grad():
        a = model(src, tok[:, :-1], None, pad, tok[:, 1:])
        model.load_state_dict(o_adt.seeded_state(model.state_dict(), 5))
        b = model(src, tok[:, :-1], None, pad, tok[:, 1:])
    fresh = make_model("int8", seed=5)
    with torch.no_grad():
        c = fresh(src, tok[:, :-1], None, pad, tok[:, 1:])
    assert float(a) != float(b) and float(b) == float(c)
    with pytest.raises(RuntimeError, match="inference"):
        model(src, tok[:, :-1], None, pad, tok[:, 1:])
    dropped = make_model("int8", dropout=0.1).train()
    with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
        dropped(src, tok[:, :-1], None, pad, tok[:, 1:])


# --------------------------------------------------------------------------------------------------- the cached decode
def forced_logits(mp, precision, kv_bits, steps, use_graph=False):
    """Logits of every step of the cached decode along fixed tokens: the tail of the step is replaced by one that writes them."""
    model = make_model(precision)
    src, _, _ = make_inputs()
    g = torch.Generator()
    g.manual_seed(4)
    table = torch.randint(4, 1400, (src.shape[0], steps + 1), generator=g).to(DEV)
    seen = []

    def tail(logits, finished, gen, t, tok, klen, done_at, end_token):
        seen.append(logits.clone())
        tok.copy_(table.index_select(1, t))
        klen.add_(1)
        t.add_(1)

    with mp.context() as m:
        m.setattr(K, "greedy_step", tail)
        mem16, B, S = model.engine.encode(src)
        model.engine.greedy_decode_cached(mem16, B, S, steps + 1, 2, 3, use_graph=use_graph, kv_bits=kv_bits)
    return torch.stack(seen)


@pytest.mark.parametrize("precision", ["bf16", "int8"])
def test_decode_over_4_bit_caches_equals_its_plain_form(monkeypatch, precision):
    got = forced_logits(monkeypatch, precision, 4, 70)                       # past two tiles of 32 positions
    with monkeypatch.context() as mp:
        use_stand_ins(mp)
        want = forced_logits(monkeypatch, precision, 4, 70)
    assert got.shape == want.shape == (70, 3, 1400)
    # against bf16 caches: a 4-bit value is off by 9 % of a normal row's deviation (64 numbers span 4.8 of it: a step is 0.32, uniformly off by half
    # of it at most); an attention's output by no more than that, and it is one of the summands of the residual stream: 0.15 bounds the logits
    wide = forced_logits(monkeypatch, precision, 16, 70)
    assert float((got - wide).norm() / wide.norm()) <= 0.15
    # Two runs that round elsewhere put some codes on the other side of a border, a whole step away.  bf16: rows differ by 2^-8 of 0.8 deviations on
    # average, 1 % of a step: sqrt(0.01) 0.32 = 3.2 % of the deviation, where the quantisation itself is 9 %: 0.15 3.2 / 9 = 0.055.  int8: of the 8-bit
    # codes behind such differences (step 3 % of the deviation) a tenth moves, sqrt(0.1) 3 % = 1 % in every product, 2.5 % of the 4-bit
    # codes: sqrt(0.025) 0.32 = 5 %: 0.085.
    assert float((got - want).norm() / want.norm()) <= (0.055 if precision == "bf16" else 0.085)


@pytest.mark.parametrize("precision", ["bf16", "int8"])
def test_every_few_bit_call_of_a_decode_equals_its_plain_form_on_the_same_inputs(monkeypatch, precision):
    """Call by call along one decode, so that no rounding difference is carried: codes and scales equal, bf16 results within a rounding each
    (2 2^-8) of the largest magnitude that meets in them."""
    plain, calls = {}, {"quant_rows_i8": 0, "gemm_i8": 0, "kv4_append": 0, "attn_kv4": 0}
    real = {n: getattr(K, n) for n in ("quant_rows_i8", "gemm_i8", "KV4Cache", "kv4_append", "attn_kv4")}

    def cache(*a, **kw):
        c = real["KV4Cache"](*a, **kw)
        plain[id(c)] = (c, PlainCache(*a, **kw))
        return c

    def quant(x):
        got, want = real["quant_rows_i8"](x), plain_quant(x)
        assert x.dtype == F32 or torch.equal(got[0], want[0])
        assert torch.equal(got[1], want[1])
        calls["quant_rows_i8"] += 1
        return got

    def gemm(a, sa, b, sb, **kw):
        got, want = real["gemm_i8"](a, sa, b, sb, **kw), plain_gemm(a, sa, b, sb, **kw)
        assert float((got - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
        calls["gemm_i8"] += 1
        return got

    def append(c, k, v, end=None, count=None):
        real["kv4_append"](c, k, v, end, count)
        plain_append(plain[id(c)][1], k, v, end, count)
        calls["kv4_append"] += 1

    def attn(q, c, key_len=None, **kw):
        got, want = real["attn_kv4"](q, c, key_len, **kw), plain_attn(q, plain[id(c)][1], key_len, **kw)
        assert float((got - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
        calls["attn_kv4"] += 1
        return got

    with monkeypatch.context() as mp:
        for name, fn in (("KV4Cache", cache), ("quant_rows_i8", quant), ("gemm_i8", gemm), ("kv4_append", append), ("attn_kv4", attn)):
            mp.setattr(K, name, fn)
        forced_logits(monkeypatch, precision, 4, 35)
    assert calls["attn_kv4"] == 2 * 2 * 35 and calls["kv4_append"] == 2 * 35 + 2
    assert (calls["gemm_i8"] > 0) == (precision == "int8") and (calls["quant_rows_i8"] > 0) == (precision == "int8")


@pytest.mark.parametrize("precision", ["bf16", "int8"])
def test_sample_over_4_bit_caches_replays_as_a_graph(precision):
    model = make_model(precision, seed=5)
    src, _, _ = make_inputs()
    eng = model.engine
    mem16, B, S = eng.encode(src)
    runs = [eng.greedy_decode_cached(mem16, B, S, 60, 2, 3, use_graph=g, kv_bits=4) for g in (False, True, True)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    assert torch.equal(model.sample(src, max_length=60, kv_bits=4), runs[0])
    assert runs[0][:, 0].eq(2).all() and 2 <= runs[0].shape[1] <= 60


def test_sample_refuses_what_it_cannot_hold():
    src, _, _ = make_inputs()
    model = make_model("bf16", 1, 1)
    with pytest.raises(ValueError):
        model.sample(src, max_length=4, kv_bits=8)
    with pytest.raises(ValueError):
        model.sample(src, max_length=4, kv_bits=4, use_cache=False)
    with pytest.raises(ValueError):
        make_model("fp32", 1, 1).sample(src, max_length=4, kv_bits=4)
    with pytest.raises(ValueError):
        model.set_precision("int4")


def test_transcribe_takes_the_few_bit_options():
    import inference
    a = inference._parser().parse_args(["x.wav", "c.yaml", "--precision", "int8", "--kv-bits", "4"])
    assert a.precision == "int8" and a.kv_bits == 4
    model = make_model("int8", 1, 1)
    cfg = dict(shared=dict(input_sec=0.5, sample_rate=16000), inference=dict(max_length=40))
    wav = 0.1 * torch.randn(20000, device=DEV)
    ids = []
    inference.transcribe(model, cfg, wav, 2, ids, kv_bits=4)
    chunks = inference._chunk_audio(wav, 8000)
    assert len(ids) == 3
    want = [r.tolist() for i in range(0, 3, 2) for r in model.sample(chunks[i:i + 2], max_length=40, kv_bits=4).cpu()]
    assert ids == want

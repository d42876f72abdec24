"""``precision="int8"`` where the network runs it, with every ``linear_i8`` call in view: call by call against the operator's definition in 64 bits, and the
whole network against itself on plain torch products."""
import pytest
import torch

from adt_str_amd import kernels as K
from tests.test_few_bits_path_gpu import forced_logits, int8_logits, make_inputs, make_model, plain_gemm, plain_quant, use_stand_ins
from tests.test_few_bits_products_gpu import check, expected

pytestmark = pytest.mark.gpu
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


def plain_linear(x, w8, w_scale, **kw):
    return plain_gemm(*plain_quant(x), w8, w_scale, **kw)


def watched(calls):
    """``linear_i8`` that checks each result (and bf16 copy) against 64 bits on the call's own inputs."""
    real = K.linear_i8

    def linear(x, w8, w_scale, *, out=None, out_dtype=BF16, bias=None, residual=None, res_row_mod=0, act=0, aux_bf16_out=None):
        codes, scale = plain_quant(x)
        acc = torch.matmul(codes.to(F64), w8.to(F64).t().contiguous())
        r = residual
        if r is not None and res_row_mod:
            r = r[torch.arange(x.shape[0], device=x.device) % res_row_mod]
        z, err = expected(acc, scale, w_scale, bias, act, r)
        y = real(x, w8, w_scale, out=out, out_dtype=out_dtype, bias=bias, residual=residual, res_row_mod=res_row_mod, act=act, aux_bf16_out=aux_bf16_out)
        check(y, z, err)
        assert aux_bf16_out is None or torch.equal(aux_bf16_out, y.to(BF16))
        calls.append((tuple(x.shape), w8.shape[0], act, residual is not None, res_row_mod, aux_bf16_out is not None))
        return y

    return linear


def test_every_linear_call_of_the_network_equals_its_definition(monkeypatch):
    calls = []
    with monkeypatch.context() as mp:
        mp.setattr(K, "linear_i8", watched(calls))
        int8_logits()
    # encoder: its input layer and four products a layer; decoder: six a layer (the memory's K and V are quantised once and multiplied)
    assert len(calls) == 1 + 2 * 4 + 2 * 6
    assert any(c[4] > 0 and c[5] for c in calls)                              # + positional rows, with the bf16 copy
    assert sum(c[2] == 1 for c in calls) == 4 and sum(c[3] for c in calls) == 1 + 2 * 2 + 2 * 3


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_every_linear_call_of_a_decode_equals_its_definition(monkeypatch, kv_bits):
    calls = []
    with monkeypatch.context() as mp:
        mp.setattr(K, "linear_i8", watched(calls))
        forced_logits(monkeypatch, "int8", kv_bits, 12)
    assert len(calls) == 1 + 2 * 4 + 12 * 2 * 6


@torch.no_grad()
def test_int8_network_on_plain_products(monkeypatch):
    got = int8_logits()
    with monkeypatch.context() as mp:
        use_stand_ins(mp)
        mp.setattr(K, "linear_i8", plain_linear)
        want = int8_logits()
    # A rounding that falls the other way moves some codes by one.  At worst the two runs' codes are as good as independent: a step is 3 % of a row's root
    # mean square (max / 127, the maximum about four of it), uniformly off by half of it at most 0.9 %, two runs 1.25 %; the sixteen products that add up in
    # the residual streams make that 5 % of the logits
    assert float((got["logits"] - want["logits"]).norm() / want["logits"].norm()) <= 0.05
    assert abs(float(got["loss"]) - float(want["loss"])) <= 0.05 * float(want["logits"].abs().max())


def test_int8_decode_replays_with_the_bits_of_its_eager_steps_over_both_caches():
    model = make_model("int8", seed=3)
    src, _, _ = make_inputs()
    mem16, B, S = model.engine.encode(src)
    for kv_bits in (16, 4):
        eager, replayed = (model.engine.greedy_decode_cached(mem16, B, S, 40, 2, -1, use_graph=g, kv_bits=kv_bits) for g in (False, True))
        assert eager.shape == (B, 40) and torch.equal(eager, replayed)


@torch.no_grad()
@pytest.mark.parametrize("precision,kv_bits", [("int8", 16), ("int8", 4), ("bf16", 4)])
def test_cached_decode_follows_the_decoder_over_the_whole_prefix(monkeypatch, precision, kv_bits):
    """``use_cache=False`` runs the decoder over the prefix at every step: its last position is what the cached step computes."""
    steps = 40
    got = forced_logits(monkeypatch, precision, kv_bits, steps)
    model = make_model(precision)
    src, _, _ = make_inputs()
    g = torch.Generator()
    g.manual_seed(4)
    table = torch.randint(4, 1400, (src.shape[0], steps + 1), generator=g).cuda()
    prefix = torch.cat([torch.full((src.shape[0], 1), 2, device="cuda"), table[:, :steps - 1]], 1)
    mem16, B, S = model.engine.encode(src)
    want = model.engine.decode_logits(prefix, mem16, B, S).transpose(0, 1)
    # int8: the bound of two runs whose codes are as good as independent (above); 4 bits: that of the quantisation itself, 0.15 (9 % of a normal row's
    # deviation in a value, and no more in an attention's output, one of the summands of the residual stream)
    assert float((got - want).norm() / want.norm()) <= (0.05 if kv_bits == 16 else 0.15)
    assert model.sample(src, max_length=6, use_cache=False).shape[0] == B

"""Few-bit serving operators (K16, K17) at the limits of what their documentation allows, each against its definition in 64 bits."""
import math

import pytest
import torch

from adt_str_amd import kernels as K
from tests.test_few_bits_gpu import attn_ref, check_attn, check_held, gen, kv_rows

pytestmark = pytest.mark.gpu
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


# --------------------------------------------------------------------------------------------------- quantiser
def nearest_codes(x):
    """The integers nearest to 127 x / max|x|, ties to even, decided exactly: 254 |x| and an odd multiple of the maximum below 255 of it have 32 bits."""
    x = x.to(F64)
    top = x.abs().amax(1, keepdim=True)
    k = torch.floor(127.0 * x.abs() / top)
    past = 254.0 * x.abs() - (2.0 * k + 1.0) * top
    return torch.sign(x) * torch.where((past > 0) | ((past == 0) & (k % 2 == 1)), k + 1.0, k)


def rows_beside_borders(rows, seed):
    """fp32 rows whose values are the nearest floats to half-integer codes, and their neighbours, of both signs, behind the row's maximum."""
    g = gen(seed)
    top = (1.0 + torch.rand(rows, 1, generator=g)) * torch.exp(8.0 * torch.randn(rows, 1, generator=g))
    half = ((torch.arange(127, dtype=F64) + 0.5)[None] * top.to(F64) / 127.0).to(F32)
    up, down = torch.nextafter(half, torch.full_like(half, math.inf)), torch.nextafter(half, torch.zeros_like(half))
    return torch.cat([top, half, -half, up, -up, down, -down], 1)


@pytest.mark.parametrize("copies", [1, 2, 4, 12])                             # 763 to 9156 columns: a row in one wave, in a workgroup, read twice
def test_quant_rows_fp32_codes_beside_borders(copies):
    x = rows_beside_borders(300, copies).repeat(1, copies)
    x[0, :5] = torch.tensor([4.0, 2.0, -2.0, 2.0 ** -140, 0.0])               # 63.5 itself, and next to nothing
    q, _ = K.quant_rows_i8(x.cuda())
    assert torch.equal(q[:, :x.shape[1]].cpu().to(F64), nearest_codes(x))
    assert torch.equal(q[0, :5].cpu()[torch.tensor([3, 4])], torch.zeros(2, dtype=torch.int8))


def test_linear_i8_fp32_codes_beside_borders():
    """The launch that quantises its rows itself makes the same codes."""
    x = rows_beside_borders(40, 9).cuda()
    k = x.shape[1]
    w8, ws = K.quant_rows_i8(torch.randn(48, k, generator=gen(1)).cuda())
    q = torch.zeros((40, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    q[:, :k] = nearest_codes(x).to(torch.int8)
    assert torch.equal(K.linear_i8(x, w8, ws, out_dtype=F32), K.gemm_i8(q, (x.abs().amax(1).to(F64) / 127.0).to(F32), w8, ws, out_dtype=F32))


# --------------------------------------------------------------------------------------------------- products
def test_products_of_2_to_the_30_rows_and_of_as_many_channels():
    """2^23 tiles, a column or a row of them; 16 GB of operands."""
    n = 1 << 30
    at = torch.tensor([0, 1, 127, 128, 65535, n // 2, n - 129, n - 128, n - 2, n - 1], device="cuda")
    many, scale = torch.zeros((n, 16), dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
    many[at, 3] = torch.arange(1, 11, dtype=torch.int8, device="cuda")
    scale[at] = 0.5
    one, s1 = torch.full((1, 16), 2, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda")
    for out in (K.gemm_i8(one, s1, many, scale)[0], K.gemm_i8(many, scale, one, s1)[:, 0]):
        assert out[at].tolist() == [float(i) for i in range(1, 11)]
        assert int((out != 0).sum()) == 10
        del out


# --------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_len,cap,lens", [
    (2, 2, 4, 100, [103, 100, 101, 99, 2 ** 31 - 1, -3]),                     # the newest rows lie behind the cache; a length no cache has
    (6, 2, 9, 33, [40, 41, 42, 33, 5]), (1, 1, 40, 64, [70, 64, 103, 104]),   # several blocks of rows, some of which see all, some less
    (4, 1, 3, 3000, [3001, 3002, 2999])])                                     # cut into spans
@pytest.mark.parametrize("causal", [True, False])
def test_attn_kv4_lengths_past_the_capacity(dim, heads, kv_heads, q_len, cap, lens, causal):
    """``key_len`` is the sequence's length, whatever part of it the cache holds: causal query i sees the first min(capacity, key_len - (q_len - 1 - i))
    positions."""
    batch = len(lens)
    k, v = kv_rows(batch * cap, kv_heads, dim, cap + q_len)
    c = K.KV4Cache(batch, cap, kv_heads, dim)
    K.kv4_append(c, k, v)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = (1.5 * torch.randn(batch * q_len, heads * dim, generator=gen(7))).to(BF16).cuda()
    scale = 1.0 / math.sqrt(dim)
    out, lse = K.attn_kv4(q, c, n, heads=heads, scale=scale, q_len=q_len, causal=causal, want_lse=True)
    check_attn(out, lse, q, k.reshape(batch, cap, -1), v.reshape(batch, cap, -1), heads, kv_heads, dim, batch, q_len, lens, scale, causal)


def test_append_and_causal_attention_of_a_sequence_that_outgrows_its_cache():
    """The chunk's rows that do not fit are left out by the append and seen by nobody; its queries see what their positions say."""
    heads, dim, cap, q_len, end = 2, 128, 50, 6, 53
    k, v = kv_rows(end, heads, dim, 4)
    c = K.KV4Cache(1, cap, heads, dim)
    at = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    K.kv4_append(c, k[:end - q_len], v[:end - q_len], at(end - q_len))
    K.kv4_append(c, k[end - q_len:], v[end - q_len:], at(end))
    held = K.kv4_read(c, out_dtype=torch.float32)
    check_held(held[0], k[:cap], heads, dim)
    check_held(held[1], v[:cap], heads, dim)
    q = torch.randn(q_len, heads * dim, generator=gen(9)).to(BF16).cuda()
    out, lse = K.attn_kv4(q, c, at(end), heads=heads, scale=dim ** -0.5, q_len=q_len, causal=True, want_lse=True)
    check_attn(out, lse, q, k[None, :cap], v[None, :cap], heads, heads, dim, 1, q_len, [end], dim ** -0.5, True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 20.0, -20.0])
@pytest.mark.parametrize("heads,kv_heads,q_len,cap,lens", [(3, 3, 1, 90, [90, 33, 0]), (6, 2, 5, 200, [200, 3, 64]), (2, 1, 1, 2500, [2500, 1, 999])])
def test_attn_kv4_scales_of_any_sign_and_size(dim, scale, heads, kv_heads, q_len, cap, lens):
    batch = len(lens)
    k, v = kv_rows(batch * cap, kv_heads, dim, cap)
    c = K.KV4Cache(batch, cap, kv_heads, dim)
    K.kv4_append(c, k, v)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(batch * q_len, heads * dim, generator=gen(2)).to(BF16).cuda()
    out, lse = K.attn_kv4(q, c, n, heads=heads, scale=scale, q_len=q_len, causal=True, want_lse=True)
    q_ref = -q if scale < 0 else q                                            # exact: a negative scale is the negative query's
    o, l, mag = attn_ref(q_ref, k.reshape(batch, cap, -1), v.reshape(batch, cap, -1), heads, kv_heads, dim, batch, q_len, lens, abs(scale), True)
    assert ((out.to(F64) - o).abs() <= 2.0 ** -8 * (o.abs() + mag) + mag).all()
    none = l == -math.inf
    assert torch.equal(lse == -math.inf, none)
    # the score's own error (8 roundings of about 31 steps of 0.4 and 1.5 against each of dim unit query values), times the scale, and two of the log-sum's
    dz = 8 * 2.0 ** -24 * 14.0 * dim * abs(scale)
    assert ((lse.to(F64) - l)[~none].abs() <= dz + 2.0 ** -23 * l[~none].abs() + 1e-6).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap", [70, 3000])                                   # one span, several
def test_attn_kv4_query_rows_without_numbers_stay_alone(dim, cap):
    heads, kv_heads, q_len = 4, 2, 6
    k, v = kv_rows(2 * cap, kv_heads, dim, 8)
    c = K.KV4Cache(2, cap, kv_heads, dim)
    K.kv4_append(c, k, v)
    q = torch.randn(2 * q_len, heads * dim, generator=gen(3)).to(BF16).cuda()
    clean = K.attn_kv4(q, c, heads=heads, scale=0.1, q_len=q_len).reshape(2 * q_len, heads, dim)
    q[3, 2 * dim + 5] = math.nan                                              # row 3, head 2
    q[7, 1] = math.inf                                                        # row 7, head 0
    out = K.attn_kv4(q, c, heads=heads, scale=0.1, q_len=q_len).reshape(2 * q_len, heads, dim)
    bad = torch.zeros(2 * q_len, heads, dtype=torch.bool, device="cuda")
    bad[3, 2] = bad[7, 0] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("dim", [64, 128])
def test_kv4_append_rows_that_begin_anywhere_and_more_of_them_than_positions(dim):
    batch, heads, cap, n = 2, 3, 37, 90
    width = heads * dim
    g = gen(11)
    kb, vb = torch.randn(batch * n, width + 3, generator=g).to(BF16).cuda(), torch.randn(batch * n, width + 16, generator=g).to(BF16).cuda()
    k, v = kb[:, 1:1 + width], vb[:, 8:8 + width]                             # keys two bytes at a time, values sixteen
    for a, b in ((k, v), (v, k)):
        c = K.KV4Cache(batch, cap, heads, dim)
        c.data.fill_(0xFF)
        K.kv4_append(c, a, b)                                                 # n rows for cap positions: the last ones
        held = K.kv4_read(c, out_dtype=F32)
        for got, src in zip(held, (a, b)):
            check_held(got, src.reshape(batch, n, width)[:, n - cap:].reshape(batch * cap, width), heads, dim)
        end = torch.tensor([60, 5], dtype=torch.int32, device="cuda")         # sequence 0: rows 30 .. 66 of 90 fit, 1: its last five
        c.data.fill_(0xFF)
        K.kv4_append(c, a, b, end)
        back = K.kv4_read(c, end, None, n, out_dtype=F32)
        for got, src in zip(back, (a, b)):
            got, src = got.reshape(batch, n, width), src.reshape(batch, n, width)
            check_held(got[0, 30:67], src[0, 30:67], heads, dim)
            check_held(got[1, 85:], src[1, 85:], heads, dim)
            assert not got[0, :30].any() and not got[0, 67:].any() and not got[1, :85].any()

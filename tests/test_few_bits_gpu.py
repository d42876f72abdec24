"""Serving in few bits on the GPU: the row quantiser and 8-bit-integer products (K16), the 4-bit K/V cache and the attention over it (K17),
each against its definition in 64 bits.  Tolerances count roundings: u = 2^-24 per fp32 operation, 2^-8 (relative) for a bf16 result."""
import math

import pytest
import torch

from adt_str_amd import kernels as K
from adt_str_amd._ffi import AdtError

pytestmark = pytest.mark.gpu
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
U = 2.0 ** -24
TINY = 2.0 ** -100


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# --------------------------------------------------------------------------------------------------- quantiser
def quant_ref(x):
    x = x.to(F64)
    top = x.abs().amax(1, keepdim=True).clamp(min=TINY)
    return x * 127.0 / top, (top[:, 0] / 127.0).to(F32)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 16), (64, 768), (7, 1001), (130, 520), (2, 5000), (33, 64), (9, 8192), (3, 2049), (70, 4096), (2, 4099), (5, 20000)])
def test_quant_rows_codes_are_the_nearest_integers(dtype, m, k):
    x = (torch.randn(m, k + 5, generator=gen(m * 1000 + k)) * torch.exp(torch.randn(m, 1, generator=gen(k)))).to(dtype).cuda()[:, 2:2 + k]
    q, s = K.quant_rows_i8(x)
    code, scale = quant_ref(x)
    assert q.shape == (m, (k + 15) // 16 * 16) and q.dtype == torch.int8
    assert torch.equal(s, scale)
    assert not q[:, k:].any()
    if dtype == BF16:
        assert torch.equal(q[:, :k].to(F64), torch.round(code))               # bf16 ratios: the quotient is decided exactly, ties to even
    else:
        assert ((q[:, :k].to(F64) - code).abs() <= 0.5 + 2.0 ** -17).all()    # an fp32 quotient of up to 127 is off by half of 2^-17


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quant_rows_ties_extremes_and_rows_without_numbers(dtype):
    big = torch.finfo(dtype).max
    rows = torch.zeros(12, 20)
    rows[0, :4] = torch.tensor([2.0, 1.0, -1.0, 0.5])                         # 127, 63.5 -> 64, -64, 31.75
    rows[1, :5] = torch.tensor([254.0, 1.0, 3.0, 5.0, -7.0])                  # halves: 0.5 -> 0, 1.5 -> 2, 2.5 -> 2, -3.5 -> -4
    rows[2, :3] = torch.tensor([big, -big, big / 2])
    rows[3, :2] = torch.tensor([2.0 ** -120, -2.0 ** -126])                   # below the smallest magnitude: codes 0
    rows[4, 0] = 2.0 ** -99
    rows[5, 3] = math.inf
    rows[6, 19] = math.nan
    rows[7, :2] = torch.tensor([-math.inf, math.nan])
    rows[9, 7] = -3.0
    x = rows.to(dtype).cuda()
    q, s = K.quant_rows_i8(x)
    good = [0, 1, 2, 3, 4, 8, 9, 10, 11]
    code, scale = quant_ref(x[good])
    assert torch.equal(q[good, :20].to(F64), torch.round(code)) and torch.equal(s[good], scale)
    assert q[0, :4].tolist() == [127, 64, -64, 32] and q[1, :5].tolist() == [127, 0, 2, 2, -4] and q[2, :3].tolist() == [127, -127, 64]
    assert torch.isnan(s[[5, 6, 7]]).all() and not q[[5, 6, 7]].any()
    assert q[8].abs().max() == 0 and float(s[8]) > 0


def test_quant_rows_more_rows_than_one_grid_holds():
    m = (1 << 27) + 3
    x = torch.full((m, 1), 2.0, dtype=BF16, device="cuda")
    x[[0, (1 << 27) - 1, 1 << 27, m - 1], 0] = torch.tensor([-1.0, 4.0, -8.0, 0.0], dtype=BF16, device="cuda")
    q, s = K.quant_rows_i8(x)
    picked = [0, 1, (1 << 27) - 1, 1 << 27, m - 2, m - 1]
    assert q[picked, 0].tolist() == [-127, 127, 127, -127, 127, 0]
    assert int((q[:, 0] == 127).sum()) == m - 3 and not q[picked, 1:].any()
    assert torch.equal(s[picked[:5]], torch.tensor([1.0, 2.0, 4.0, 8.0, 2.0], device="cuda") / 127)


# --------------------------------------------------------------------------------------------------- products
def gelu64(z):
    return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))


def check_product(a, sa, b, sb, out, bias=None, residual=None, act=0, rows=None):
    acc = torch.matmul(a.to(F64), b.to(F64).t())
    prod = acc * sa.to(F64)[:, None] * sb.to(F64)
    z = prod if bias is None else prod + bias.to(F64)
    # float(acc), two scales, the bias: four roundings of at most the magnitudes that meet in them
    err = 4 * U * (prod.abs() + (0 if bias is None else bias.to(F64).abs()))
    if act == 1:
        # erf is approximated to 1.5e-7; its polynomial, reciprocal and exponential are about ten fp32 operations; |gelu'| <= 1.13
        y = gelu64(z)
        err = 1.13 * err + z.abs() * (0.75e-7 + 10 * U)
        z = y
    elif act == 2:
        z = z.clamp(min=0)
    if residual is not None:
        z = z + residual.to(F64)
        err = err + U * z.abs()
    if out.dtype == BF16:
        err = err + 2.0 ** -8 * (z.abs() + err)
    d = (out.to(F64) - z).abs()
    assert (d <= err + 1e-37).all(), float((d - err).max())


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 2304, 768), (3, 5, 32), (64, 1400, 768), (65, 129, 144), (127, 128, 128), (128, 257, 1008), (200, 70, 4096),
                                   (1000, 768, 768), (8192, 768, 256), (513, 1001, 1536), (16, 768, 2048), (4097, 2304, 784), (700, 5000, 80)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_gemm_i8_matches_integer_products(m, n, k, out):
    g = gen(m + 3 * n + 7 * k)
    a = torch.randint(-127, 128, (m, k + 16), generator=g, dtype=torch.int8).cuda()[:, :k]
    b = torch.randint(-127, 128, (n, k + 32), generator=g, dtype=torch.int8).cuda()[:, 16:16 + k]
    sa, sb = (0.5 + torch.rand(m, generator=g)).cuda() / 127, (0.5 + torch.rand(n, generator=g)).cuda() / 127
    bias, res = torch.randn(n, generator=g).cuda(), torch.randn(m, n, generator=g).cuda()
    check_product(a, sa, b, sb, K.gemm_i8(a, sa, b, sb, out_dtype=out), None)
    check_product(a, sa, b, sb, K.gemm_i8(a, sa, b, sb, out_dtype=out, bias=bias, residual=res), bias, res)


@pytest.mark.parametrize("m,n,k", [(2, 96, 64), (64, 768, 768), (300, 1000, 256), (2100, 1536, 768)])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("act", [1, 2])
def test_gemm_i8_activations(m, n, k, out, act):
    g = gen(m + n + k + act)
    a, b = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((m, k), (n, k)))
    sa, sb = (0.5 + torch.rand(m, generator=g)).cuda() / 127, (0.5 + torch.rand(n, generator=g)).cuda() / (127 * math.sqrt(k) / 3)
    bias = torch.randn(n, generator=g).cuda()
    check_product(a, sa, b, sb, K.gemm_i8(a, sa, b, sb, out_dtype=out, bias=bias, act=act), bias, act=act)


@pytest.mark.parametrize("m", [1, 50, 260, 5000])
def test_gemm_i8_views_periodic_residual_and_bf16_copy(m):
    n, k = 264, 192
    g = gen(m)
    a, b = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((m, k), (n, k)))
    sa, sb = torch.rand(m, generator=g).cuda() / 100, torch.rand(n, generator=g).cuda() / 100
    table = torch.randn(37, n, generator=g).cuda()
    wide, wide16 = torch.full((m, n + 24), 7.0, device="cuda"), torch.full((m, n + 24), 7.0, device="cuda", dtype=BF16)
    res = table[torch.arange(m, device="cuda") % 37]
    K.gemm_i8(a, sa, b, sb, out=wide[:, 8:8 + n], residual=table, res_row_mod=37, aux_bf16_out=wide16[:, 8:8 + n])
    check_product(a, sa, b, sb, wide[:, 8:8 + n], residual=res)
    assert torch.equal(wide16[:, 8:8 + n], wide[:, 8:8 + n].to(BF16))
    for t in (wide, wide16):
        assert (t[:, :8] == 7).all() and (t[:, 8 + n:] == 7).all()
    for lo, w in ((1, n), (3, n - 5)):                                        # rows that are not 16-byte aligned, a width that is no multiple of 8
        w32 = torch.full((m, n + 24), 7.0, device="cuda")
        K.gemm_i8(a, sa, b[:w], sb[:w].contiguous(), out=w32[:, lo:lo + w])
        check_product(a, sa, b[:w], sb[:w], w32[:, lo:lo + w])
        assert (w32[:, :lo] == 7).all() and (w32[:, lo + w:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(20, 1001, 80), (40, 301, 2000), (300, 1003, 400), (1282, 2263, 144), (4400, 2301, 640), (4400, 2304, 640), (1, 1, 16)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_gemm_i8_odd_widths_activation_residual_and_what_lies_around(m, n, k, out):
    """Every tile size at widths that no 16-byte piece divides, rows that begin anywhere, and the whole epilogue at once."""
    g = gen(m + n + k)
    a, b = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((m, k), (n, k)))
    sa, sb = (0.5 + torch.rand(m, generator=g)).cuda() / 127, (0.5 + torch.rand(n, generator=g)).cuda() / (127 * math.sqrt(k) / 3)
    bias, res = torch.randn(n, generator=g).cuda(), torch.randn(m, n + 3, generator=g).cuda()[:, 2:2 + n]
    for lo, width, r, act in ((0, n, res, 1), (3, n + 7, None, 2), (5, n + 6, res, 0)):
        wide = torch.full((m, width + lo), 7.0, device="cuda", dtype=out)
        copy = torch.full((m, width + lo), 7.0, device="cuda", dtype=BF16) if out == F32 else None
        o = wide[:, lo:lo + n]
        K.gemm_i8(a, sa, b, sb, out=o, bias=bias, residual=r, act=act, aux_bf16_out=None if copy is None else copy[:, lo:lo + n])
        check_product(a, sa, b, sb, o, bias, r, act)
        assert (wide[:, :lo] == 7).all() and (wide[:, lo + n:] == 7).all()
        if copy is not None:
            assert torch.equal(copy[:, lo:lo + n], o.to(BF16)) and (copy[:, :lo] == 7).all() and (copy[:, lo + n:] == 7).all()


def test_few_bits_offsets_past_32_bits():
    m, n, k = 70001, 32768, 48                                                # 2.3e9 results
    g = gen(5)
    x = torch.randn(m, k, generator=g).cuda()
    w8, ws = K.quant_rows_i8(torch.randn(n, k, generator=g).cuda())
    q, s = K.quant_rows_i8(x)
    out = K.linear_i8(x, w8, ws)
    for r in (0, 65535, 65537, m - 1):
        check_product(q[r:r + 1], s[r:r + 1], w8, ws, out[r:r + 1])
    del out
    rows = 540000
    x = torch.ones(1, 4096, dtype=BF16, device="cuda").repeat(rows, 1)        # 2.2e9 values
    x[-1] = -2.0
    x[-1, 5] = 4.0
    q, s = K.quant_rows_i8(x)
    assert int(q[-1, 5]) == 127 and int(q[-1, 4]) == -64 and float(s[-1]) == float(torch.tensor(4.0) / 127) and bool((q[-2] == 127).all())


@pytest.mark.parametrize("m,n,k", [(7, 40, 64), (300, 776, 768), (1300, 2264, 144), (5000, 2304, 768)])
def test_gemm_i8_adds_to_the_residual_in_place(m, n, k):
    g = gen(m * n)
    a, b = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((m, k), (n, k)))
    sa, sb = torch.rand(m, generator=g).cuda() / 100, torch.rand(n, generator=g).cuda() / 100
    x = torch.randn(m, n, generator=g).cuda()
    expected = K.gemm_i8(a, sa, b, sb, out_dtype=F32, residual=x)
    check_product(a, sa, b, sb, expected, residual=x)
    K.gemm_i8(a, sa, b, sb, out=x, residual=x)
    assert torch.equal(x, expected)


def test_gemm_i8_sums_stay_exact_at_the_longest_k():
    k = 131072
    a = torch.full((3, k), 127, dtype=torch.int8, device="cuda")
    b = torch.full((2, k), -127, dtype=torch.int8, device="cuda")
    b[1] = 127
    b[1, -1] = 126
    one = torch.ones(3, device="cuda")
    out = K.gemm_i8(a, one, b, one[:2].contiguous(), out_dtype=F32)
    assert out[0].tolist() == [float(torch.tensor(-127 * 127 * k, dtype=F32)), float(torch.tensor(127 * 127 * k - 127, dtype=F32))]


@pytest.mark.parametrize("m", [1, 16, 40, 64, 65, 500, 900])
@pytest.mark.parametrize("k", [50, 768, 2300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_i8_is_quantise_then_multiply(m, k, dtype):
    g = gen(m * k)
    x = torch.randn(m, k, generator=g).to(dtype).cuda()
    w8, ws = K.quant_rows_i8(torch.randn(200, k, generator=g).cuda())
    bias = torch.randn(200, generator=g).cuda()
    x[0, 0] = float("nan") if m > 2 else 1.0
    out = K.linear_i8(x, w8, ws, bias=bias, act=1)
    q, s = K.quant_rows_i8(x)
    assert torch.equal(out, K.gemm_i8(q, s, w8, ws, bias=bias, act=1)) or (m > 2 and torch.equal(out[1:], K.gemm_i8(q, s, w8, ws, bias=bias, act=1)[1:]))
    if m > 2:
        assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()


@pytest.mark.parametrize("m,n", [(5, 40), (300, 700), (2100, 1536), (4400, 2304)])
@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("out", [BF16, F32])
def test_linear_i8_rows_without_numbers_stay_so_behind_every_activation(m, n, act, out):
    x = torch.randn(m, 128, generator=gen(m)).cuda()
    x[m // 2, 7] = math.inf
    w8, ws = K.quant_rows_i8(torch.randn(n, 128, generator=gen(n)).cuda())
    y = K.linear_i8(x, w8, ws, act=act, out_dtype=out, residual=torch.ones(m, n, device="cuda"))
    none = torch.isnan(y)
    assert none[m // 2].all() and int(none.sum()) == n


def test_few_bits_refuse_rows_that_share_memory():
    """A broadcast row has pitch 0: read as rows of its width it would run past its memory."""
    w8, ws = K.quant_rows_i8(torch.randn(32, 64, device="cuda"))
    row, many = torch.randn(1, 64, device="cuda"), torch.randn(5, 64, device="cuda")
    q8, s8 = K.quant_rows_i8(many)
    c = K.KV4Cache(5, 10, 1, 64)
    kv = many.to(BF16)
    for call in (lambda: K.quant_rows_i8(row.expand(5, 64)), lambda: K.linear_i8(row.expand(5, 64), w8, ws), lambda: K.gemm_i8(q8[:1].expand(5, 64), s8, w8, ws),
                 lambda: K.gemm_i8(q8, s8, w8[:1].expand(32, 64), ws), lambda: K.linear_i8(many, w8, ws, residual=torch.zeros(1, 32, device="cuda").expand(5, 32)),
                 lambda: K.linear_i8(many, w8, ws, out=torch.zeros(1, 32, device="cuda").expand(5, 32)), lambda: K.kv4_append(c, kv, kv[:1].expand(5, 64)),
                 lambda: K.attn_kv4(kv[:1].expand(5, 64), c, heads=1, scale=1.0)):
        with pytest.raises(AdtError):
            call()


def test_few_bits_empty_calls():
    w8, ws = K.quant_rows_i8(torch.randn(8, 20, device="cuda"))
    assert K.linear_i8(torch.empty(0, 20, device="cuda"), w8, ws).shape == (0, 8)
    q, s = K.quant_rows_i8(torch.randn(3, 20, device="cuda"))
    assert K.gemm_i8(q, s, w8[:0], ws[:0]).shape == (3, 0)
    c = K.KV4Cache(0, 10, 2, 64)
    empty = torch.empty((0, 128), dtype=BF16, device="cuda")
    K.kv4_append(c, empty, empty)
    assert K.kv4_read(c)[0].shape == (0, 128) and K.attn_kv4(empty, c, heads=2, scale=1.0).shape == (0, 128)


# --------------------------------------------------------------------------------------------------- cache
def held(x, heads, dim):
    """(value, scale, minimum) in 64 bits of bf16 rows [n, heads * dim]."""
    g = x.to(F64).reshape(x.shape[0], heads, dim // 64, 64)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi.to(F32) - lo.to(F32)).to(F64) / 15.0).clamp(min=TINY).to(F32).to(BF16).to(F64)
    c = torch.round((g - lo) / s).clamp(max=15)
    return (lo + c * s).reshape(x.shape), s, lo


def kv_rows(n, heads, dim, seed, spread=1.0):
    g = gen(seed)
    x = torch.randn(n, 2 * heads * dim + 16, generator=g) * spread + torch.randn(1, 2 * heads * dim + 16, generator=g)
    x = x.to(BF16).cuda()
    return x[:, 8:8 + heads * dim], x[:, 8 + heads * dim:8 + 2 * heads * dim]


def check_held(out, x, heads, dim):
    ref, s, lo = held(x, heads, dim)
    mag = (15 * s + lo.abs()).expand(-1, -1, -1, 64).reshape(x.shape)
    err = 2 * U * mag if out.dtype == F32 else 2 * U * mag + 2.0 ** -8 * (ref.abs() + 2 * U * mag)
    assert ((out.to(F64) - ref).abs() <= err).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads,cap,n", [(1, 1, 1, 1), (2, 3, 33, 33), (1, 6, 986, 986), (3, 2, 64, 31), (2, 1, 100, 65)])
def test_kv4_append_and_read(dim, batch, heads, cap, n):
    c = K.KV4Cache(batch, cap, heads, dim)
    assert c.nbytes == batch * heads * -(-cap // 32) * 36 * dim
    c.data.fill_(0xFF)
    k, v = kv_rows(batch * n, heads, dim, cap + n)
    end = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    K.kv4_append(c, k, v, end)
    for dt in (F32, BF16):
        rk, rv = K.kv4_read(c, end, None, n, out_dtype=dt)
        check_held(rk, k, heads, dim)
        check_held(rv, v, heads, dim)


@pytest.mark.parametrize("dim", [64, 128])
def test_kv4_append_piecewise_equals_whole_and_keeps_what_was_there(dim):
    batch, heads, cap = 4, 3, 150
    k, v = kv_rows(batch * cap, heads, dim, 5)
    whole, parts = K.KV4Cache(batch, cap, heads, dim), K.KV4Cache(batch, cap, heads, dim)
    K.kv4_append(whole, k, v)
    parts.data.random_(0, 256)
    pos = torch.zeros(batch, dtype=torch.int64)
    k4, v4 = k.reshape(batch, cap, -1), v.reshape(batch, cap, -1)
    g = gen(9)
    while int(pos.min()) < cap:                                               # ragged pieces of 0 .. 40 rows, single tokens among them
        n = int(torch.randint(1, 41, (1,), generator=g)) if int(pos[0]) % 3 else 1
        count = torch.minimum(torch.randint(0, n + 1, (batch,), generator=g), cap - pos)
        idx = (pos[:, None] + torch.arange(n)).clamp(max=cap - 1)
        rows = [t[torch.arange(batch)[:, None], idx].reshape(batch * n, -1) for t in (k4.cpu(), v4.cpu())]
        pos = pos + count
        K.kv4_append(parts, rows[0].cuda(), rows[1].cuda(), pos.to(torch.int32).cuda(), count.to(torch.int32).cuda())
        seen = pos.to(torch.int32).cuda()
        a, b = K.kv4_read(parts, seen, seen, cap), K.kv4_read(whole, seen, seen, cap)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_kv4_positions_outside_the_cache_are_left_out():
    batch, heads, dim, cap, n = 5, 2, 64, 40, 8
    k, v = kv_rows(batch * n, heads, dim, 1)
    c = K.KV4Cache(batch, cap, heads, dim)
    base_k, base_v = kv_rows(batch * cap, heads, dim, 2)
    K.kv4_append(c, base_k, base_v)
    before = K.kv4_read(c, out_dtype=F32)
    end = torch.tensor([3, 44, -5, 2 ** 31 - 1, 0], dtype=torch.int32, device="cuda")
    K.kv4_append(c, k, v, end)                                                # rows 5.. of 0, rows ..3 of 1, none of the others
    after = K.kv4_read(c, out_dtype=F32)
    for x, src, b0, b1 in ((k, k, before[0], after[0]), (v, v, before[1], after[1])):
        b0, b1, src = b0.reshape(batch, cap, -1), b1.reshape(batch, cap, -1), src.reshape(batch, n, -1)
        assert torch.equal(b1[2:], b0[2:]) and torch.equal(b1[0, 3:], b0[0, 3:]) and torch.equal(b1[1, :36], b0[1, :36])
        check_held(b1[0, :3], src[0, 5:], heads, dim)
        check_held(b1[1, 36:], src[1, :4], heads, dim)
    r = K.kv4_read(c, end, None, n, out_dtype=F32)[0].reshape(batch, n, -1)
    assert not r[2:].any() and not r[0, :5].any() and not r[1, 4:].any()
    count = torch.tensor([-1, 100, 0, 1, 2], dtype=torch.int32, device="cuda")      # counts are taken into 0 .. n
    r = K.kv4_read(c, torch.full_like(end, cap), count, n, out_dtype=F32)[0].reshape(batch, n, -1)
    assert not r[0].any() and torch.equal(r[1], after[0].reshape(batch, cap, -1)[1, cap - n:]) and not r[3, 1:].any() and not r[4, 2:].any()


def test_kv4_equal_values_extremes_and_groups_without_numbers():
    heads, dim = 1, 128
    x = torch.zeros(6, 128)
    x[0] = 3.0
    x[1, :2] = torch.tensor([1e38, -1e38])
    x[2, 70] = math.inf
    x[3, 5] = math.nan
    x[4, :2] = torch.tensor([3e38, -3e38])                                    # the range exceeds fp32
    x[5] = 1e-38
    x = x.to(BF16).cuda()
    c = K.KV4Cache(1, 6, heads, dim)
    K.kv4_append(c, x, x.flip(0).contiguous())
    k, v = K.kv4_read(c, out_dtype=F32)
    assert torch.equal(v.flip(0).isnan(), k.isnan())
    bad = torch.zeros(6, 128, dtype=torch.bool)
    bad[2, 64:] = bad[3, :64] = bad[4, :64] = True
    assert torch.equal(k.isnan().cpu(), bad)
    check_held(k[[0, 1, 5]], x[[0, 1, 5]], heads, dim)
    assert (k[0] == 3.0).all()


def test_kv4_offsets_past_32_bits():
    batch, heads, dim, cap = 40, 8, 128, 100000                               # 4.6 GB
    c = K.KV4Cache(batch, cap, heads, dim)
    assert c.nbytes > 2 ** 32
    k, v = kv_rows(batch * 3, heads, dim, 3)
    end = torch.full((batch,), cap, dtype=torch.int32, device="cuda")
    K.kv4_append(c, k, v, end)
    rk, rv = K.kv4_read(c, end, None, 3)
    check_held(rk, k, heads, dim)
    check_held(rv, v, heads, dim)
    # the last sequence's last span is read by the attention too: a cleared cache is rows of zeros (equal weights), three rows at its end
    last = c.data[-heads * -(-cap // 32) * 36 * dim:]
    last.zero_()
    K.kv4_append(c, k, v, end)
    q = torch.zeros((batch, heads * dim), dtype=BF16, device="cuda")
    n = torch.zeros(batch, dtype=torch.int32, device="cuda")
    n[-1] = cap
    out = K.attn_kv4(q, c, n, heads=heads, scale=1.0)
    ref, s, lo = held(v[-3:], heads, dim)
    mag = (31 * s + lo.abs()).expand(-1, -1, -1, 64).reshape(3, -1).sum(0) / cap
    ref = ref.sum(0) / cap
    assert not out[:-1].any()
    assert ((out[-1].to(F64) - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -14 * mag).all()


# --------------------------------------------------------------------------------------------------- attention
def attn_ref(q, k, v, heads, kv_heads, dim, batch, q_len, key_len, scale, causal):
    """(o, lse, magnitude) in 64 bits; k, v [batch, keys, kv_heads * dim] as bf16 rows."""
    keys = k.shape[1]
    o = torch.zeros(batch, q_len, heads, dim, dtype=F64, device="cuda")
    mag = torch.zeros_like(o)
    lse = torch.full((batch, heads, q_len), -math.inf, dtype=F64, device="cuda")
    g = heads // kv_heads
    qq = q.to(F64).reshape(batch, q_len, heads, dim)
    for b in range(batch):
        kk, ks, km = held(k[b], kv_heads, dim)
        vv, vs, vm = held(v[b], kv_heads, dim)
        kk, vv = kk.reshape(keys, kv_heads, dim), vv.reshape(keys, kv_heads, dim)
        kmag = (31 * ks + km.abs()).expand(-1, -1, -1, 64).reshape(keys, kv_heads, dim)
        vmag = (31 * vs + vm.abs()).expand(-1, -1, -1, 64).reshape(keys, kv_heads, dim)
        for i in range(q_len):
            n = key_len[b] - (q_len - 1 - i) if causal else key_len[b]
            n = min(n, keys)
            if n <= 0:
                continue
            for h in range(heads):
                z = kk[:n, h // g] @ qq[b, i, h] * scale
                p = torch.softmax(z, 0)
                o[b, i, h] = p @ vv[:n, h // g]
                lse[b, h, i] = torch.logsumexp(z, 0)
                # a score is off by a few roundings of the magnitudes that meet in it (64 products and their sum: 8 of them), a weight
                # by that much and 2^-22 of its exponential, a weighted value by 2^-16 (two bf16 halves) -- twice, numerator and sum
                dz = 8 * U * float((kmag[:n, h // g] @ qq[b, i, h].abs()).max()) * scale
                mag[b, i, h] = (2 * dz + 2.0 ** -21 + 2.0 ** -16) * (p @ vmag[:n, h // g])
    return o.reshape(batch * q_len, -1), lse, mag.reshape(batch * q_len, -1)


def check_attn(out, lse, q, k, v, heads, kv_heads, dim, batch, q_len, key_len, scale, causal):
    o, l, mag = attn_ref(q, k, v, heads, kv_heads, dim, batch, q_len, key_len, scale, causal)
    d = (out.to(F64) - o).abs()
    assert (d <= 2.0 ** -8 * (o.abs() + mag) + mag).all(), float((d - 2.0 ** -8 * o.abs() - mag).max())
    none = l == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert ((lse.to(F64) - l)[~none].abs() <= 1e-4).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,q_len,causal,lens,cap", [
    (1, 1, 1, False, [1], 1), (6, 6, 1, False, [0, 1, 2, 31, 32, 33, 64, 100], 100), (6, 2, 1, True, [5, 77, 129], 150), (8, 1, 3, True, [1, 2, 3, 40], 45),
    (5, 5, 7, True, [0, 6, 7, 8, 90], 96), (32, 2, 2, False, [3, 70], 70), (4, 2, 40, True, [50, 33, 12], 64), (1, 1, 1, False, [700, 1234], 1300),
    (6, 3, 5, False, [300, 0, 999], 1000)])
def test_attn_kv4_against_its_definition(dim, heads, kv_heads, q_len, causal, lens, cap):
    batch = len(lens)
    k, v = kv_rows(batch * cap, kv_heads, dim, cap + q_len + heads)
    c = K.KV4Cache(batch, cap, kv_heads, dim)
    c.data.fill_(0xFF)                                                        # NaN parameters wherever nothing is appended
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    K.kv4_append(c, k, v, n, n)                                               # sequence b's first lens[b] rows, and nothing behind them
    q = (1.5 * torch.randn(batch * q_len, (heads + 2) * dim, generator=gen(7))).to(BF16).cuda()[:, dim:dim + heads * dim]
    scale = 1.0 / math.sqrt(dim)
    out, lse = K.attn_kv4(q, c, n, heads=heads, scale=scale, q_len=q_len, causal=causal, want_lse=True)
    check_attn(out, lse, q, k.reshape(batch, cap, -1), v.reshape(batch, cap, -1), heads, kv_heads, dim, batch, q_len, lens, scale, causal)
    wide = torch.full((batch * q_len, heads * dim + 9), 5.0, dtype=BF16, device="cuda")      # unaligned rows in and out
    odd = torch.empty((batch * q_len, heads * dim + 3), dtype=BF16, device="cuda")
    odd[:, 1:1 + heads * dim] = q
    K.attn_kv4(odd[:, 1:1 + heads * dim], c, n, heads=heads, scale=scale, q_len=q_len, causal=causal, out=wide[:, 3:3 + heads * dim])
    assert torch.equal(wide[:, 3:3 + heads * dim], out) and (wide[:, :3] == 5).all() and (wide[:, 3 + heads * dim:] == 5).all()


@pytest.mark.parametrize("dim,heads,kv_heads,cap,lens", [(128, 4, 1, 20000, [20000, 1, 0, 12345]), (64, 2, 2, 9001, [9001, 8800])])
def test_attn_kv4_long_contexts_in_spans(dim, heads, kv_heads, cap, lens):
    batch = len(lens)
    k, v = kv_rows(batch * cap, kv_heads, dim, 11)
    c = K.KV4Cache(batch, cap, kv_heads, dim)
    K.kv4_append(c, k, v)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = (2 * torch.randn(batch, heads * dim, generator=gen(3))).to(BF16).cuda()
    out, lse = K.attn_kv4(q, c, n, heads=heads, scale=dim ** -0.5, want_lse=True)
    check_attn(out, lse, q, k.reshape(batch, cap, -1), v.reshape(batch, cap, -1), heads, kv_heads, dim, batch, 1, lens, dim ** -0.5, False)
    full = K.attn_kv4(q, c, heads=heads, scale=dim ** -0.5)
    assert torch.equal(full[0], out[0])
    again = K.attn_kv4(q, c, n, heads=heads, scale=dim ** -0.5)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads,kv_heads,q_len,causal,cap", [
    (180, 3, 3, 1, False, 9), (180, 6, 3, 2, True, 150), (100, 3, 3, 1, False, 1600), (150, 4, 2, 3, True, 1400), (40, 2, 2, 9, True, 900), (30, 4, 4, 1, False, 2500)])
def test_attn_kv4_many_sequences_of_all_lengths(dim, batch, heads, kv_heads, q_len, causal, cap):
    """Every way a call is cut into waves and spans, with sequences from empty to full side by side."""
    k, v = kv_rows(batch * cap, kv_heads, dim, cap + batch)
    c = K.KV4Cache(batch, cap, kv_heads, dim)
    c.data.fill_(0xFF)
    lens = torch.randint(0, cap + 1, (batch,), generator=gen(cap)).tolist()
    lens[0], lens[batch // 2], lens[-1] = cap, 0, 1
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    K.kv4_append(c, k, v, n, n)
    q = (1.5 * torch.randn(batch * q_len, heads * dim, generator=gen(batch))).to(BF16).cuda()
    out, lse = K.attn_kv4(q, c, n, heads=heads, scale=dim ** -0.5, q_len=q_len, causal=causal, want_lse=True)
    check_attn(out, lse, q, k.reshape(batch, cap, -1), v.reshape(batch, cap, -1), heads, kv_heads, dim, batch, q_len, lens, dim ** -0.5, causal)


def test_attn_kv4_rising_scores_and_far_apart_maxima():
    """Every tile raises the maximum, by more than the lazy threshold and by less; scores of hundreds."""
    dim, cap = 128, 640
    x = torch.linspace(0.01, 4.0, cap)[:, None] * torch.ones(1, dim)
    k = (x + 0.02 * torch.randn(cap, dim, generator=gen(1))).to(BF16).cuda()
    v = torch.randn(cap, dim, generator=gen(2)).to(BF16).cuda()
    c = K.KV4Cache(1, cap, 1, dim)
    K.kv4_append(c, k, v)
    for gain in (0.05, 1.0, 20.0, -20.0):
        q = torch.full((1, dim), gain, dtype=BF16, device="cuda")
        n = torch.tensor([cap], dtype=torch.int32, device="cuda")
        out, lse = K.attn_kv4(q, c, n, heads=1, scale=dim ** -0.5, want_lse=True)
        o, l, mag = attn_ref(q, k[None], v[None], 1, 1, dim, 1, 1, [cap], dim ** -0.5, False)
        assert ((out.to(F64) - o).abs() <= 2.0 ** -8 * (o.abs() + mag) + mag).all()
        assert float((lse.to(F64) - l).abs()) <= 1e-6 * abs(float(l)) + 1e-4


@pytest.mark.parametrize("dim", [64, 128])
def test_attn_kv4_numbers_that_are_none_stay_where_they_are_seen(dim):
    """A NaN key or value reaches the rows that see it, and no other row, head or sequence; behind the lengths it reaches nothing."""
    batch, heads, cap, q_len = 2, 2, 80, 4
    k, v = (t.clone() for t in kv_rows(batch * cap, heads, dim, 2))
    k[70, 3] = float("nan")                                                   # sequence 0, head 0, position 70
    v[cap + 75, dim + 1] = float("inf")                                       # sequence 1, head 1, position 75
    c = K.KV4Cache(batch, cap, heads, dim)
    K.kv4_append(c, k, v)
    q = torch.randn(batch * q_len, heads * dim, generator=gen(5)).to(BF16).cuda()
    n = torch.tensor([72, 76], dtype=torch.int32, device="cuda")              # causal: query i sees 69 .. 72 and 73 .. 76 positions
    out = K.attn_kv4(q, c, n, heads=heads, scale=0.1, q_len=q_len, causal=True).reshape(batch, q_len, heads, dim)
    bad = torch.isnan(out).any(-1).cpu()
    want = torch.zeros(batch, q_len, heads, dtype=torch.bool)
    want[0, 2:, 0] = True
    want[1, 3:, 1] = True
    assert torch.equal(bad, want)
    assert torch.isfinite(out[~torch.isnan(out)]).all()
    clean = K.KV4Cache(batch, cap, heads, dim)
    k2, v2 = torch.nan_to_num(k), torch.nan_to_num(v, posinf=1.0)
    K.kv4_append(clean, k2, v2)
    ref = K.attn_kv4(q, clean, n, heads=heads, scale=0.1, q_len=q_len, causal=True).reshape(batch, q_len, heads, dim)
    assert torch.equal(out[~want.cuda()], ref[~want.cuda()])


def test_few_bits_on_another_stream_and_in_graphs():
    """append + attention + linear layers as one decode step would run them: eagerly, on a side stream, and captured (two graphs, replayed in
    turn with eager work between), all with the same bits."""
    torch.manual_seed(0)
    batch, heads, dim, cap = 3, 2, 128, 3000
    d = heads * dim
    w8, ws = K.quant_rows_i8(torch.randn(3 * d, d, device="cuda") / 16)
    o8, os_ = K.quant_rows_i8(torch.randn(d, d, device="cuda") / 16)
    k, v = kv_rows(batch * cap, heads, dim, 8)
    c = K.KV4Cache(batch, cap, heads, dim)
    K.kv4_append(c, k, v)
    x = torch.randn(batch, d, device="cuda").to(BF16)
    n = torch.tensor([2999, 1500, 40], dtype=torch.int32, device="cuda")

    def step(x):
        qkv = K.linear_i8(x, w8, ws)
        K.kv4_append(c, qkv[:, d:2 * d], qkv[:, 2 * d:], n)
        o = K.attn_kv4(qkv[:, :d], c, n, heads=heads, scale=dim ** -0.5)
        return K.linear_i8(o, o8, os_, out_dtype=F32)

    x2 = torch.randn_like(x)
    want, want2 = step(x).clone(), step(x2).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = []
    for inp in (x, x2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(inp)
        graphs.append((g, out))
    for rep in range(3):
        for (g, out), ref in zip(graphs, (want, want2)):
            out.zero_()
            g.replay()
            assert torch.equal(out, ref)
            torch.cuda.synchronize()
            assert torch.equal(step(x), want)
            junk = torch.randn(1 << 20, device="cuda").sum()
            del junk


@pytest.mark.parametrize("m,n,k", [(40, 300, 200), (300, 700, 2500), (1300, 2264, 144), (4400, 2304, 768)])
def test_linear_i8_of_every_size_replays_as_a_graph(m, n, k):
    g = gen(n)
    w8, ws = K.quant_rows_i8(torch.randn(n, k, generator=g).cuda())
    x = torch.randn(m, k, generator=g).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.linear_i8(x, w8, ws, act=1)
    for rep in range(3):
        x.copy_(torch.randn(m, k, generator=g))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, K.linear_i8(x, w8, ws, act=1))

"""8-bit-integer products (K16) in every kernel form, epilogue and output type against sums in 64 bits, where the other tests do not look: workgroups that walk
several 256 x 256 tiles, the few-token kernels, and ``linear_i8`` with all that the network gives it."""
import math

import pytest
import torch

from adt_str_amd import kernels as K
from tests.test_few_bits_limits_gpu import gen, nearest_codes

pytestmark = pytest.mark.gpu
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
U = 2.0 ** -24
# |x| Q(|x|) of the GELU: the polynomial and its fp32 rounding 4.1e-8 at most (at 1.54), 4.8e-8 with an exponential that is off by a unit in its last place (at
# 1.42), maxima over all a up to 14 of fp32 arithmetic with the kernel's coefficients
GELU_ERR = 4.9e-8
SWEEP = [("plain", 0, False), ("gelu", 1, False), ("relu", 2, False), ("residual", 0, True), ("gelu_residual", 1, True)]


def expected(acc, sa, sb, bias, act, residual):
    """Values and how far fp32 may be from them: the sum as a float, two scales, the bias, each rounded once; |gelu'| <= 1.13; one rounding of the GELU's last
    operation and one of the residual's."""
    prod = acc * sa.to(F64)[:, None] * sb.to(F64)
    z = prod if bias is None else prod + bias.to(F64)
    err = 4 * U * (prod.abs() + (0 if bias is None else bias.abs().to(F64)))
    del prod
    if act == 1:
        z, err = 0.5 * z * torch.erfc(-z / math.sqrt(2.0)), 1.13 * err + GELU_ERR
        err = err + U * (z.abs() + err)
    elif act == 2:
        z = z.clamp(min=0)
    if residual is not None:
        z = z + residual.to(F64)
        err = err + U * (z.abs() + err)
    return z, err


def check(out, z, err):
    if out.dtype == BF16:
        err = err + 2.0 ** -8 * (z.abs() + err)
    d = (out.to(F64) - z).abs()
    assert (d <= err + 1e-37).all(), float((d - err).max())


def operands(m, n, k, pad=0):
    g = gen(m + 3 * n + 7 * k)
    a, b = (torch.randint(-127, 128, (r, k + pad), generator=g, dtype=torch.int8).cuda()[:, :k] for r in (m, n))
    sa, sb = (0.5 + torch.rand(m, generator=g)).cuda() / 127, (0.5 + torch.rand(n, generator=g)).cuda() / (127 * math.sqrt(k) / 3)
    return a, b, sa, sb, torch.randn(n, generator=g).cuda(), torch.randn(m, n, generator=g).cuda()


# 79 x 9, 71 x 9 and 80 x 9 tiles on 256 CUs: two or three a workgroup, edge tiles in front of interior ones and behind them; one step of K to seven, and
# with a tail
@pytest.mark.parametrize("m,n,k", [(20001, 2304, 128), (20001, 2301, 256), (18001, 2304, 384), (20480, 2304, 784), (20001, 2304, 768), (20001, 2304, 96)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_workgroups_that_walk_several_large_tiles(m, n, k, out):
    a, b, sa, sb, bias, res = operands(m, n, k)
    acc = torch.matmul(a.to(F64), b.to(F64).t().contiguous())
    for name, act, with_res in SWEEP:
        r = res if with_res else None
        copy = torch.empty((m, n), dtype=BF16, device="cuda") if with_res and out == F32 else None
        y = K.gemm_i8(a, sa, b, sb, out_dtype=out, bias=bias, act=act, residual=r, aux_bf16_out=copy)
        check(y, *expected(acc, sa, sb, bias, act, r))
        assert copy is None or torch.equal(copy, y.to(BF16)), name
    if out == F32:
        want = K.gemm_i8(a, sa, b, sb, out_dtype=out, residual=res)
        K.gemm_i8(a, sa, b, sb, out=res, residual=res)
        assert torch.equal(res, want)
    else:                                                                      # rows that are not whole lines, in a wider buffer
        wide = torch.full((m, n + 9), 7.0, dtype=BF16, device="cuda")
        K.gemm_i8(a, sa, b, sb, out=wide[:, 5:5 + n])
        check(wide[:, 5:5 + n], *expected(acc, sa, sb, None, 0, None))
        assert (wide[:, :5] == 7).all() and (wide[:, 5 + n:] == 7).all()


# 16, 32 and 64 tokens a workgroup at widths of all remainders (16: (40, 95), (16, 7999); 32: (64, 1401), (260, 263), (30, 8001); 64: (64, 4001), (300, 701))
@pytest.mark.parametrize("m,n,k", [(40, 95, 80), (16, 7999, 64), (64, 1401, 768), (260, 263, 192), (30, 8001, 208), (64, 4001, 768), (300, 701, 400)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_few_tokens_in_every_form(m, n, k, out):
    a, b, sa, sb, bias, res = operands(m, n, k, 16)
    acc = torch.matmul(a.to(F64), b.to(F64).t().contiguous())
    for name, act, with_res in SWEEP:
        r = res if with_res else None
        wide = torch.full((m, n + 8), 7.0, dtype=out, device="cuda")
        copy = torch.full((m, n + 8), 7.0, dtype=BF16, device="cuda") if out == F32 else None
        y = wide[:, 3:3 + n]
        K.gemm_i8(a, sa, b, sb, out=y, bias=bias, act=act, residual=r, aux_bf16_out=None if copy is None else copy[:, 1:1 + n])
        check(y, *expected(acc, sa, sb, bias, act, r))
        assert (wide[:, :3] == 7).all() and (wide[:, 3 + n:] == 7).all()
        if copy is not None:
            assert torch.equal(copy[:, 1:1 + n], y.to(BF16)) and (copy[:, :1] == 7).all() and (copy[:, 1 + n:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(40, 96, 64), (300, 776, 768), (1000, 1000, 256), (2100, 1537, 64), (4400, 2304, 128), (20001, 2304, 128)])
def test_gelu_over_its_range(m, n, k):
    """Arguments from -14 to 14: every piece of the curve, to the polynomial's own error."""
    a, b = torch.zeros((m, k), dtype=torch.int8, device="cuda"), torch.zeros((n, k), dtype=torch.int8, device="cuda")
    a[:, 0], b[:, 0] = 100, 1
    sa = (torch.linspace(-14, 14, m, dtype=F64) / 100).to(F32).cuda()
    sb = torch.linspace(0.25, 1.0, n).cuda()
    y = K.gemm_i8(a, sa, b, sb, act=1, out_dtype=F32)
    check(y, *expected(torch.full((m, n), 100.0, dtype=F64, device="cuda"), sa, sb, None, 1, None))


@pytest.mark.parametrize("m,n,k", [(1, 2303, 768), (16, 48, 2048), (33, 257, 50), (64, 768, 767), (200, 300, 100),                  # one launch
                                   (300, 1001, 768), (7, 40, 2300), (64, 2304, 768), (2100, 1537, 272), (5, 700, 9000), (20001, 2304, 200)])      # two
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("out", [BF16, F32])
def test_linear_i8_against_its_definition(m, n, k, dtype, out):
    g = gen(m + n + k)
    # rows of a packed buffer, 16-byte aligned; then rows that begin anywhere
    packed = (torch.randn(m, k + 24, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype).cuda()
    w8, ws = K.quant_rows_i8((torch.randn(n, k, generator=g) / math.sqrt(k)).cuda())
    bias, res, table = torch.randn(n, generator=g).cuda(), torch.randn(m, n + 5, generator=g).cuda()[:, 2:2 + n], torch.randn(37, n, generator=g).cuda()
    for lo in (8, 3):
        x = packed[:, lo:lo + k]
        codes, scale = nearest_codes(x), (x.to(F64).abs().amax(1) / 127.0).to(F32)
        acc = torch.matmul(codes, w8[:, :k].to(F64).t().contiguous())
        for name, act, with_res in SWEEP:
            r = res if with_res else None
            copy = torch.empty((m, n), dtype=BF16, device="cuda") if out == F32 else None
            y = K.linear_i8(x, w8, ws, out_dtype=out, bias=bias, act=act, residual=r, aux_bf16_out=copy)
            check(y, *expected(acc, scale, ws, bias, act, r))
            assert copy is None or torch.equal(copy, y.to(BF16)), name
        wide = torch.full((m, n + 7), 7.0, dtype=out, device="cuda")
        K.linear_i8(x, w8, ws, out=wide[:, 6:6 + n], residual=table, res_row_mod=37)
        check(wide[:, 6:6 + n], *expected(acc, scale, ws, None, 0, table[torch.arange(m, device="cuda") % 37]))
        assert (wide[:, :6] == 7).all() and (wide[:, 6 + n:] == 7).all()

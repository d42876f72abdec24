"""The 256 x 256 products with epilogues that read their flags at run time (combinations that have no compiled form of their own), over more tiles than
there are workgroups and ragged edges, against 64-bit references.  Operands are small integers, so that every sum is exact in fp32.  Tolerance: four
roundings in the epilogue, half a step of the output's type."""
import pytest
import torch

from adt_str_amd import kernels as K

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def rnd(shape, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(shape, generator=g).cuda()


def whole(shape, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=g).to(BF16).cuda()


def reference(a, b, bias, residual, act, alpha):
    z = torch.matmul(a.to(F64), b.to(F64)) * alpha
    mag = z.abs()
    if bias is not None:
        z, mag = z + bias.to(F64), mag + bias.abs().to(F64)
    if act == 2:
        z = z.clamp(min=0)
    if residual is not None:
        z, mag = z + residual.to(F64), mag + residual.abs().to(F64)
    return z, 4 * 2.0 ** -24 * mag


def check(out, z, err):
    step = 2.0 ** -8 if out.dtype == BF16 else 2.0 ** -24
    assert ((out.to(F64) - z).abs() <= err + step * (z.abs() + err)).all()


@pytest.mark.parametrize("m,n,k", [(8232, 2312, 256), (9001, 2304, 320), (4096, 4096, 512)])
@pytest.mark.parametrize("form", ["relu_residual_copy", "scaled", "relu_colsum"])
def test_nt(m, n, k, form):
    a, b = whole((m, k), m), whole((n, k), n)
    bias, res = rnd((n,), 3), rnd((m, n), 4)
    bt = b.t().contiguous()
    if form == "relu_residual_copy":
        copy = torch.empty((m, n), dtype=BF16, device="cuda")
        out = K.gemm(a, b, bias=bias, act=2, residual=res, out_dtype=F32, aux_bf16_out=copy)
        z, err = reference(a, bt, bias, res, 2, 1.0)
        assert torch.equal(copy, out.to(BF16))
    elif form == "scaled":
        out = K.gemm(a, b, alpha=0.375)
        z, err = reference(a, bt, None, None, 0, 0.375)
    else:
        sums = torch.empty(n, device="cuda")
        out = K.gemm(a, b, bias=bias, act=2, colsum_out=sums)
        z, err = reference(a, bt, bias, None, 2, 1.0)
        assert ((sums.to(F64) - out.to(F64).sum(0)).abs() <= m * 2.0 ** -24 * out.to(F64).abs().sum(0)).all()
    check(out, z, err)


@pytest.mark.parametrize("kd,m,n", [(4096, 4352, 4104), (4160, 768, 2304), (8192, 1032, 520)])
@pytest.mark.parametrize("form", ["plain", "bias_residual", "scaled_bf16"])
def test_tn(kd, m, n, form):
    a, b = whole((kd, m), m), whole((kd, n), n + 1)
    bias, res = rnd((n,), 5), rnd((m, n), 6)
    at = a.t().contiguous()
    if form == "plain":
        out = K.gemm(a, b, trans=True, out_dtype=F32)
        z, err = reference(at, b, None, None, 0, 1.0)
    elif form == "bias_residual":
        out = K.gemm(a, b, trans=True, out_dtype=F32, bias=bias, residual=res)
        z, err = reference(at, b, bias, res, 0, 1.0)
    else:
        out = K.gemm(a, b, trans=True, alpha=-0.5)
        z, err = reference(at, b, None, None, 0, -0.5)
    check(out, z, err)

"""Refusals of the few-bit serving operators (K16, K17): argument checks that need no GPU."""
import ctypes as C

import pytest
import torch

from adt_str_amd import _ffi
from adt_str_amd import kernels as K


@pytest.fixture(scope="module")
def lib():
    return _ffi.load()


ONE = 16                                       # a 16-byte aligned address that no refused call follows


def test_quant_rows_i8_refusals(lib):
    f = lib.adt_quant_rows_i8
    assert f(None, 0, 16, 1, 16, ONE, 16, ONE, None) == -1 and f(ONE, 0, 16, 1, 16, None, 16, ONE, None) == -1 and f(ONE, 0, 16, 1, 16, ONE, 16, None, None) == -1
    assert f(ONE, 0, 16, -1, 16, ONE, 16, ONE, None) == -2 and f(ONE, 0, 16, 1, 0, ONE, 16, ONE, None) == -2 and f(ONE, 0, 1 << 18, 1, (1 << 17) + 1, ONE, 1 << 18, ONE, None) == -2
    assert f(ONE, 0, 15, 1, 16, ONE, 16, ONE, None) == -1 and f(ONE, 0, 17, 1, 17, ONE, 16, ONE, None) == -1       # rows that do not hold K, or K rounded up
    assert f(ONE, 0, 16, 1, 16, ONE, 24, ONE, None) == -1 and f(ONE, 0, 16, 1, 16, ONE + 8, 16, ONE, None) == -1
    assert b"16-byte aligned" in lib.adt_last_error()
    assert f(ONE, 0, 16, 0, 16, ONE, 16, ONE, None) == 0                       # no rows: nothing to do


def test_gemm_i8_refusals(lib):
    def call(M=4, N=8, K_=32, A=ONE, lda=32, sa=ONE, B=ONE, ldb=32, sb=ONE, Cp=ONE, ldc=8, ep=True, **kw):
        e = _ffi.GemmEpilogue()
        e.alpha = 1.0
        for name, val in kw.items():
            if name == "drop":
                e.drop.p = val
            else:
                setattr(e, name, val)
        return lib.adt_gemm_i8(M, N, K_, A, lda, sa, B, ldb, sb, Cp, ldc, C.byref(e) if ep else None, None)

    for null in ("A", "sa", "B", "sb", "Cp"):
        assert call(**{null: None}) == -1
    assert call(ep=False) == -1
    assert call(K_=24, lda=32, ldb=32) == -2 and call(K_=0) == -2 and call(K_=131088, lda=131088, ldb=131088) == -2 and call(M=-1) == -2
    assert call(lda=16) == -1 and call(ldb=16) == -1 and call(ldc=7) == -1 and call(lda=40) == -1 and call(A=ONE + 4) == -1
    assert call(act=3) == -1 and call(alpha=0.5) == -1
    for field in ("gelu_grad_of", "pre_act_out", "colsum_out", "res_ln_mean"):
        assert call(**{field: ONE}) == -1
    assert b"inference product" in lib.adt_last_error()
    assert call(drop=0.1) == -1 and call(act_grad_mode=1) == -1 and call(side_fp32=1) == -1
    assert call(aux_bf16_out=ONE, ld_aux=8) == -1 and call(aux_bf16_out=ONE, ld_aux=7, out_fp32=1) == -1
    assert call(residual=ONE, ld_res=7) == -1 and call(residual=ONE, ld_res=8, res_row_mod=-1) == -1
    assert call(M=0) == 0 and call(N=0, ldc=0) == 0


def test_kv4_refusals(lib):
    assert lib.adt_kv4_bytes(2, 3, 128, 33) == 2 * 3 * 2 * 4608 and lib.adt_kv4_bytes(1, 1, 64, 1) == 2304
    assert lib.adt_kv4_bytes(1, 1, 96, 1) == 0 and lib.adt_kv4_bytes(0, 1, 64, 1) == 0
    ap = lambda cache=ONE, b=2, h=2, d=64, cap=10, k=ONE, ldk=128, v=ONE, ldv=128, n=3: lib.adt_kv4_append(cache, b, h, d, cap, k, ldk, v, ldv, n, None, None, None)  # noqa: E731
    assert ap(cache=None) == -1 and ap(cache=ONE + 8) == -1 and ap(k=None) == -1 and ap(v=None) == -1 and ap(n=-1) == -1
    assert ap(d=96) == -2 and ap(d=32) == -2 and ap(cap=0) == -1 and ap(h=0) == -1 and ap(b=-1) == -1 and ap(b=70000) == -2
    assert ap(ldk=127) == -1 and ap(ldv=100) == -1
    assert b"kv_heads * head_dim" in lib.adt_last_error()
    assert ap(b=0) == 0 and ap(n=0) == 0
    rd = lambda k=ONE, ldk=128, v=ONE, ldv=128, f32=0: lib.adt_kv4_read(ONE, 2, 2, 64, 10, k, ldk, v, ldv, f32, 3, None, None, None)  # noqa: E731
    assert rd(k=None) == -1 and rd(k=ONE + 2) == -1 and rd(ldk=129) == -1 and rd(ldv=130, f32=1) == -1


def test_attn_kv4_refusals(lib):
    def call(q=ONE, cache=ONE, o=ONE, ws=ONE, nb=None, desc=True, **kw):
        d = _ffi.AttnKv4Desc(2, 4, 2, 128, 1, 100, 0, 1.0, 512, 512, None)
        for name, val in kw.items():
            setattr(d, name, val)
        need = lib.adt_attn_kv4_workspace_bytes(C.byref(d))
        return lib.adt_attn_kv4(C.byref(d) if desc else None, q, cache, o, None, ws, need if nb is None else nb, None)

    assert call(desc=False) == -1 and call(q=None) == -1 and call(cache=None) == -1 and call(o=None) == -1 and call(cache=ONE + 4) == -1
    assert call(heads=3) == -2 and call(heads=0) == -2 and call(kv_heads=0) == -1 and call(head_dim=96) == -2 and call(q_len=0) == -1 and call(capacity=0) == -1
    assert call(ldq=511) == -1 and call(ldo=256) == -1 and call(batch=-1) == -1
    assert call(capacity=100000, ws=None) == -1 and call(capacity=100000, nb=8) == -1
    assert b"workspace" in lib.adt_last_error()
    assert call(batch=0) == 0


def test_python_wrappers_refuse_cpu_tensors_and_wrong_shapes():
    x = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        K.quant_rows_i8(x)
    with pytest.raises(AssertionError):
        K.quant_rows_i8(x.to(torch.float16))
    with pytest.raises(AssertionError):
        K.quant_rows_i8(x[:, ::2])
    a, s = torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        K.gemm_i8(a, s, a, s)
    for bad in (dict(a=a[:, :24]), dict(b=a[:, :16]), dict(a_scale=s[:3]), dict(b_scale=s.double())):
        kw = dict(a=a, a_scale=s, b=a, b_scale=s)
        kw.update(bad)
        with pytest.raises(AssertionError):
            K.gemm_i8(**kw)
    with pytest.raises(AssertionError):
        K.linear_i8(torch.zeros(2, 40), a, s)
    with pytest.raises(NotImplementedError):
        K.KV4Cache(1, 8, 2, 96, "cpu")
    with pytest.raises(ValueError):
        K.KV4Cache(1, 0, 2, 64, "cpu")
    c = K.KV4Cache(2, 8, 2, 64, "cpu")
    assert c.nbytes == 2 * 2 * 2304
    rows = torch.zeros((4, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        K.kv4_append(c, rows, rows)
    for bad in (dict(k=rows.float()), dict(k=rows[:3], v=rows[:3]), dict(k=rows[:, :64], v=rows[:, :64]), dict(end=torch.zeros(2)), dict(count=torch.zeros(3, dtype=torch.int32))):
        kw = dict(k=rows, v=rows)
        kw.update(bad)
        with pytest.raises(AssertionError):
            K.kv4_append(c, **kw)
    for bad in (dict(q=rows[:1]), dict(q=rows.float()), dict(heads=3), dict(q_len=0), dict(key_len=torch.zeros(2, dtype=torch.int64)), dict(q=rows[:2, :64])):
        kw = dict(q=rows[:2], heads=2)
        kw.update(bad)
        with pytest.raises(AssertionError):
            K.attn_kv4(kw.pop("q"), c, kw.pop("key_len", None), scale=1.0, **kw)

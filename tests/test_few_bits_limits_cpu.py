"""Refusals of the few-bit serving operators (K16, K17) that need no GPU, beside those of test_few_bits_cpu.py."""
import ctypes as C

import pytest

from adt_str_amd import _ffi


@pytest.fixture(scope="module")
def lib():
    return _ffi.load()


X, W, SCALE, OUT, AUX, RES, WS = (16 << i for i in range(1, 8))               # aligned addresses that no refused call follows


def product(lib, linear, M=4, N=8, K=32, x=X, ldx=32, sa=SCALE, w=W, ldw=32, sw=SCALE, c=OUT, ldc=8, ws=WS, ws_bytes=0, ep=True, x_fp32=0, **kw):
    e = _ffi.GemmEpilogue()
    e.alpha = 1.0
    for name, val in kw.items():
        setattr(e, name, val)
    e = C.byref(e) if ep else None
    if linear:
        return lib.adt_linear_i8(M, N, K, x, x_fp32, ldx, w, ldw, sw, c, ldc, e, ws, ws_bytes, None)
    return lib.adt_gemm_i8(M, N, K, x, ldx, sa, w, ldw, sw, c, ldc, e, None)


@pytest.mark.parametrize("linear", [False, True])
def test_i8_products_refuse_results_on_top_of_what_they_read(lib, linear):
    """A periodic residual in place would be added to before other rows read it; an operand would be overwritten while it is multiplied."""
    call = lambda **kw: product(lib, linear, **kw)  # noqa: E731
    in_place = dict(c=OUT, residual=OUT, ld_res=8, out_fp32=1)
    assert call(**dict(in_place, res_row_mod=2)) == -1
    assert b"in place" in lib.adt_last_error()
    assert call(**dict(in_place, ld_res=16)) == -1 and call(**dict(in_place, out_fp32=0)) == -1
    assert call(c=X) == -1 and call(c=W) == -1
    assert b"share no memory" in lib.adt_last_error()
    for at in (X, W, OUT, RES):
        assert call(aux_bf16_out=at, ld_aux=8, out_fp32=1, residual=RES, ld_res=8) == -1


def test_linear_i8_refusals(lib):
    need = lib.adt_linear_i8_workspace_bytes(3000, 2000, 100)
    assert need == 3000 * 112 + 3000 * 4                                      # too many products for one launch: codes and scales
    assert lib.adt_linear_i8_workspace_bytes(8, 8, 100) == 0 and lib.adt_linear_i8_workspace_bytes(0, 8, 100) == 0
    big = lambda **kw: product(lib, True, **dict(dict(M=3000, N=2000, K=100, ldx=100, ldw=112, ldc=2000, ws_bytes=need), **kw))  # noqa: E731
    assert big(ws=None) == -1 and big(ws_bytes=need - 1) == -1 and big(ws=WS + 4) == -1
    assert b"workspace" in lib.adt_last_error()
    for kw in (dict(x=None), dict(w=None), dict(sw=None), dict(c=None), dict(ep=False), dict(ldx=99), dict(ldw=96), dict(ldw=104), dict(w=W + 8), dict(ldc=1999), dict(act=3),
               dict(alpha=2.0), dict(residual=RES, ld_res=1999), dict(residual=RES, ld_res=2000, res_row_mod=-1), dict(aux_bf16_out=AUX, ld_aux=2000),
               dict(aux_bf16_out=AUX, ld_aux=1999, out_fp32=1), dict(colsum_out=RES), dict(pre_act_out=RES)):
        assert big(**kw) == -1, kw
    for kw in (dict(K=0), dict(K=131073, ldx=1 << 18, ldw=1 << 18), dict(M=-1), dict(N=-1), dict(M=(1 << 30) + 1)):
        assert big(**kw) == -2, kw
    assert big(M=0) == 0 and big(N=0, ldc=0) == 0

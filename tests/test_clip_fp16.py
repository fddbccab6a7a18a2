"""CPU-side checks of the updates that take a factor of the gradient: what they refuse before they touch a device."""
import ctypes

import pytest

import tbe_native

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
NULL = ctypes.c_void_p(0)


@pytest.mark.parametrize("dtype", [tbe_native.DTYPE_F32, tbe_native.DTYPE_F64])
def test_a_factor_goes_with_fp16_tables(dtype):
    lib = tbe_native.load()
    rcs = [lambda factor: lib.tbe_backward_planned_scaled(
               tbe_native.OPT_SGD, P, factor, P, dtype, 100, 4, 1, 1, 10, NULL, NULL, 0.1, 0.0, NULL, 0, 0, 0, P, 16, NULL),
           lambda factor: lib.tbe_backward_approx_adagrad_scaled(
               P, factor, P, dtype, 100, 0, 4, P, 1, P, 10, P, 1, NULL, P, 0.1, 0.1, NULL, 0, 0, 0, P, 16, NULL)]
    for call in rcs:
        assert call(P) == 1 and "factor" in lib.tbe_last_error().decode()
        assert call(NULL) == 2 and "workspace" in lib.tbe_last_error().decode()


def test_the_other_checks_are_those_of_the_plain_calls():
    lib = tbe_native.load()
    f16 = tbe_native.DTYPE_F16
    planned = lambda optimizer=0, psw=NULL, D=4, nbytes=16: lib.tbe_backward_planned_scaled(
        optimizer, P, P, P, f16, 100, D, 1, 1, 10, psw, P, 0.1, 0.0, psw, 0, 0, 0, P, nbytes, NULL)
    for kwargs, code, needle in [(dict(optimizer=2), 1, "optimizer"), (dict(psw=P), 1, "per-sample"),
                                 (dict(D=6), 1, "multiple of 4"), (dict(), 2, "workspace")]:
        assert planned(**kwargs) == code and needle in lib.tbe_last_error().decode()
    approx = lambda state=P, D=4: lib.tbe_backward_approx_adagrad_scaled(
        P, P, P, f16, 100, 0, D, P, 1, P, 10, P, 1, NULL, state, 0.1, 0.1, NULL, 0, 0, 0, P, 16, NULL)
    for kwargs, code, needle in [(dict(state=NULL), 1, "null"), (dict(D=6), 1, "multiple of 4"), (dict(), 2, "workspace")]:
        assert approx(**kwargs) == code and needle in lib.tbe_last_error().decode()

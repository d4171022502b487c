"""RMS norm's, the 8-bit matrices' and the gated layers' entry points refuse calls
that their header rules out, before any device work.  CPU only: addresses are made
up and never reached."""

import math

import pytest

from ember_amd import capi

INVALID, UNSUPPORTED = 1, 2
P, Q, R, S = 4096, 8192, 1 << 20, 1 << 21  # aligned addresses


def refused(status, want=INVALID):
    assert status == want
    assert capi.lib().ember_get_last_error() == want


def rows8(codes=P, scales=Q, rows=3, cols=200):
    return capi.Rows8View(codes, scales, rows, cols)


BAD_MATRICES = [dict(codes=None), dict(scales=None), dict(codes=P + 8), dict(scales=Q + 4), dict(rows=-1), dict(rows=2 ** 26 + 1), dict(cols=0),
                dict(cols=-5), dict(cols=2 ** 23 + 1)]


def write(m=None, x=R, ld=200, trans=0):
    return capi.lib().rows8_write(m or rows8(), x, ld, trans)


def read(m=None, out=R, ld=200):
    return capi.lib().rows8_read(m or rows8(), out, ld)


def linear(a=None, w=None, bias=None, residual=None, out=R, act=0):
    return capi.lib().linear8_fwd(a or rows8(), w or rows8(rows=7), bias, residual, out, act)


def gated8(a=None, w=None, bias=None, h=None, act=1):
    return capi.lib().gated8_fwd(a or rows8(), w or rows8(rows=14), bias, h or rows8(R, S, 3, 7), act)


def norm8(x=R, residual=None, gamma=S, total=None, y=None, eps=1e-5):
    return capi.lib().rmsnorm_fwd8(x, residual, gamma, total, y or rows8(), eps)


@pytest.mark.parametrize("bad", BAD_MATRICES)
@pytest.mark.parametrize("call", [write, read, lambda m: linear(a=m), lambda m: linear(w=m), lambda m: gated8(a=m), lambda m: gated8(w=m),
                                  lambda m: gated8(h=m), lambda m: norm8(y=m)])
def test_matrices_that_cannot_be(call, bad):
    refused(call(rows8(**bad)))


@pytest.mark.parametrize("call", [lambda: capi.lib().rows8_write(None, R, 200, 0), lambda: capi.lib().rows8_read(None, R, 200),
                                  lambda: capi.lib().linear8_fwd(None, rows8(), None, None, R, 0),
                                  lambda: capi.lib().linear8_fwd(rows8(), None, None, None, R, 0),
                                  lambda: capi.lib().gated8_fwd(rows8(), rows8(rows=14), None, None, 1),
                                  lambda: capi.lib().rmsnorm_fwd8(R, None, S, None, None, 1e-5)])
def test_no_matrix(call):
    refused(call())


@pytest.mark.parametrize("change", [dict(x=None), dict(x=R + 2), dict(ld=199), dict(ld=2 ** 40 + 1), dict(trans=2), dict(trans=-1),
                                    dict(trans=1, ld=2)])
def test_write(change):
    refused(write(**change))


@pytest.mark.parametrize("change", [dict(out=None), dict(out=R + 1), dict(ld=199), dict(ld=-200), dict(ld=2 ** 40 + 1)])
def test_read(change):
    refused(read(**change))


@pytest.mark.parametrize("change", [dict(a=rows8(cols=201)), dict(w=rows8(cols=72)), dict(bias=R + 2), dict(residual=R + 1), dict(out=None),
                                    dict(out=R + 3), dict(act=-1), dict(act=2)])
def test_linear8(change):
    refused(linear(**change))


@pytest.mark.parametrize("change", [dict(a=rows8(cols=201)), dict(w=rows8(rows=13)), dict(w=rows8(rows=7)), dict(h=rows8(R, S, 4, 7)),
                                    dict(h=rows8(R, S, 3, 8)), dict(bias=R + 2), dict(act=0), dict(act=3)])
def test_gated8(change):
    refused(gated8(**change))


def fwd(x=P, residual=None, gamma=Q, total=None, y=R, rstd=None, rows=3, d=64, eps=1e-5):
    return capi.lib().rmsnorm_fwd(x, residual, gamma, total, y, rstd, rows, d, eps)


def bwd(s=P, gamma=Q, rstd=P, dy=P, dres=None, dx=R, dgamma=S, rows=3, d=64):
    return capi.lib().rmsnorm_bwd(s, gamma, rstd, dy, dres, dx, dgamma, rows, d)


@pytest.mark.parametrize("call", [fwd, bwd])
@pytest.mark.parametrize("change", [dict(gamma=None), dict(gamma=Q + 4), dict(rows=-1), dict(rows=2 ** 31), dict(d=0), dict(d=-4), dict(d=6)])
def test_norm(call, change):
    refused(call(**change))


@pytest.mark.parametrize("change", [dict(x=None), dict(x=P + 8), dict(residual=P + 4), dict(total=P + 8), dict(y=None), dict(y=R + 4), dict(rstd=P + 2),
                                    dict(total=R), dict(eps=-1e-5), dict(eps=math.inf), dict(eps=math.nan)])
def test_norm_forward(change):
    refused(fwd(**change))


@pytest.mark.parametrize("change", [dict(x=None), dict(x=P + 8), dict(residual=P + 4), dict(gamma=None), dict(total=P + 8), dict(eps=-1.0),
                                    dict(eps=math.nan), dict(y=rows8(cols=202))])
def test_norm_forward_in_8_bits(change):
    refused(norm8(**change))


@pytest.mark.parametrize("change", [dict(s=None), dict(rstd=None), dict(rstd=P + 2), dict(dy=None), dict(dy=P + 4), dict(dres=P + 8), dict(dx=None),
                                    dict(dgamma=None), dict(dgamma=S + 8)])
def test_norm_backward(change):
    refused(bwd(**change))


def test_rows_too_long_for_the_norm():
    refused(fwd(d=16388), UNSUPPORTED)
    refused(bwd(d=16388), UNSUPPORTED)
    refused(norm8(y=rows8(cols=16388)), UNSUPPORTED)


def gated_fwd(x=P, w=Q, bias=None, h=R, pre=None, n=2, hidden=3, d=4, act=1):
    return capi.lib().gated_fwd(x, w, bias, h, pre, n, hidden, d, act)


def gated_bwd(dy=P, w=Q, pre=S, dpre=R, n=2, hidden=3, d=4, act=1):
    return capi.lib().gated_bwd(dy, w, pre, dpre, n, hidden, d, act)


@pytest.mark.parametrize("call", [gated_fwd, gated_bwd])
@pytest.mark.parametrize("change", [dict(w=None), dict(w=Q + 2), dict(n=-1), dict(hidden=0), dict(hidden=2 ** 29), dict(d=0), dict(d=-3), dict(act=0),
                                    dict(act=3), dict(pre=P + 1)])
def test_gated(call, change):
    refused(call(**change))


@pytest.mark.parametrize("change", [dict(x=None), dict(x=P + 2), dict(h=None), dict(h=R + 1), dict(bias=P + 2)])
def test_gated_forward(change):
    refused(gated_fwd(**change))


@pytest.mark.parametrize("change", [dict(dy=None), dict(dy=P + 2), dict(pre=None), dict(dpre=None), dict(dpre=R + 1)])
def test_gated_backward(change):
    refused(gated_bwd(**change))


@pytest.mark.parametrize("name", ["rmsnorm_fwd", "rmsnorm_fwd8", "rmsnorm_bwd", "rows8_write", "rows8_read", "linear8_fwd", "gated_fwd", "gated_bwd",
                                  "gated8_fwd", "linear_fwd", "gemm_ex", "col_sum", "gelu_bwd", "gelu_bwd_col_sum", "layernorm_fwd",
                                  "layernorm_bwd", "mse_loss", "cross_entropy_loss"])
def test_arguments_are_declared(name):
    """Without declared types a device address would be passed in 32 bits."""
    import re

    with open(capi.HEADER) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    params = re.search(r"\bint " + name + r"\((.*?)\)", text, re.S).group(1).split(",")
    f = getattr(capi.lib(), name)
    assert len(f.argtypes) == len(params)
    for param, kind in zip(params, f.argtypes):
        size = 8 if "*" in param or "int64_t" in param else 4
        assert capi.C.sizeof(kind) == size, (name, param)

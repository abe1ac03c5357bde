"""Argument checks of the layer norm, checkpoint and linear-head loss entry points at the C ABI.  They come before any launch,
so they run without a GPU; the addresses are never followed."""
import ctypes as C

import pytest

from pacednegatives_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


A = 4096            # a 16-byte aligned address
ODD = 4096 + 2      # an element-aligned one


def refused(lib, rc, words):
    assert rc == -1 and words in lib.paced_last_error().decode(), (rc, lib.paced_last_error())


def ln_fwd(lib, **kw):
    a = dict(x=A, ldx=64, res=0, ldr=0, xsum=0, lds=0, w=A, b=A, y=A, ldy=64, mean=A, rstd=A, M=4, d=64, f32=0, eps=1e-5) | kw
    return lib.paced_layernorm_fwd(*a.values(), None)


def ln_bwd(lib, **kw):
    a = dict(dy=A, lddy=64, x=A, ldx=64, w=A, mean=A, rstd=A, dres=0, ldr=0, dx=A, lddx=64, dw=A, db=A, M=4, d=64, f32=0, ws=A, bytes=1 << 30) | kw
    return lib.paced_layernorm_bwd(*a.values(), None)


@pytest.mark.parametrize("kw,words", [(dict(d=8193), "[1, 8192]"), (dict(d=0), "[1, 8192]"), (dict(M=-1), "M >= 0"), (dict(x=0), "null"), (dict(b=0), "null"),
                                      (dict(res=A), "go together"), (dict(xsum=A), "go together"), (dict(ldx=63), "row strides"), (dict(ldy=0), "row strides"),
                                      (dict(res=A, xsum=A, ldr=64, lds=8), "row strides"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")])
def test_layernorm_fwd(lib, kw, words):
    refused(lib, ln_fwd(lib, **kw), words)


@pytest.mark.parametrize("kw,words", [(dict(d=9000), "[1, 8192]"), (dict(mean=0), "null"), (dict(dx=0), "null"), (dict(lddy=32), "row strides"), (dict(dres=A, ldr=1), "row strides"),
                                      (dict(ws=0), "workspace"), (dict(bytes=8), "workspace"), (dict(ws=ODD), "workspace")])
def test_layernorm_bwd(lib, kw, words):
    refused(lib, ln_bwd(lib, **kw), words)


@pytest.mark.parametrize("n,T,ldx,x,words", [(24, 8, 24, A, "multiple of 16"), (0, 8, 16, A, "multiple of 16"), (32, -1, 32, A, "T >= 0"), (32, 8, 16, A, "row stride"),
                                             (32, 8, 36, A, "row stride"), (32, 8, 32, ODD, "aligned"), (32, 8, 32, 0, "null")])
def test_act8_quantize_and_dequantize(lib, n, T, ldx, x, words):
    refused(lib, lib.paced_act8_quantize(x, ldx, A, A, T, n, None), words)
    refused(lib, lib.paced_act8_dequantize(A, A, x, ldx, T, n, None), words)


def dweight(lib, **kw):
    a = dict(dy=A, lddy=64, heads=0, q=A, scale=A, dw=A, lddw=32, T=100, M=64, N=32, acc=0, ws=A, bytes=1 << 40) | kw
    return lib.paced_act8_dweight(*a.values(), None)


@pytest.mark.parametrize("kw,words", [(dict(M=60), "multiple of 8"), (dict(N=24), "multiple of 16"), (dict(T=-1), "T >= 0"), (dict(dw=0), "dw must be"), (dict(dw=ODD), "dw must be"),
                                      (dict(lddw=30), "dw must be"), (dict(lddw=34), "dw must be"), (dict(q=ODD), "aligned"), (dict(dy=0), "aligned"), (dict(lddy=60), "row stride"),
                                      (dict(lddy=68), "row stride"), (dict(heads=64 * 99, lddy=64), "head-major"), (dict(heads=6400, lddy=72, M=64), "head-major"),
                                      (dict(T=5000, acc=1, ws=0), "workspace"), (dict(T=5000, acc=1, bytes=64), "workspace"), (dict(T=1 << 20, lddy=1 << 30, ws=A, bytes=1 << 60), "2 GiB")])
def test_act8_dweight(lib, kw, words):
    refused(lib, dweight(lib, **kw), words)


def ce_fwd(lib, **kw):
    a = dict(h=A, ldh=64, w=A, ldw=64, labels=A, loss=A, lse=A, R=8, V=100, d=64, ign=-100, scale=1.0, ws=A, bytes=1 << 40) | kw
    return lib.paced_linear_ce_fwd(*a.values(), None)


def ce_bwd(lib, **kw):
    a = dict(h=A, ldh=64, w=A, ldw=64, labels=A, lse=A, g=A, dh=A, lddh=64, dw=A, lddw=64, f32=0, R=8, V=100, d=64, ign=-100, scale=1.0, ws=A, bytes=1 << 40) | kw
    return lib.paced_linear_ce_bwd(*a.values(), None)


@pytest.mark.parametrize("kw,words", [(dict(d=96), "multiple of 64"), (dict(d=0), "multiple of 64"), (dict(V=0), "V > 0"), (dict(R=-1), "R >= 0"), (dict(h=0), "null"), (dict(labels=0), "null"),
                                      (dict(h=ODD), "aligned"), (dict(ldw=68), "multiples of 8"), (dict(ldh=56), "at least d"), (dict(ldh=1 << 23), "2^22"),
                                      (dict(ldw=1 << 23), "2^22")])
def test_linear_ce(lib, kw, words):
    refused(lib, ce_fwd(lib, **kw), words)
    refused(lib, ce_bwd(lib, **kw), words)


@pytest.mark.parametrize("kw,words", [(dict(loss=0), "null"), (dict(ws=0), "workspace"), (dict(bytes=100), "workspace"), (dict(ws=ODD), "workspace")])
def test_linear_ce_fwd(lib, kw, words):
    refused(lib, ce_fwd(lib, **kw), words)


@pytest.mark.parametrize("kw,words", [(dict(lse=0), "null"), (dict(g=0), "null"), (dict(dh=ODD), "dh needs"), (dict(lddh=60), "dh needs"), (dict(dw=ODD), "dw needs"), (dict(lddw=68), "dw needs"),
                                      (dict(ws=0), "workspace"), (dict(bytes=100), "workspace"), (dict(ws=ODD), "workspace"),
                                      (dict(R=1 << 21, ldh=1 << 11, d=64), "4 GiB"), (dict(ldw=1 << 26), "4 GiB")])
def test_linear_ce_bwd(lib, kw, words):
    refused(lib, ce_bwd(lib, **kw), words)


def test_empty_calls_are_no_errors_and_need_no_workspace(lib):
    assert lib.paced_layernorm_workspace_bytes(0, 64) == 0 and lib.paced_act8_dweight_workspace_bytes(0, 64, 32) == 0
    assert lib.paced_linear_ce_fwd_workspace_bytes(0, 100) == 0 and lib.paced_linear_ce_bwd_workspace_bytes(0, 100, 64) == 0
    assert ln_fwd(lib, M=0, x=0, y=0) == 0 and ln_bwd(lib, M=0, x=0) == 0
    assert lib.paced_act8_quantize(0, 32, 0, 0, 0, 32, None) == 0 and dweight(lib, T=0, acc=1, dy=0, q=0, scale=0, ws=0, bytes=0) == 0
    assert ce_fwd(lib, R=0, h=0) == 0 and ce_bwd(lib, R=0, h=0, f32=1) == 0


def test_workspaces_stay_bounded_as_the_vocabulary_grows(lib):
    for R in (1, 16, 1088, 8192, 65536):
        sizes = [lib.paced_linear_ce_bwd_workspace_bytes(R, V, 1024) for V in (100, 32128, 250000, 2000000)]
        assert max(sizes) <= (256 << 20) + max(96 << 20, R * 1024 * 4) + (64 << 20), (R, sizes)

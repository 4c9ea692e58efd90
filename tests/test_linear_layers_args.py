"""What the cross-entropy and INT8 linear entries refuse, all before any CUDA
call, and the sizes of their scratch memory."""
import ctypes as C

import pytest
import torch

from turboocr_b200 import linear_i8, rec_head

INVALID = 1
P = C.c_void_p(256)


def ce(lib, feat=P, w=P, targets=P, rows=4, K=64, V=10, dtype=0, loss=P, lse=P, ws=P,
       n=1 << 30, err=P):
    return lib.tocr_rec_head_ce(feat, w, None, targets, 0, rows, K, V, dtype, loss, lse, ws, n, err,
                                None)


def test_cross_entropy_refusals(tocr):
    lib = tocr.lib()
    for bad in (dict(K=12), dict(K=0), dict(K=264), dict(rows=-1), dict(rows=(1 << 24) + 1),
                dict(V=0), dict(dtype=2), dict(dtype=7), dict(feat=None), dict(w=None),
                dict(targets=None), dict(loss=None), dict(lse=None), dict(ws=None), dict(err=None),
                dict(feat=C.c_void_p(264)), dict(w=C.c_void_p(258)), dict(ws=C.c_void_p(272)),
                dict(n=16), dict(targets=C.c_void_p(258)), dict(loss=C.c_void_p(257)),
                dict(err=C.c_void_p(258))):
        assert ce(lib, **bad) == INVALID, bad
        assert tocr._lib.last_error()
    assert ce(lib, rows=0, feat=None, targets=None, ws=None) == 0


def ce_back(lib, feat=P, w=P, targets=P, rows=4, K=64, V=10, dtype=0, lse=P, g=P, dfeat=P, dw=P,
            db=P, ws=P, n=1 << 30, err=P):
    return lib.tocr_rec_head_ce_backward(feat, w, None, targets, 0, rows, K, V, dtype, lse, g, dfeat,
                                         dw, db, ws, n, err, None)


def test_cross_entropy_backward_refusals(tocr):
    lib = tocr.lib()
    for bad in (dict(K=12), dict(rows=-1), dict(V=0), dict(dtype=2), dict(feat=None), dict(w=None),
                dict(targets=None), dict(lse=None), dict(g=None), dict(ws=None), dict(err=None),
                dict(dfeat=C.c_void_p(264)), dict(dw=C.c_void_p(8)), dict(n=16),
                dict(g=C.c_void_p(258)), dict(lse=C.c_void_p(257)), dict(db=C.c_void_p(258))):
        assert ce_back(lib, **bad) == INVALID, bad
    assert ce_back(lib, dfeat=None, dw=None, db=None, feat=None, w=None) == 0
    assert ce_back(lib, rows=0, dw=None, db=None, feat=None, w=None) == 0


def test_workspace_sizes(tocr):
    f = tocr.lib().tocr_rec_head_ce_workspace_bytes
    assert f(-1, 64, 10, 0) == 0 and f(4, 12, 10, 0) == 0 and f(4, 64, 0, 1) == 0
    assert 0 < f(100, 64, 10, 0) < f(100000, 64, 10, 0)
    assert f(100000, 64, 10, 1) > 100000 * 64 * 2
    g = tocr.lib().tocr_linear_i8_workspace_bytes
    assert g(-1, 64) == 0 and g(4, 0) == 0
    assert g(1, 512) == 0                       # few tokens need none
    assert g(4096, 100) >= 4096 * (112 + 4)


def linear(lib, x=P, xt=0, rows=4, K=64, wq=P, sw=P, N=10, act=0, yt=0, y=P, ws=P, n=1 << 30, err=P):
    return lib.tocr_linear_i8(x, xt, rows, K, wq, sw, None, N, act, yt, y, ws, n, err, None)


def test_linear_refusals(tocr):
    lib = tocr.lib()
    many = dict(rows=5000)
    for bad in (dict(rows=-1), dict(rows=(1 << 24) + 1), dict(K=0), dict(K=(1 << 17) + 1), dict(N=0),
                dict(act=3), dict(act=-1), dict(xt=3), dict(yt=-1), dict(x=None), dict(wq=None),
                dict(sw=None), dict(y=None), dict(err=None), dict(wq=C.c_void_p(264)),
                dict(x=C.c_void_p(257)), dict(y=C.c_void_p(257)), dict(x=C.c_void_p(258), xt=2),
                dict(sw=C.c_void_p(258)), dict(err=C.c_void_p(257)),
                dict(ws=None, **many), dict(ws=C.c_void_p(272), **many), dict(n=16, **many)):
        assert linear(lib, **bad) == INVALID, bad
    assert linear(lib, rows=0, x=None, y=None) == 0
    q = lib.tocr_quant_rows_i8
    assert q(P, 0, -1, 64, P, P, None) == INVALID
    assert q(P, 5, 4, 64, P, P, None) == INVALID
    assert q(P, 0, 4, 64, C.c_void_p(8), P, None) == INVALID
    assert q(None, 0, 4, 64, P, P, None) == INVALID
    assert q(None, 0, 0, 64, None, None, None) == 0
    c = lib.tocr_linear_i8_codes
    assert c(P, P, 4, 64, P, P, None, 10, 0, 0, None, P, None) == INVALID
    assert c(C.c_void_p(8), P, 4, 64, P, P, None, 10, 0, 0, P, P, None) == INVALID
    assert c(None, None, 0, 64, P, P, None, 10, 0, 0, None, P, None) == 0


def test_injected_errors(tocr):
    lib = tocr.lib()
    lib.tocr_debug_inject_error(5, 2)
    try:
        assert ce(lib) == 5 and linear(lib) == 5
    finally:
        lib.tocr_debug_inject_error(0, 0)


def test_tensors_refused():
    f, w = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(10, 64, dtype=torch.float16)
    t, e = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        rec_head.cross_entropy(f, w, None, t, err=e)
    with pytest.raises(ValueError, match="features are"):
        rec_head.cross_entropy(f[0], w, None, t, err=e)
    with pytest.raises(ValueError, match="weight must have shape"):
        rec_head.cross_entropy(f, w[:, :32], None, t, err=e)
    with pytest.raises(ValueError, match="targets must have shape"):
        rec_head.cross_entropy(f, w, None, t[:2], err=e)
    with pytest.raises(ValueError, match="CUDA device"):
        linear_i8.quantize_rows(f)
    with pytest.raises(ValueError, match="x is"):
        linear_i8.linear(f[0], w, e, err=e)
    assert linear_i8.pitch(1) == 16 and linear_i8.pitch(16) == 16 and linear_i8.pitch(1001) == 1008


def test_codes_whose_sum_could_pass_32_bits(tocr):
    """128^2 * 2^17 is 2^31: one feature more than the sums of any codes have room for."""
    c = tocr.lib().tocr_linear_i8_codes
    assert c(P, P, 4, 1 << 17, P, P, None, 10, 0, 0, P, P, None) == INVALID
    assert tocr._lib.last_error()
    assert 128 ** 2 * ((1 << 17) - 1) < 1 << 31
    assert c(None, None, 0, (1 << 17) - 1, P, P, None, 10, 0, 0, None, P, None) == 0
    assert tocr.lib().tocr_linear_i8_workspace_bytes(100, 1 << 17) > 100 << 17


def test_more_classes_than_the_calls_take(tocr):
    """The workspace function gives 0 for sizes that the calls refuse."""
    lib = tocr.lib()
    f = lib.tocr_rec_head_ce_workspace_bytes
    most = 1 << 24
    for back in (0, 1):
        assert f(4, 64, most, back) > 0 and f(4, 64, most + 1, back) == 0
        assert f(4, 64, (1 << 31) - 1, back) == 0
    assert ce(lib, V=most + 1) == INVALID and ce_back(lib, V=most + 1) == INVALID


@pytest.mark.parametrize("which", [0, 1, 2])
def test_cross_entropy_of_tensors_that_require_grad(which):
    """It builds no graph, so it says so; under no_grad, and detached, the call is
    as any other (here it gets as far as the device check)."""
    x = [torch.zeros(4, 64, dtype=torch.float16), torch.zeros(10, 64, dtype=torch.float16),
         torch.zeros(10)]
    t, e = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x[which].requires_grad_()
    with pytest.raises(ValueError, match="no graph"):
        rec_head.cross_entropy(*x, t, err=e)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
        rec_head.cross_entropy(*x, t, err=e)
    with pytest.raises(ValueError, match="CUDA device"):
        rec_head.cross_entropy(*(y.detach() for y in x), t, err=e)

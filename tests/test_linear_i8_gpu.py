"""The INT8 linear layer (turboocr_b200.linear_i8) against its definition in 64
bits. Codes and scales must be equal. The sum of the products of codes is
exact; behind it come the conversion to fp32 (2^-24, exact below 2^24), two
products, the bias and the activation in fp32 (each at most 2^-24 of the
largest term: 8 * 2^-24 together) and one rounding to the output type (half a
step of the value, or half of the least subnormal)."""
import math

import pytest
import torch

from turboocr_b200 import linear_i8

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def quantized(x):
    """Codes (fp64) and fp32 scales by the definition. The fp64 quotient of two
    fp32 numbers is a tie only where the exact one is: q + 1/2 and its
    neighbours in reach differ by far more than 2^-45."""
    x32 = x.float()
    top = x32.abs().amax(1).cpu().double()
    s = (top * torch.tensor(1 / 127).double()).float().clamp_min(2.0 ** -126).to(x.device)
    bad = ~torch.isfinite(x32).all(1)
    q = torch.round(x32.double() / s.double()[:, None])
    q[bad] = 0
    s[bad] = math.nan
    return q, s


def act64(y, act):
    if act == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if act == "hardswish":
        return y * (y + 3).clamp(0, 6) / 6
    return y


def check(x, w, bias, act, out, err):
    K = x.shape[1]
    wq, ws = linear_i8.quantize_rows(w)
    q, s = quantized(w)
    assert torch.equal(wq[:, :K].double(), q) and torch.equal(ws, s)
    assert int(wq[:, K:].abs().sum()) == 0
    xq, sx = linear_i8.quantize_rows(x)
    qx, s2 = quantized(x)
    assert torch.equal(xq[:, :K].double(), qx) and torch.equal(sx, s2)
    assert int(xq[:, K:].abs().sum()) == 0
    y = linear_i8.linear(x, wq, ws, bias, act=act, out_dtype=out, err=err)
    y2 = linear_i8.linear_codes(xq, sx, K, wq, ws, bias, act=act, out_dtype=out, err=err)
    torch.cuda.synchronize()
    assert int(err) == 0
    assert torch.equal(y, y2)
    z = (qx @ q.T) * s2.double()[:, None] * s.double()
    b = bias.double() if bias is not None else 0.0
    want = act64(z + b, act)
    # the activation's slope is at most 1.5; hardswish multiplies by up to |z + b|
    mag = (z.abs() + (bias.abs().double() if bias is not None else 0.0)) * 1.5
    u = torch.finfo(out).eps / 2
    tiny = torch.finfo(out).smallest_normal * torch.finfo(out).eps / 2
    tol = 8 * 2.0 ** -24 * mag + u * want.abs() + tiny
    d = (y.double() - want).abs()
    assert bool((d <= tol).all()), float((d / tol).max())
    return y


SIZES = [(1, 1, 1), (1, 512, 18385), (3, 17, 5), (80, 128, 384), (127, 100, 130), (129, 260, 255),
         (128, 261, 64), (200, 1001, 257), (2560, 256, 1024), (5, 5000, 33), (1000, 64, 2049),
         (257, 2048, 16), (33, 8200, 100)]


@pytest.mark.parametrize("xt,yt", [(F16, F16), (BF16, BF16), (F32, F32), (F16, F32), (F32, BF16)])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_linear(tocr, cuda, rows, K, N, xt, yt):
    g = torch.Generator(device="cpu").manual_seed(rows + 31 * K + 7 * N)
    gain = torch.exp(torch.randn(K, generator=g))
    x = (torch.randn(rows, K, generator=g) * gain).to(xt).to(cuda)
    w = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(cuda)
    bias = torch.randn(N, generator=g).to(cuda) if (rows + N) % 2 else None
    act = ["none", "relu", "hardswish"][(rows + K + N) % 3]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    check(x, w, bias, act, yt, err)


@pytest.mark.parametrize("rows,K,N,out", [(2100, 40, 18385, F16), (1000, 33, 18387, F32),
                                          (8400, 300, 4099, BF16), (37, 16, 1000003, F16),
                                          (70001, 16, 500, F16)])
def test_outputs_larger_than_l2(tocr, cuda, rows, K, N, out):
    """Outputs of more than 64 MB whose rows are not sector-aligned take their
    own way out of the kernel."""
    g = torch.Generator(device="cpu").manual_seed(rows)
    x = torch.randn(rows, K, generator=g).half().to(cuda)
    w = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(cuda)
    bias = torch.randn(N, generator=g).to(cuda)
    check(x, w, bias, "none", out, torch.zeros(1, dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("rows,N,out", [(2100, 18385, F16), (2100, 18384, BF16), (130, 77, F16),
                                        (1100, 16385, F32)])
def test_output_at_any_element_and_nothing_written_around_it(tocr, cuda, rows, N, out):
    K, pad = 48, 67
    g = torch.Generator(device="cpu").manual_seed(N)
    x = torch.randn(rows, K, generator=g).half().to(cuda)
    w = torch.randn(N, K, generator=g).to(cuda)
    wq, ws = linear_i8.quantize_rows(w)
    xq, sx = linear_i8.quantize_rows(x)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    want = linear_i8.linear_codes(xq, sx, K, wq, ws, None, out_dtype=out, err=err)
    for off in (0, 1, 3, 8):
        buf = torch.full((pad + off + rows * N + pad,), -7.0, dtype=out, device=cuda)
        at = buf.data_ptr() + (pad + off) * buf.element_size()
        st = tocr.lib().tocr_linear_i8_codes(
            xq.data_ptr(), sx.data_ptr(), rows, K, wq.data_ptr(), ws.data_ptr(), None, N, 0,
            {F16: 0, BF16: 1, F32: 2}[out], at, err.data_ptr(),
            torch.cuda.current_stream().cuda_stream)
        assert st == 0
        assert torch.equal(buf[pad + off:pad + off + rows * N].view(rows, N), want), off
        assert bool((buf[:pad + off] == -7).all()) and bool((buf[pad + off + rows * N:] == -7).all())
    assert int(err) == 0


@pytest.mark.parametrize("rows", [5, 600])   # few tokens and many take different kernels
@pytest.mark.parametrize("xt", [F16, BF16, F32])
def test_rows_of_any_numbers(tocr, cuda, rows, xt):
    """Zero rows, rows of the least and the largest numbers, rows whose quotients
    are ties, and rows with an infinity or a NaN (NaN outputs, the others as
    without them)."""
    K, N = 96, 130
    g = torch.Generator(device="cpu").manual_seed(rows)
    x = torch.randn(rows, K, generator=g).to(xt)
    x[0] = 0
    x[1] = torch.finfo(xt).smallest_normal * torch.finfo(xt).eps * torch.randint(-9, 10, (K,)).to(xt)
    x[2] = torch.finfo(xt).max * (torch.rand(K, generator=g) * 2 - 1).to(xt)
    x[3] = torch.arange(K).to(xt) / 2           # half of the maximum is a tie
    x[4] = (torch.arange(K) % 3 - 1).to(xt) * 12.7
    w = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(cuda)
    w[7] = 0
    bias = torch.randn(N, generator=g).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    x = x.to(cuda)
    check(x[torch.arange(rows) != 2].contiguous(), w, bias, "none", F32, err)
    y = check(x, w * 1e-3, bias, "none", F32, err)
    assert torch.equal(y[0], bias)
    bad = x.clone()
    bad[1, 5], bad[4, 95] = math.inf, math.nan
    wq, ws = linear_i8.quantize_rows(w * 1e-3)
    codes, scales = linear_i8.quantize_rows(bad)
    assert bool(torch.isnan(scales[[1, 4]]).all()) and int(codes[[1, 4]].abs().sum()) == 0
    for act in ("none", "relu", "hardswish"):
        z = linear_i8.linear(bad, wq, ws, bias, act=act, out_dtype=F32, err=err)
        ref = linear_i8.linear(x, wq, ws, bias, act=act, out_dtype=F32, err=err)
        assert bool(torch.isnan(z[[1, 4]]).all())
        rest = [r for r in range(rows) if r not in (1, 4)]
        assert torch.equal(z[rest], ref[rest])
    assert int(err) == 0


def test_weights_with_a_nan_channel(tocr, cuda):
    w = torch.randn(40, 64, device=cuda)
    w[3, 3] = math.nan
    wq, ws = linear_i8.quantize_rows(w)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    for rows in (3, 700):
        y = linear_i8.linear(torch.randn(rows, 64, device=cuda), wq, ws, None, err=err)
        assert bool(torch.isnan(y[:, 3]).all())
        assert bool(torch.isfinite(y[:, :3]).all()) and bool(torch.isfinite(y[:, 4:]).all())


def test_few_tokens_border(tocr, cuda):
    """Sizes at both sides of the rule that has the product quantise its tokens."""
    g = torch.Generator(device="cpu").manual_seed(2)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    for rows, K, N in ((128, 256, 300), (129, 250, 300), (128, 257, 300), (17, 1900, 5),
                       (16, 2048, 20000), (8, 4096, 129), (1, 4097, 128), (1, 32768, 40),
                       (1, 40000, 40), (3, 13, 19000)):
        x = torch.randn(rows, K, generator=g).to(BF16).to(cuda)
        w = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(cuda)
        check(x, w, None, "relu", BF16, err)


@pytest.mark.parametrize("rows,K,N", [(3, 17, 5), (300, 17, 40), (130, 256, 33), (130, 260, 200),
                                      (2100, 41, 18385)])
def test_codes_of_any_origin(tocr, cuda, rows, K, N):
    """All of int8, the code -128 and its largest sums among them, and anything
    behind K. With scales of 1 the sums come out exactly (K 128^2 < 2^24)."""
    g = torch.Generator(device="cpu").manual_seed(rows + K + N)
    P = linear_i8.pitch(K)
    xq = torch.randint(-128, 128, (rows, P), generator=g, dtype=torch.int8)
    wq = torch.randint(-128, 128, (N, P), generator=g, dtype=torch.int8)
    xq[0], wq[0], wq[1] = -128, -128, 127
    xq, wq = xq.to(cuda), wq.to(cuda)
    one = torch.ones(max(rows, N), device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    y = linear_i8.linear_codes(xq, one[:rows], K, wq, one[:N], None, out_dtype=F32, err=err)
    want = xq[:, :K].double() @ wq[:, :K].double().T
    assert int(err) == 0
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("rows", [5, 300])
def test_weights_with_anything_behind_their_features(tocr, cuda, rows):
    g = torch.Generator(device="cpu").manual_seed(rows)
    x = torch.randn(rows, 21, generator=g).to(cuda)
    wq, ws = linear_i8.quantize_rows(torch.randn(50, 21, generator=g).to(cuda))
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    a = linear_i8.linear(x, wq, ws, err=err)
    wq[:, 21:] = 99
    assert torch.equal(a, linear_i8.linear(x, wq, ws, err=err))
    assert int(err) == 0


def test_empty_and_other_streams_and_graphs(tocr, cuda):
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    w = torch.randn(500, 200, device=cuda)
    wq, ws = linear_i8.quantize_rows(w)
    assert linear_i8.linear(torch.zeros(0, 200, device=cuda), wq, ws, err=err).shape == (0, 500)
    assert linear_i8.quantize_rows(torch.zeros(0, 200, device=cuda))[0].shape == (0, 208)
    xs = [torch.randn(r, 200, device=cuda, dtype=F16) for r in (3, 900)]
    want = [linear_i8.linear(x, wq, ws, err=err) for x in xs]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [linear_i8.linear(x, wq, ws, err=err, stream=s) for _ in range(8)
           for x, s in zip(xs, (s1, s2))]
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert torch.equal(y, want[k % 2])
    held = [x.clone() for x in xs]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = [linear_i8.linear(x, wq, ws, err=err) for x in held]
    for x in held:
        x.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    for x, y in zip(held, out):
        assert torch.equal(y, linear_i8.linear(x, wq, ws, err=err))
    assert int(err) == 0


def test_output_beyond_32_bits(tocr, cuda):
    rows, K, N = 120001, 32, 18385             # 4.4 GB of fp16
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.randn(rows, K, generator=g, device=cuda, dtype=F16)
    wq, ws = linear_i8.quantize_rows(torch.randn(N, K, generator=g, device=cuda))
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    y = linear_i8.linear(x, wq, ws, None, err=err)
    for at in (slice(0, 300), slice(116700, 117000), slice(rows - 300, rows)):
        part = linear_i8.linear(x[at].contiguous(), wq, ws, None, err=err)
        assert torch.equal(y[at], part)
    y = linear_i8.linear(x, wq[:18368].contiguous(), ws[:18368].contiguous(), None, err=err)
    assert torch.equal(y[-300:], linear_i8.linear(x[-300:].contiguous(), wq, ws, None,
                                                  err=err)[:, :18368])
    assert int(err) == 0


@pytest.mark.parametrize("rows,N", [(300, 640), (2100, 18385)])
def test_one_workspace_for_call_after_call(tocr, cuda, rows, N):
    """Calls in a row on one stream with the same scratch memory, whose scales and
    codes the product reads while it may already have begun beside the quantiser:
    each has the bits of a call by itself."""
    K = 200
    g = torch.Generator(device="cpu").manual_seed(rows)
    xs = [(torch.randn(rows, K, generator=g) * 4.0 ** k).half().to(cuda) for k in range(3)]
    wq, ws = linear_i8.quantize_rows((torch.randn(N, K, generator=g) / math.sqrt(K)).to(cuda))
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    want = [linear_i8.linear(x, wq, ws, err=err) for x in xs]
    n = tocr.lib().tocr_linear_i8_workspace_bytes(rows, K)
    buf = torch.zeros(n, dtype=torch.uint8, device=cuda)
    got = [torch.empty_like(y) for y in want * 4]
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert tocr.lib().tocr_linear_i8(
            xs[k % 3].data_ptr(), 0, rows, K, wq.data_ptr(), ws.data_ptr(), None, N, 0, 0,
            y.data_ptr(), buf.data_ptr(), n, err.data_ptr(),
            torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert torch.equal(y, want[k % 3]), k
    assert int(err) == 0


def test_longest_sums_of_any_codes(tocr, cuda):
    """The largest sums, of either sign, at the longest rows of codes: exact to the
    one rounding to fp32."""
    K = (1 << 17) - 1
    xq = torch.full((40, K + 1), -128, dtype=torch.int8, device=cuda)
    wq = torch.full((6, K + 1), -128, dtype=torch.int8, device=cuda)
    wq[1::2] = 127
    xq[5, ::2] = 127
    one = torch.ones(40, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    y = linear_i8.linear_codes(xq, one, K, wq, one[:6].contiguous(), None, out_dtype=F32, err=err)
    assert int(err) == 0
    assert torch.equal(y, (xq[:, :K].double() @ wq[:, :K].double().T).float())
    with pytest.raises(ValueError):
        linear_i8.linear_codes(xq, one, K + 1, wq, one[:6].contiguous(), None, out_dtype=F32, err=err)

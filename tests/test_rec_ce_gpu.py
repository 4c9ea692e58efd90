"""Cross entropy of the recognizer's head and its gradient
(turboocr_b200.rec_head) against the definition in 64 bits on the same 16-bit
inputs.

Tolerances, all derived from the arithmetic (u = half a step of the type):
- a logit: K exact products summed in fp32, (K + 2) 2^-23 sum_k |x_k w_k| (the
  tensor cores may truncate, hence 2^-23 and not 2^-24);
- loss and lse: that, plus the rounding of y = l log2(e) + b log2(e) (three
  fp32 roundings of numbers up to 1.5 max|l|), plus the fp32 sum, exp2 and log
  (2^-18 in all);
- a gradient: each term G_ij w_jk is off by the rounding of G to 16 bits (u),
  by the relative error of exp(l - lse) (twice the logit's error) and by the
  fp32 sum of n terms (n 2^-24), all relative to the sum of |terms|; the result
  is rounded once to 16 bits (u of it, and half of the least subnormal);
  fp16 terms below 2^-28 of the largest weight are off by 2^-39 of it;
- dbias: as a gradient, without the 16-bit roundings."""
import math

import pytest
import torch

from turboocr_b200 import rec_head

pytestmark = pytest.mark.gpu


def make(rows, K, V, dtype, seed, dev, pad=0.0, bias=True, gain=3.0, wide=False):
    g = torch.Generator(device="cpu").manual_seed(seed)
    feat = torch.randn(rows, K, generator=g)
    w = (torch.randn(V, K, generator=g) * (gain / math.sqrt(K))).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g)
    t = torch.where(torch.rand(rows, generator=g) < 0.3, torch.zeros_like(t), t)
    known = torch.rand(rows, generator=g) < 0.4
    feat = torch.where(known[:, None], w[t].float() * (math.sqrt(K) / gain) + 0.3 * feat, feat)
    t = torch.where(torch.rand(rows, generator=g) < pad, torch.full_like(t, -1), t)
    b = (torch.randn(V, generator=g) * 0.5).to(dev) if bias else None
    gl = (torch.rand(rows, generator=g) * 2 - 0.5).to(dev)
    return (feat.to(dtype).to(dev), w.to(dev), b,
            t.to(torch.int64 if wide else torch.int32).to(dev), gl)


def exact(feat, w, b, t, gl):
    """The definition in fp64; per output (value, tolerance)."""
    V, K = w.shape
    u = torch.finfo(feat.dtype).eps / 2
    tiny = torch.finfo(feat.dtype).smallest_normal * torch.finfo(feat.dtype).eps / 2
    keep = (t >= 0) & (t < V)
    x = torch.where(keep[:, None], feat.double(), torch.zeros((), dtype=torch.float64,
                                                              device=feat.device))
    wd = w.double()
    tt = torch.where(keep, t, torch.zeros_like(t)).long()[:, None]
    l = x @ wd.T
    if b is not None:
        l = l + b.double()
    lse = torch.logsumexp(l, 1)
    loss = lse - l.gather(1, tt)[:, 0]
    mag = (x.abs() @ wd.abs().T).amax(1)
    big = l.masked_fill(torch.isinf(l), 0).abs().amax(1)
    tl = (K + 2) * 2.0 ** -23 * mag + 6 * 2.0 ** -24 * 1.5 * big + 2.0 ** -18
    k = keep.double()
    out = {"loss": (loss.masked_fill(~keep, 0), 2 * tl * k), "lse": (lse * k, 2 * tl * k)}
    gr = gl.double() * k
    p = torch.exp(l - lse[:, None])
    G = p.clone().scatter_add_(1, tt, torch.full_like(tt, -1, dtype=torch.float64))
    G = torch.where(keep[:, None], G * gr[:, None], torch.zeros_like(G))
    # |error| of G before its rounding to 16 bits
    dG = p * (3 * tl)[:, None] * gr.abs()[:, None] + G.abs() * 2.0 ** -22
    gm = float(gr.abs().max()) if gr.numel() else 0.0
    floor = gm * 2.0 ** -39 if feat.dtype == torch.float16 else gm * 1e-38
    n = int(keep.sum())
    eG = dG + u * G.abs() + floor * k[:, None]
    df = G @ wd
    dw = G.T @ x
    out["dfeat"] = (df, (eG + V * 2.0 ** -24 * G.abs()) @ wd.abs() + u * df.abs() + tiny)
    out["dweight"] = (dw, (eG + n * 2.0 ** -24 * G.abs()).T @ x.abs() + u * dw.abs() + tiny)
    out["dbias"] = (G.sum(0), (dG + (n + 2) * 2.0 ** -24 * G.abs()).sum(0) + 1e-30)
    return out


def run(feat, w, b, t, gl, dev, **kw):
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    loss, lse = rec_head.cross_entropy(feat, w, b, t, err=err)
    df, dw, db = rec_head.cross_entropy_backward(feat, w, b, t, lse, gl, err=err, **kw)
    torch.cuda.synchronize()
    assert int(err) == 0
    return {"loss": loss, "lse": lse, "dfeat": df, "dweight": dw, "dbias": db}


def near(got, want, names=("loss", "lse", "dfeat", "dweight", "dbias")):
    for name in names:
        if got[name] is None:
            continue
        v, tol = want[name]
        d = (got[name].double() - v).abs()
        assert bool(torch.isfinite(got[name]).all()), name
        worst = float((d / tol.clamp_min(1e-300)).max()) if d.numel() else 0.0
        assert bool((d <= tol).all()), (name, worst, float(d.max()))


SIZES = [(1, 8, 1), (1, 128, 18385), (5, 16, 7), (127, 64, 129), (128, 128, 128), (129, 72, 257),
         (300, 200, 1000), (513, 256, 2049), (80, 120, 6625), (2000, 136, 5000), (257, 192, 20000),
         (30000, 64, 300)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,K,V", SIZES)
def test_loss_and_gradients(tocr, cuda, rows, K, V, dtype):
    a = make(rows, K, V, dtype, 7 * rows + K + V, cuda, pad=0.0 if rows < 8 else 0.3,
             bias=(rows + K) % 3 != 0, wide=V % 2 == 0)
    near(run(*a, cuda), exact(*a))


def err_word(dev):
    return torch.zeros(1, dtype=torch.int32, device=dev)


def check(a, cuda, **kw):
    near(run(*a, cuda, **kw), exact(*a))


@pytest.mark.parametrize("want", ["all", "feat", "weight", "bias"])
@pytest.mark.parametrize("rows,K,V", [(40, 256, 30000), (80, 128, 18385), (40000, 128, 100),
                                      (20000, 200, 130), (700, 64, 9000)])
def test_tiles_in_many_pieces(tocr, cuda, rows, K, V, want):
    """Few rows or few classes: one tile is cut by most of the ranges' borders."""
    a = make(rows, K, V, torch.bfloat16, rows + V, cuda, bias=True)
    kw = {} if want == "all" else {f"need_{n}": n == want for n in ("feat", "weight", "bias")}
    near(run(*a, cuda, **kw), exact(*a))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_padding_rows_cost_and_reach_nothing(tocr, cuda, dtype):
    """NaN and infinities in padding rows leave every output as it is with zeros
    there, bit for bit; their own outputs are zero."""
    f, w, b, t, gl = make(700, 72, 3001, dtype, 5, cuda, pad=0.4, wide=True)
    pad = torch.nonzero(t < 0).flatten()
    t[pad[::3]] = 3001
    t[pad[1::3]] = 2 ** 40 + 7
    t[pad[2::3]] = -100
    clean = f.clone()
    clean[pad] = 0
    f[pad[::2]] = float("nan")
    f[pad[1::2]] = float("inf")
    gl2 = gl.clone()
    gl2[pad] = float("nan")
    one, two = run(f, w, b, t, gl2, cuda), run(clean, w, b, t, gl, cuda)
    for k in one:
        assert torch.equal(one[k], two[k]), k
    for k in ("loss", "lse"):
        assert bool((one[k][pad] == 0).all())
    assert bool((one["dfeat"][pad] == 0).all())
    near(two, exact(clean, w, b, t, gl))


@pytest.mark.parametrize("rows", [0, 1, 300])
def test_no_row_with_a_target(tocr, cuda, rows):
    f, w, b, t, gl = make(rows, 64, 500, torch.float16, 9, cuda)
    t.fill_(-1)
    got = run(f, w, b, t, gl, cuda)
    for k, v in got.items():
        assert v.shape[0] == (500 if k in ("dweight", "dbias") else rows)
        assert bool((v == 0).all()), k


def test_masked_classes(tocr, cuda):
    """A bias of -inf takes a class out: probability and gradients zero, an
    infinite loss where it is the target; a row all of whose classes are masked
    is NaN, others are untouched by it."""
    f, w, b, t, gl = make(200, 64, 700, torch.bfloat16, 21, cuda)
    b[::3] = -math.inf
    b[:130] = -math.inf      # whole columns groups at the start of the vocabulary
    t = torch.where(torch.isinf(b[t.long()]), torch.full_like(t, 131), t)
    t[5] = 0                 # masked
    got = run(f, w, b, t, gl, cuda)
    assert got["loss"][5] == math.inf
    keep = torch.ones_like(t, dtype=torch.bool)
    keep[5] = False
    t2 = torch.where(keep, t, torch.full_like(t, -1))
    two = run(f, w, b, t2, gl, cuda)
    near(two, exact(f, w, b, t2, gl))
    masked = torch.isinf(b)
    assert bool((two["dweight"][masked] == 0).all()) and bool((two["dbias"][masked] == 0).all())
    all_out = run(f, w, torch.full_like(b, -math.inf), t, gl, cuda)
    assert bool(torch.isnan(all_out["loss"]).all())


@pytest.mark.parametrize("kind", ["far below", "far above", "rising", "falling", "spread"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_logits_of_any_size(tocr, cuda, kind, dtype):
    V = 2500
    f, w, b, t, gl = make(300, 128, V, dtype, 31, cuda)
    ramp = torch.linspace(-900, 900, V, device=cuda)
    if kind == "far below":
        b = b - 5000
    elif kind == "far above":
        b = b + 5000
    elif kind == "rising":
        b = b + ramp
    elif kind == "falling":
        b = b - ramp
    else:
        f = (f.float() * 40).to(dtype)
    check((f, w, b, t, gl), cuda)


def test_infinite_and_nan_rows_stay_their_own(tocr, cuda):
    """A row of features with a NaN has a NaN loss and gradient; the other rows'
    losses and gradients are as without it."""
    f, w, b, t, gl = make(130, 64, 900, torch.float16, 41, cuda)
    f2 = f.clone()
    f2[7, 3] = float("nan")
    f2[129, 0] = float("inf")
    one, two = run(f, w, b, t, gl, cuda), run(f2, w, b, t, gl, cuda)
    bad = torch.zeros(130, dtype=torch.bool, device=cuda)
    bad[7] = bad[129] = True
    assert not bool(torch.isfinite(two["loss"][bad]).any())
    for k in ("loss", "lse", "dfeat"):
        assert torch.equal(one[k][~bad], two[k][~bad]), k
    assert bool(torch.isnan(two["dweight"]).any())


def test_gradients_against_differences(tocr, cuda):
    """Directional derivatives: the kernels' gradients times a direction against
    central differences of the 64-bit loss (step 1e-4: truncation below 1e-7 of
    the direction's norm, rounding below 1e-11), within what the entries'
    tolerances add up to."""
    a = make(60, 48, 400, torch.float16, 51, cuda, pad=0.2)
    f, w, b, t, gl = a
    got, want = run(*a, cuda), exact(*a)
    keep = (t >= 0).double()
    at = t.clamp_min(0).long()[:, None]

    def loss(x, ww, bb):
        l = x @ ww.T + bb
        return ((torch.logsumexp(l, 1) - l.gather(1, at)[:, 0]) * gl.double() * keep).sum()

    g = torch.Generator(device=cuda).manual_seed(3)
    p = [f.double(), w.double(), b.double()]
    for k, name in enumerate(("dfeat", "dweight", "dbias")):
        d = torch.randn(p[k].shape, generator=g, device=cuda, dtype=torch.float64)
        up = [q + 1e-4 * d if i == k else q for i, q in enumerate(p)]
        down = [q - 1e-4 * d if i == k else q for i, q in enumerate(p)]
        diff = (loss(*up) - loss(*down)) / 2e-4
        tol = (want[name][1] * d.abs()).sum() + 1e-5 * d.norm()
        assert abs(float((got[name].double() * d).sum() - diff)) <= float(tol), name


def test_parts_of_the_gradient(tocr, cuda):
    f, w, b, t, gl = make(257, 120, 1500, torch.float16, 61, cuda, pad=0.1)
    whole = run(f, w, b, t, gl, cuda)
    err = err_word(cuda)
    for nf in (False, True):
        for nw in (False, True):
            for nb in (False, True):
                got = rec_head.cross_entropy_backward(f, w, b, t, whole["lse"], gl, err=err,
                                                      need_feat=nf, need_weight=nw, need_bias=nb)
                for v, name, need in zip(got, ("dfeat", "dweight", "dbias"), (nf, nw, nb)):
                    assert (v is None) == (not need)
                    if need:
                        near({name: v}, exact(f, w, b, t, gl), (name,))
    assert int(err) == 0


def test_same_inputs_same_bits_and_streams(tocr, cuda):
    a = make(1300, 128, 6000, torch.bfloat16, 71, cuda, pad=0.2)
    c = make(900, 64, 2000, torch.float16, 72, cuda)
    wa, wc = run(*a, cuda), run(*c, cuda)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    err = err_word(cuda)
    torch.cuda.synchronize()
    out = []
    for _ in range(4):  # two calls at once, each with its own scratch
        for s, (f, w, b, t, gl) in ((s1, a), (s2, c)):
            loss, lse = rec_head.cross_entropy(f, w, b, t, err=err, stream=s)
            g = rec_head.cross_entropy_backward(f, w, b, t, lse, gl, err=err, stream=s)
            out.append((loss, lse, *g))
    torch.cuda.synchronize()
    assert int(err) == 0
    for k, o in enumerate(out):
        for v, want in zip(o, (wa if k % 2 == 0 else wc).values()):
            assert torch.equal(v, want)


def test_captured_and_replayed(tocr, cuda):
    """Two captured graphs replayed in turn and at once, on changing inputs."""
    sets = [make(400, 128, 3000, torch.float16, s, cuda, pad=0.3) for s in (81, 82, 83)]
    want = [run(*s, cuda) for s in sets]
    err = err_word(cuda)
    graphs = []
    for _ in range(2):
        held = [x.clone() for x in sets[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            rec_head.cross_entropy(held[0], held[1], held[2], held[3], err=err)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, lse = rec_head.cross_entropy(held[0], held[1], held[2], held[3], err=err)
            grads = rec_head.cross_entropy_backward(held[0], held[1], held[2], held[3], lse,
                                                    held[4], err=err)
        graphs.append((g, held, (loss, lse, *grads)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in (1, 2, 0):
        for j, (g, held, _) in enumerate(graphs):
            for x, y in zip(held, sets[(k + j) % 3]):
                x.copy_(y)
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for j, (_, _, out) in enumerate(graphs):
            for v, w in zip(out, want[(k + j) % 3].values()):
                assert torch.equal(v, w)
    assert int(err) == 0


def test_targets_from_the_serving_head(tocr, cuda):
    """The step indices that the fused head writes are targets as they are, and
    exp(-loss) is the probability that it gives them (its own tolerance: 1e-4)."""
    B, T, K, V = 6, 40, 128, 18385
    f, w, b, _, _ = make(B * T, K, V, torch.float16, 91, cuda)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=cuda)
    toks, lens, idx, err = i32(B * T), i32(B), i32(B * T), err_word(cuda)
    sc, prob = torch.zeros(B, device=cuda), torch.zeros(B * T, device=cuda)
    assert tocr.lib().tocr_rec_head_ctc_f16(
        f.data_ptr(), B, T, K, w.data_ptr(), b.data_ptr(), V, V, toks.data_ptr(), lens.data_ptr(),
        sc.data_ptr(), idx.data_ptr(), prob.data_ptr(), err.data_ptr(),
        torch.cuda.current_stream().cuda_stream) == 0
    loss, _ = rec_head.cross_entropy(f, w, b, idx, err=err)
    torch.cuda.synchronize()
    assert int(err) == 0
    assert torch.allclose(torch.exp(-loss), prob, rtol=1e-4, atol=0)


def test_train_quantize_serve(tocr, cuda):
    """The operators as they are used together: some steps of gradient descent on
    the head, its weights laid out in INT8, the logits of the INT8 layer decoded
    by the stored-logits decoder. Each step's gradients are checked against the
    64-bit formula, the INT8 logits against the layer on the dequantised codes."""
    from turboocr_b200 import kernels, linear_i8
    B, T, K, V = 8, 20, 64, 500
    f, w, b, t, _ = make(B * T, K, V, torch.float16, 95, cuda, pad=0.1)
    n = float((t >= 0).sum())
    gl = torch.full((B * T,), 1.0 / n, device=cuda)
    w32 = w.float()
    err = err_word(cuda)
    for _ in range(3):
        w = w32.half()
        got = run(f, w, b, t, gl, cuda)
        near(got, exact(f, w, b, t, gl))
        w32 = w32 - 2.0 * got["dweight"].float()
        b = b - 2.0 * got["dbias"]
    wq, ws = linear_i8.quantize_rows(w32)
    logits = linear_i8.linear(f, wq, ws, b, err=err)
    fq, fs = linear_i8.quantize_rows(f)
    ref = (fq.double() * fs.double()[:, None]) @ (wq.double() * ws.double()[:, None]).T + b.double()
    assert float((logits.double() - ref).abs().max()) <= 2.0 ** -10 * float(ref.abs().max())
    out = kernels.CtcOutputs(B, T, cuda)
    kernels.ctc_greedy_f16(logits.view(B, T, V), V, out)
    torch.cuda.synchronize()
    assert int(err) == 0
    top = logits.float().max(1, keepdim=True).values
    first = (logits.float() == top).float().argmax(1)
    assert torch.equal(out.step_idx.long(), first)


def test_offsets_beyond_32_bits(tocr, cuda):
    """Feature and weight matrices of more than 2^32 bytes."""
    err = err_word(cuda)
    K, V, rows = 256, 70, (1 << 23) + 3001
    g = torch.Generator(device=cuda).manual_seed(1)
    f = torch.randn(rows, K, generator=g, device=cuda, dtype=torch.float16)
    w = torch.randn(V, K, generator=g, device=cuda, dtype=torch.float16) * 0.1
    t = torch.randint(0, V, (rows,), generator=g, device=cuda, dtype=torch.int32)
    gl = torch.ones(rows, device=cuda)
    loss, lse = rec_head.cross_entropy(f, w, None, t, err=err)
    df, _, _ = rec_head.cross_entropy_backward(f, w, None, t, lse, gl, err=err, need_weight=False)
    at = torch.cat([torch.arange(0, 200, device=cuda), torch.arange(rows - 300, rows, device=cuda)])
    want = exact(f[at], w, None, t[at], gl[at])
    near({"loss": loss[at], "lse": lse[at], "dfeat": df[at]}, want, ("loss", "lse", "dfeat"))
    assert int(err) == 0
    del f, df, loss, lse
    V, rows = (1 << 23) + 777, 3
    w = torch.empty(V, K, dtype=torch.float16, device=cuda)
    for k in range(0, V, 1 << 20):
        w[k:k + (1 << 20)].normal_(generator=g)
    w *= 0.1
    f = torch.randn(rows, K, generator=g, device=cuda, dtype=torch.float16)
    t = torch.tensor([0, V - 1, V // 2], dtype=torch.int64, device=cuda)
    loss, lse = rec_head.cross_entropy(f, w, None, t, err=err)
    _, dw, _ = rec_head.cross_entropy_backward(f, w, None, t, lse, gl[:rows].contiguous(), err=err,
                                               need_feat=False)
    x = f.double()
    parts = [x @ w[k:k + (1 << 20)].double().T for k in range(0, V, 1 << 20)]
    z = torch.logsumexp(torch.stack([torch.logsumexp(p, 1) for p in parts]), 0)
    # the sum over 2^23 classes: 1e-5 covers its fp32 rounding (pieces of 64)
    assert bool(((lse.double() - z).abs() < 1e-5 * z.abs()).all())
    lt = (x * w[t].double()).sum(1)
    assert bool(((loss.double() - (z - lt)).abs() < 2e-5 * z.abs()).all())
    rows_at = torch.cat([t, torch.tensor([V - 2, 5, V // 2 + 1], device=cuda)])
    p = torch.exp(x @ w[rows_at].double().T - z[:, None])
    p[torch.arange(3), torch.arange(3)] -= 1
    ref = p.T @ x
    assert bool(((dw[rows_at].double() - ref).abs() <= 2e-3 * ref.abs() + 1e-7).all())
    assert int(err) == 0


# ---- several chunks of classes per CTA: 4096 rows are 32 tiles, 18385 classes 144 chunks, so
# that each of 148 CTAs has 31 steps, and a class in the 64th chunk is not the first that a warp
# sees but in the few CTAs whose range begins there
MANY, CLASSES, FAR = 4096, 18385, 8192


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("column", [0, 1, 2, 3, 4, 18, 31])
def test_one_class_far_above_the_others(tocr, cuda, column, dtype):
    """A class whose logit is 90 to 1000 above the rest, at columns of every
    kind, behind the chunks in which the sums got their base."""
    f, w, b, t, gl = make(MANY, 64, CLASSES, dtype, 101 + column, cuda, pad=0.1)
    t = torch.where(t == FAR + column, torch.ones_like(t), t)
    for above in (90.0, 100.0, 176.0, 200.0, 300.0, 400.0, 1000.0):
        b2 = b.clone()
        b2[FAR + column] = above
        check((f, w, b2, t, gl), cuda)


@pytest.mark.parametrize("other", [FAR, FAR + 3, FAR + 4])
def test_classes_masked_by_a_large_finite_bias(tocr, cuda, other):
    """All classes but two masked with -1e4; the two have equal logits, so the
    loss of one as the target is log 2."""
    f, w, b, t, gl = make(MANY, 64, CLASSES, torch.float16, 111, cuda)
    w[other], w[9000] = 0, 0
    b = torch.full_like(b, -1e4)
    b[other], b[9000] = 0, 0
    t = torch.full_like(t, 9000)
    got = run(f, w, b, t, gl, cuda)
    near(got, exact(f, w, b, t, gl))
    assert float((got["loss"] - math.log(2)).abs().max()) < 1e-5


@pytest.mark.parametrize("kind", ["rising", "falling", "steps", "far below", "spread"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_logits_of_any_size_over_many_chunks(tocr, cuda, kind, dtype):
    f, w, b, t, gl = make(MANY, 64, CLASSES, dtype, 121, cuda, pad=0.1)
    at = torch.arange(CLASSES, device=cuda)
    ramp = torch.linspace(-900, 900, CLASSES, device=cuda)
    if kind == "rising":
        b = b + ramp
    elif kind == "falling":
        b = b - ramp
    elif kind == "steps":        # every 1000 classes another level, up and down
        b = b + ((at // 1000 * 7) % 19 - 9).float() * 37
    elif kind == "far below":
        b = b - 5000
    else:
        f = (f.float() * 40).to(dtype)
    check((f, w, b, t, gl), cuda)


@pytest.mark.parametrize("rows,V,at", [(200, 700, 96), (MANY, CLASSES, FAR)])
@pytest.mark.parametrize("column", [0, 1, 2, 3, 4, 18, 31])
def test_nan_class_shows_in_every_loss(tocr, cuda, rows, V, at, column):
    """A NaN in the weights or the bias of one class, whatever its column, is a
    NaN in the logits and so in the loss and lse of all rows but padding; an
    infinite bias leaves no finite loss either."""
    f, w, b, t, gl = make(rows, 64, V, torch.bfloat16, 131, cuda, pad=0.2)
    t = torch.where(t == at + column, torch.zeros_like(t), t)
    keep = t >= 0
    err = err_word(cuda)
    w2, b2, b3 = w.clone(), b.clone(), b.clone()
    w2[at + column, 5] = math.nan
    b2[at + column] = math.nan
    b3[at + column] = math.inf
    for ww, bb in ((w2, b), (w, b2)):
        loss, lse = rec_head.cross_entropy(f, ww, bb, t, err=err)
        assert bool(torch.isnan(loss[keep]).all()) and bool(torch.isnan(lse[keep]).all())
        assert bool((loss[~keep] == 0).all()) and bool((lse[~keep] == 0).all())
    loss, lse = rec_head.cross_entropy(f, w, b3, t, err=err)
    assert not bool(torch.isfinite(loss[keep]).any()) and not bool(torch.isfinite(lse[keep]).any())
    assert int(err) == 0


@pytest.mark.parametrize("K", [64, 200])
@pytest.mark.parametrize("rows,kept", [(0, 0), (5, 5), (300, 300), (700, 200), (700, 513),
                                       (1500, 1000), (1500, 1490)])
def test_infinite_weights_meet_no_padding(tocr, cuda, rows, kept, K):
    """Without a row that has a target every gradient is zero, whatever the
    weights hold. A class whose logit is -inf for every row (features above zero,
    an infinite weight below) has probability zero and a zero gradient, also
    where the rows do not fill their last tile."""
    f, w, b, t, gl = make(rows, K, 500, torch.float16, 141, cuda)
    f = f.abs() + 0.25
    t = torch.where(t == 77, torch.zeros_like(t), t)
    t[kept:] = -1
    w[77] = -math.inf
    got = run(f, w, b, t, gl, cuda, need_feat=False)
    assert bool((got["dweight"][77] == 0).all()) and float(got["dbias"][77]) == 0
    w2 = w.clone()
    w2[77] = 0
    b2 = b.clone()
    b2[77] = -math.inf
    two = run(f, w2, b2, t, gl, cuda, need_feat=False)
    for k in ("loss", "lse", "dweight", "dbias"):
        assert torch.equal(got[k], two[k]), k
    w[78], w[79, 3] = math.inf, math.nan
    got = run(f, w, b, torch.full_like(t, -1), gl, cuda)
    for k, v in got.items():
        assert bool((v == 0).all()), k


@pytest.mark.parametrize("rows", [200, 1500])
def test_one_workspace_for_backward_after_backward(tocr, cuda, rows):
    """Backward calls in a row on one stream with the same scratch memory, in which
    one kernel lays out the rows that the next one reads: each has the bits of a
    call by itself."""
    K, V = 72, 3000
    sets = [make(rows, K, V, torch.float16, s, cuda, pad=0.3) for s in (151, 152, 153)]
    want = [run(*s, cuda) for s in sets]
    err = err_word(cuda)
    n = tocr.lib().tocr_rec_head_ce_workspace_bytes(rows, K, V, 1)
    buf = torch.zeros(n, dtype=torch.uint8, device=cuda)
    got = [(torch.empty_like(f), torch.empty_like(w), torch.empty_like(b))
           for f, w, b, _, _ in sets * 4]
    torch.cuda.synchronize()
    for k, o in enumerate(got):
        f, w, b, t, gl = sets[k % 3]
        assert tocr.lib().tocr_rec_head_ce_backward(
            f.data_ptr(), w.data_ptr(), b.data_ptr(), t.data_ptr(), 0, rows, K, V, 0,
            want[k % 3]["lse"].data_ptr(), gl.data_ptr(), *(x.data_ptr() for x in o),
            buf.data_ptr(), n, err.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    for k, o in enumerate(got):
        for v, name in zip(o, ("dfeat", "dweight", "dbias")):
            assert torch.equal(v, want[k % 3][name]), (k, name)
    assert int(err) == 0

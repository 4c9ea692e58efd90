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

"""The INT8 linear layer and the recognizer head's cross entropy, as workloads.

Two operators of the recognizer's linear layers, each with a plain form in
elementary torch operations and the calls of this package that do the same:

``linear_i8``   y = act(sx[m] * sw[n] * sum_k qx[m][k] qw[n][k] + bias[n]): the
                rows of x are quantised to INT8 with one scale per token as the
                call begins, the weights were quantised with one scale per
                output channel when they were laid out. A row's scale is
                max|x| / 127 rounded to fp32 (2^-126 at least); a code is x
                divided by that scale, rounded to the nearest integer (ties to
                even).
``cross_entropy``  loss[i] = log sum_j exp(l[i][j]) - l[i][t[i]] with the logits
                l = feat W^T + bias never stored, and its gradient with respect
                to feat, W and bias for a weight per row; a row whose target is
                outside the vocabulary is padding: loss, lse and gradient zero.

``own`` chooses which of the two ``run`` calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False

F16, BF16, F32 = "float16", "bfloat16", "float32"
BYTES = {F16: 2, BF16: 2, F32: 4}
V_DICT = 18385            # classes of the shipped dictionary, blank included


def listed() -> list[dict]:
    return [
        # --- INT8 linear layer ---
        # one time step through a wide-feature recognizer head: latency, the weights are the bytes
        {"name": "i8_one_step", "op": "linear_i8", "rows": 1, "K": 512, "N": V_DICT,
         "x": F16, "y": F16, "bias": True, "act": "none"},
        # one text line (80 steps) through an encoder projection: the smallest call of a served line
        {"name": "i8_line", "op": "linear_i8", "rows": 80, "K": 128, "N": 384,
         "x": F16, "y": F16, "bias": True, "act": "none"},
        # 32 lines (one recognizer batch) through an encoder's expanding layer with its activation
        {"name": "i8_batch", "op": "linear_i8", "rows": 2560, "K": 256, "N": 1024,
         "x": F16, "y": F16, "bias": True, "act": "hardswish"},
        # odd sizes throughout, fp32 activations, no bias
        {"name": "i8_ragged", "op": "linear_i8", "rows": 4099, "K": 1001, "N": 2049,
         "x": F32, "y": F32, "bias": False, "act": "relu"},
        # the INT8 head writing the logits of 512 lines for the stored-logits decode: the output is the bytes
        {"name": "i8_logits", "op": "linear_i8", "rows": 512 * 80, "K": 128, "N": V_DICT,
         "x": F16, "y": F16, "bias": True, "act": "none"},
        # a large square-ish layer: the matrix product itself
        {"name": "i8_wide", "op": "linear_i8", "rows": 16384, "K": 4096, "N": 4096,
         "x": BF16, "y": BF16, "bias": True, "act": "none"},
        # --- cross entropy of the recognizer head ---
        # scoring one line against a given transcript: forward only, latency
        {"name": "ce_score_line", "op": "cross_entropy", "rows": 80, "K": 128, "V": V_DICT,
         "x": F16, "pad": 0.0, "grad": False, "bias": True},
        # scoring 512 lines
        {"name": "ce_score_lines", "op": "cross_entropy", "rows": 512 * 80, "K": 128, "V": V_DICT,
         "x": F16, "pad": 0.0, "grad": False, "bias": True},
        # a small training step: seven short lines over a small dictionary
        {"name": "ce_train_small", "op": "cross_entropy", "rows": 7 * 25, "K": 64, "V": 5000,
         "x": F16, "pad": 0.2, "grad": True, "bias": True},
        # an ordinary training step: 128 lines of 80 steps, half of the steps padding
        {"name": "ce_train", "op": "cross_entropy", "rows": 128 * 80, "K": 128, "V": V_DICT,
         "x": F16, "pad": 0.5, "grad": True, "bias": True},
        # bf16, an odd row count and a feature width that fills no whole tile, no bias
        {"name": "ce_train_bf16", "op": "cross_entropy", "rows": 8191, "K": 200, "V": V_DICT,
         "x": BF16, "pad": 0.0, "grad": True, "bias": False},
        # a large vocabulary
        {"name": "ce_train_large", "op": "cross_entropy", "rows": 16384, "K": 256, "V": 65537,
         "x": BF16, "pad": 0.1, "grad": True, "bias": True},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    """One more case: sizes spread over their logarithm, odd ones among them."""
    if rng.random() < 0.5:
        while True:
            c = {"op": "linear_i8", "rows": _log_int(rng, 1, 40960), "K": _log_int(rng, 16, 4096),
                 "N": _log_int(rng, 16, V_DICT), "x": rng.choice([F16, BF16, F32]),
                 "y": rng.choice([F16, BF16, F32]), "bias": rng.random() < 0.7,
                 "act": rng.choice(["none", "relu", "hardswish"])}
            if c["rows"] * c["N"] * c["K"] <= 16384 * 4096 * 4096 and \
                    c["rows"] * c["N"] * BYTES[c["y"]] <= 512 * 80 * V_DICT * 2:
                return c
    while True:
        c = {"op": "cross_entropy", "rows": _log_int(rng, 1, 40960), "K": 8 * rng.randint(1, 32),
             "V": _log_int(rng, 100, 65537), "x": rng.choice([F16, BF16]),
             "pad": rng.choice([0.0, 0.0, 0.1, 0.5]), "grad": rng.random() < 0.6,
             "bias": rng.random() < 0.7}
        if c["rows"] < 32:
            c["pad"] = 0.0                      # a handful of steps is not padded
        if c["rows"] * c["V"] * c["K"] <= 16384 * 65537 * 256:
            return c


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (as whole fp32 numbers) and fp32 scales of the rows of x. The
    division is in 64 bits: half of a row's maximum is a tie up to the
    rounding of the scale."""
    x = x.float()
    s = (x.abs().amax(dim=1) / 127.0).clamp_min(2.0 ** -126)
    return torch.round(x.double() / s.double()[:, None]).float(), s


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    dev = "cuda"
    if case["op"] == "linear_i8":
        M, K, N = case["rows"], case["K"], case["N"]
        # activations with a few channels larger than the rest, as after a norm's gain
        gain = torch.exp(0.7 * torch.randn(K, generator=g, device=dev))
        x = (torch.randn(M, K, generator=g, device=dev) * gain).to(getattr(torch, case["x"]))
        w = torch.randn(N, K, generator=g, device=dev) * (1.0 / math.sqrt(K))
        # the weights as laid out once: codes in rows of a multiple of 16 bytes, zero behind K
        q, ws = _quantize(w)
        wq = torch.zeros(N, (K + 15) // 16 * 16, dtype=torch.int8, device=dev)
        wq[:, :K] = q.to(torch.int8)
        bias = 0.5 * torch.randn(N, generator=g, device=dev) if case["bias"] else None
        return {"case": case, "x": x, "wq": wq, "ws": ws, "bias": bias,
                "err": torch.zeros(1, dtype=torch.int32, device=dev)}
    M, K, V = case["rows"], case["K"], case["V"]
    dt = getattr(torch, case["x"])
    w = (torch.randn(V, K, generator=g, device=dev) * (3.0 / math.sqrt(K))).to(dt)
    bias = 0.5 * torch.randn(V, generator=g, device=dev) if case["bias"] else None
    feat = torch.randn(M, K, generator=g, device=dev)
    # half of the steps are blank, the others any class; some steps are already recognised well
    t = torch.randint(0, V, (M,), generator=g, device=dev, dtype=torch.int32)
    t = torch.where(torch.rand(M, generator=g, device=dev) < 0.5, torch.zeros_like(t), t)
    known = torch.rand(M, generator=g, device=dev) < 0.5
    feat = torch.where(known[:, None], w[t.long()].float() * (math.sqrt(K) / 3.0) + 0.3 * feat, feat)
    # the steps behind a line's end are padding
    pad = torch.rand(M, generator=g, device=dev) < case["pad"]
    t = torch.where(pad, torch.full_like(t, -1), t)
    weight = 0.25 + 0.75 * torch.rand(M, generator=g, device=dev)
    return {"case": case, "feat": feat.to(dt), "w": w, "bias": bias, "t": t, "g": weight,
            "err": torch.zeros(1, dtype=torch.int32, device=dev)}


def _act(y: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return y.clamp_min(0.0)
    if act == "hardswish":
        return y * (y + 3.0).clamp(0.0, 6.0) / 6.0
    return y


def _plain_linear(s: dict) -> torch.Tensor:
    c = s["case"]
    qx, sx = _quantize(s["x"])
    K = c["K"]
    wq = s["wq"][:, :K]
    # sums of up to 1024 products of codes are whole numbers below 2^24, exact in 32 bits:
    # the pieces of K are one batch, and their sums are added as integers
    P = (K + 1023) // 1024
    a = torch.nn.functional.pad(qx, (0, P * 1024 - K)).view(-1, P, 1024).transpose(0, 1)
    b = torch.nn.functional.pad(wq.float(), (0, P * 1024 - K)).view(-1, P, 1024).permute(1, 2, 0)
    if P == 1:
        acc = qx @ wq.float().T
    else:
        acc = torch.matmul(a, b).to(torch.int32).sum(dim=0).float()
    y = acc * sx[:, None] * s["ws"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"]
    return _act(y, c["act"]).to(getattr(torch, c["y"]))


def _plain_ce(s: dict) -> dict:
    V = s["case"]["V"]
    t = s["t"].long()
    keep = (t >= 0) & (t < V)
    at = torch.where(keep, t, torch.zeros_like(t))[:, None]
    x, w = s["feat"].float(), s["w"].float()
    logits = x @ w.T
    if s["bias"] is not None:
        logits = logits + s["bias"]
    m = logits.amax(dim=1, keepdim=True)
    lse = m + torch.log(torch.exp(logits - m).sum(dim=1, keepdim=True))
    zero = torch.zeros((), device=x.device)
    loss = torch.where(keep, (lse - logits.gather(1, at))[:, 0], zero)
    out = {"loss": loss, "lse": torch.where(keep, lse[:, 0], zero)}
    if s["case"]["grad"]:
        d = torch.exp(logits - lse)
        d.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
        d = torch.where(keep, s["g"], zero)[:, None] * d
        out["dfeat"] = (d @ w).to(s["feat"].dtype)
        out["dweight"] = (d.T @ x).to(s["w"].dtype)
        if s["bias"] is not None:
            out["dbias"] = d.sum(dim=0)
    return out


def run(state: dict):
    c = state["case"]
    if c["op"] == "linear_i8":
        if not own:
            return _plain_linear(state)
        from turboocr_b200 import linear_i8
        return linear_i8.linear(state["x"], state["wq"], state["ws"], state["bias"],
                                act=c["act"], out_dtype=getattr(torch, c["y"]), err=state["err"])
    if not own:
        return _plain_ce(state)
    from turboocr_b200 import rec_head
    loss, lse = rec_head.cross_entropy(state["feat"], state["w"], state["bias"], state["t"],
                                       err=state["err"])
    out = {"loss": loss, "lse": lse}
    if c["grad"]:
        dfeat, dweight, dbias = rec_head.cross_entropy_backward(
            state["feat"], state["w"], state["bias"], state["t"], lse, state["g"],
            err=state["err"])
        out["dfeat"], out["dweight"] = dfeat, dweight
        if dbias is not None:
            out["dbias"] = dbias
    return out


def work(case: dict) -> dict:
    if case["op"] == "linear_i8":
        M, K, N = case["rows"], case["K"], case["N"]
        return {"bytes": M * K * BYTES[case["x"]] + N * K + 4 * N * (2 if case["bias"] else 1)
                + M * N * BYTES[case["y"]], "flops": 2 * M * N * K}
    M, K, V = case["rows"], case["K"], case["V"]
    kept = M * (1.0 - case["pad"])              # padded steps need no product
    nbytes = 2 * K * (kept + V) + 4 * M + 8 * M + (4 * V if case["bias"] else 0)
    flops = 2.0 * kept * V * K
    if case["grad"]:                            # both gradients; the logits' second making is not counted
        nbytes += 2 * K * (M + V) + 4 * M + (4 * V if case["bias"] else 0)
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "linear_i8":
        x = s["x"].double()
        sx = torch.maximum((x.abs().max(dim=1).values.float() / 127.0).double(),
                           torch.tensor(2.0 ** -126, dtype=torch.float64, device=x.device))
        y = torch.div(x, sx.unsqueeze(1)).round_() @ s["wq"][:, :case["K"]].double().t()
        y.mul_(sx.unsqueeze(1)).mul_(s["ws"].double())
        if s["bias"] is not None:
            y.add_(s["bias"].double())
        if case["act"] == "relu":
            y.clamp_(min=0.0)
        elif case["act"] == "hardswish":
            y.mul_((y + 3.0).clamp_(0.0, 6.0)).div_(6.0)
        return y
    M, K, V = case["rows"], case["K"], case["V"]
    x, w = s["feat"].double(), s["w"].double()
    loss = torch.zeros(M, dtype=torch.float64, device=x.device)
    lse = torch.zeros_like(loss)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    db = torch.zeros(V, dtype=torch.float64, device=x.device)
    rows = torch.nonzero((s["t"] >= 0) & (s["t"] < V)).flatten()
    for part in torch.split(rows, 4096):        # pieces of the rows: 64-bit logits of all do not fit well
        p = x[part] @ w.t()
        if s["bias"] is not None:
            p += s["bias"].double()
        z = torch.logsumexp(p, dim=1)
        t = s["t"][part].long()
        k = torch.arange(part.numel(), device=x.device)
        lse[part] = z
        loss[part] = z - p[k, t]
        if case["grad"]:
            p = p.sub_(z.unsqueeze(1)).exp_()
            p[k, t] -= 1.0
            p *= s["g"][part].double().unsqueeze(1)
            dx[part] = p @ w
            dw += p.t() @ x[part]
            db += p.sum(dim=0)
    out = {"loss": loss, "lse": lse}
    if case["grad"]:
        out["dfeat"], out["dweight"] = dx, dw
        if s["bias"] is not None:
            out["dbias"] = db
    return out

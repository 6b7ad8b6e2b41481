"""The dense operators around a sparse layer, as a program that trains or serves
a pruned model calls them: layer norm, the dense layer with its epilogue, and
distillation from a teacher's top logits.

A case is a dict of plain values.  ``op`` names the operator:

  norm     layer norm over the last axis of rows x features values,
  linear   activation(x W^T + bias) + residual, x tokens x inner, W outer x inner,
  distill  T^2 KL(teacher's top k || student) over a vocabulary, one row per token.

``train`` cases return the gradients too.  With ``own`` false, ``run`` computes
the operators in elementary torch operations in 32 bits; with ``own`` true it
calls void_amd.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}

# Work of the largest listed cases: drawn cases stay below.
NORM_MOST = 16384 * 8192
LINEAR_MOST = 8192 * 4096 * 14336
DISTILL_MOST = 8192 * 131072


def _norm(name, rows, features, dtype, train):
    return dict(name=name, op="norm", rows=rows, features=features, dtype=dtype, train=train)


def _linear(name, tokens, inner, outer, dtype, act, residual, train):
    return dict(name=name, op="linear", tokens=tokens, inner=inner, outer=outer, dtype=dtype, act=act,
                residual=residual, train=train)


def _distill(name, rows, vocab, k, dtype, form, temperature, prompt, ragged, scale=1.0):
    return dict(name=name, op="distill", rows=rows, vocab=vocab, k=k, dtype=dtype, form=form, train=form != "eval",
                temperature=temperature, prompt=prompt, ragged=ragged, scale=scale)


def listed():
    return [
        # Serving one token: the norm in front of a layer, where latency counts.
        _norm("norm_one_token", 1, 4096, "bf16", False),
        # Fine-tuning in float32 on a matrix with no size a multiple of anything.
        _norm("norm_ragged_fp32", 5003, 3001, "fp32", True),
        # Fine-tuning a layer of the usual width on 2048 tokens.
        _norm("norm_train_bf16", 2048, 4096, "bf16", True),
        # A long batch of a wide model.
        _norm("norm_large_bf16", 16384, 8192, "bf16", True),
        # Serving one token: the FFN up-projection that was left dense.
        _linear("linear_one_token", 1, 4096, 14336, "bf16", "gelu", False, False),
        # Prefill of the down-projection, added to the residual stream.
        _linear("linear_prefill_fp16", 2048, 14336, 4096, "fp16", "none", True, False),
        # Fine-tuning in float32, odd sizes throughout.
        _linear("linear_ragged_fp32", 730, 3001, 5003, "fp32", "silu", True, True),
        # Fine-tuning the dense up-projection of the FFN on a long batch.
        _linear("linear_train_bf16", 8192, 4096, 14336, "bf16", "gelu", False, True),
        # A few tokens over a long vocabulary: loss and gradient in one call.
        _distill("distill_few_rows", 8, 131072, 64, "bf16", "step", 2.0, 0.0, False),
        # float32 logits of an odd vocabulary, lists of different lengths, a
        # quarter of the rows prompt tokens that the loss leaves out.
        _distill("distill_ragged_fp32", 730, 50021, 100, "fp32", "autograd", 2.0, 0.25, True),
        # A training step through autograd.
        _distill("distill_train_bf16", 4096, 32768, 64, "bf16", "autograd", 1.0, 0.0, False),
        # A long batch over a long vocabulary: loss and gradient in one call.
        _distill("distill_large_bf16", 8192, 131072, 128, "bf16", "step", 2.0, 0.25, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, multiple=160):
    """A size in [lo, hi], log-uniform; a multiple of 32 (of 160) half of the time."""
    v = _log(rng, lo, hi)
    return max(lo, v // multiple * multiple) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["norm", "linear", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        features = _size(rng, 64, 16384)
        rows = min(_log(rng, 1, 32768), NORM_MOST * 2 // SIZE[dtype] // features)
        c = _norm("", rows, features, dtype, rng.random() < 0.7)
    elif op == "linear":
        # Tokens: one to sixteen (serving) or up to a long batch.
        tokens = _log(rng, 1, 16) if rng.random() < 0.3 else _size(rng, 16, 8192)
        inner, outer = _size(rng, 64, 14336), _size(rng, 64, 14336)
        most = LINEAR_MOST // (16 if dtype == "fp32" else 1)
        tokens = max(1, min(tokens, most // (inner * outer)))
        c = _linear("", tokens, inner, outer, dtype, rng.choice(["none", "relu", "gelu", "silu"]),
                    rng.random() < 0.5, tokens > 16 and rng.random() < 0.5)
    else:
        vocab = _size(rng, 512, 131072)
        rows = max(1, min(_log(rng, 1, 8192), DISTILL_MOST * 2 // SIZE[dtype] // vocab))
        form = rng.choice(["eval", "autograd", "step", "step"])
        # float16 gradients are scaled up, as a loss scaler does.
        c = _distill("", rows, vocab, min(vocab, _log(rng, 1, 256)), dtype, form, rng.choice([1.0, 2.0, 4.0]),
                     rng.choice([0.0, 0.25]), rng.random() < 0.5, 4096.0 if dtype == "fp16" else 1.0)
    del c["name"]
    return c


# ---- inputs ---------------------------------------------------------------

def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device=DEV).mul_(std).add_(mean)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    if case["op"] == "norm":
        R, C = case["rows"], case["features"]
        # Rows of different scales around a common offset, as a residual stream holds.
        x = randn(R, C) * (0.5 + 2 * uniform(R, 1)) + randn(1, C, std=0.3)
        st = {"x": x.to(dt), "weight": randn(C, std=0.1, mean=1.0).to(dt), "bias": randn(C, std=0.1).to(dt)}
        if case["train"]:
            st["dy"] = randn(R, C).to(dt)
        return st
    if case["op"] == "linear":
        M, K, N = case["tokens"], case["inner"], case["outer"]
        st = {"x": randn(M, K).to(dt), "weight": randn(N, K, std=1 / math.sqrt(K)).to(dt),
              "bias": randn(N, std=0.1).to(dt)}
        if case["residual"]:
            st["residual"] = randn(M, N).to(dt)
        if case["train"]:
            st["dy"] = randn(M, N).to(dt)
        return st
    R, V, k = case["rows"], case["vocab"], case["k"]
    # The teacher's k tokens, scattered over the vocabulary, best first.
    start = (uniform(R, 1) * V).long().clamp_(max=V - 1)
    step = (1 + uniform(R, 1) * (V // k)).long().clamp_(max=max(1, V // k))
    index = (start + torch.arange(k, device=DEV) * step) % V
    top = randn(R, k, std=2.0, mean=8.0).sort(dim=1, descending=True).values
    # A student that has learned part of it.
    logits = randn(R, V, std=2.0).scatter_add_(1, index, 0.7 * top).to(dt)
    length = torch.full((R, 1), k, device=DEV)
    if case["ragged"]:
        length = (k / 2 + uniform(R, 1) * (k / 2 + 1)).long().clamp_(1, k)
    # Prompt tokens have no teacher's list; entries past a list's end are -1.
    prompt = torch.randperm(R, generator=g, device=DEV)[:int(R * case["prompt"])]
    length[prompt] = 0
    index = torch.where(torch.arange(k, device=DEV) < length, index, -1)
    return {"logits": logits, "top": top.to(dt), "index": index,
            "scale": torch.full((), case["scale"], device=DEV)}


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["train"]:
        for name in ("x", "weight", "bias", "residual", "logits"):
            if name in st:
                st[name].requires_grad_()
    st["case"] = case
    return st


# ---- one pass -------------------------------------------------------------

def _norm_own(st, case):
    import void_amd
    y = void_amd.layer_norm(st["x"], st["weight"], st["bias"], eps=1e-5)
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])]


def _norm_plain(st, case):
    dt = st["x"].dtype
    x, w, b = st["x"].float(), st["weight"].float(), st["bias"].float()
    d = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + 1e-5)
    xhat = d * rstd
    y = (xhat * w + b).to(dt)
    if not case["train"]:
        return y
    dy = st["dy"].float()
    wdy = dy * w
    dx = rstd * (wdy - wdy.mean(1, keepdim=True) - xhat * (wdy * xhat).mean(1, keepdim=True))
    return [y, dx.to(dt), (dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)]


def _linear_own(st, case):
    import void_amd
    y = void_amd.fused_linear(st["x"], st["weight"], st["bias"], activation=case["act"], residual=st.get("residual"))
    if not case["train"]:
        return y
    wrt = [st[n] for n in ("x", "weight", "bias", "residual") if n in st]
    return [y.detach(), *torch.autograd.grad(y, wrt, st["dy"])]


def _activate(z, act):
    """act(z) and its derivative; GELU in its tanh form."""
    if act == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).float()
    if act == "gelu":
        t = torch.tanh(0.7978845608 * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608 * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, None


def _linear_plain(st, case):
    dt = st["x"].dtype
    x, w = st["x"].float(), st["weight"].float()
    y, slope = _activate(x @ w.t() + st["bias"].float(), case["act"])
    if "residual" in st:
        y = y + st["residual"].float()
    y = y.to(dt)
    if not case["train"]:
        return y
    dz = st["dy"].float()
    if slope is not None:
        dz = dz * slope
    out = [y, (dz @ w).to(dt), (dz.t() @ x).to(dt), dz.sum(0).to(dt)]
    return out + [st["dy"]] if "residual" in st else out


def _distill_own(st, case):
    import void_amd
    T = case["temperature"]
    if case["form"] == "eval":
        return void_amd.distillation_loss(st["logits"], st["top"], st["index"], temperature=T, reduction="none")
    if case["form"] == "autograd":
        loss = void_amd.distillation_loss(st["logits"], st["top"], st["index"], temperature=T)
        return [loss.detach(), *torch.autograd.grad(loss, st["logits"], st["scale"])]
    return list(void_amd.distillation_loss_and_grad(st["logits"], st["top"], st["index"], temperature=T,
                                                    grad_scale=case["scale"]))


def _distill_plain(st, case):
    T = case["temperature"]
    index, valid = st["index"].clamp(min=0), st["index"] >= 0
    some = valid.any(1, keepdim=True)
    t = torch.where(valid, st["top"].float() / T, float("-inf"))
    e = torch.exp(t - torch.where(some, t.amax(1, keepdim=True), 0.0))
    p = e / torch.where(some, e.sum(1, keepdim=True), 1.0)
    s = st["logits"].float() / T
    top = s.amax(1, keepdim=True)
    q = torch.exp(s - top)
    total = q.sum(1, keepdim=True)
    lse = top + torch.log(total)
    term = p * (torch.log(torch.where(p > 0, p, 1.0)) + lse - s.gather(1, index))
    rows = T * T * torch.where(p > 0, term, 0.0).sum(1)
    if case["form"] == "eval":
        return rows
    count = some.sum().clamp(min=1)
    grad = torch.where(some, q / total, 0.0).scatter_add_(1, index, -p) * (T * st["scale"] / count)
    return [rows.sum() / count, grad.to(st["logits"].dtype)]


def run(state):
    case = state["case"]
    form = globals()["_%s_%s" % (case["op"], "own" if own else "plain")]
    if case["train"] and own:
        return form(state, case)
    with torch.no_grad():
        return form(state, case)


# ---- what a pass cannot do without ----------------------------------------

def work(case):
    esz = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, C = case["rows"] * case["features"], case["features"]
        if case["train"]:  # x, dy in; y, dx out
            return {"bytes": esz * (4 * n + 4 * C), "flops": 20 * n}
        return {"bytes": esz * (2 * n + 2 * C), "flops": 8 * n}
    if case["op"] == "linear":
        M, K, N = case["tokens"], case["inner"], case["outer"]
        n = M * K + N * K + N + M * N * (2 if case["residual"] else 1)
        if case["train"]:  # dy in; the gradients of x, W and bias out
            n += M * N + M * K + N * K + N
        return {"bytes": esz * n, "flops": 2 * M * N * K * (3 if case["train"] else 1)}
    R, V, k = case["rows"], case["vocab"], case["k"]
    rows = R - int(R * case["prompt"])  # the others' logits need not be read
    n = rows * V * esz + R * k * 8 + rows * k * esz + (R * V * esz + 4 if case["train"] else 4 * R)
    return {"bytes": n, "flops": rows * V * (8 if case["train"] else 5)}


# ---- 64-bit results -------------------------------------------------------

def _act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * torch.sigmoid(2 * 0.7978845608 * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if act == "silu" else z


def exact(case, seed):
    st = _inputs(case, seed)
    d = {n: v.double() for n, v in st.items() if n != "index"}
    if case["op"] == "distill":
        return _distill64(st, d, case)
    wrt = [d[n].requires_grad_(case["train"]) for n in ("x", "weight", "bias", "residual") if n in d]
    if case["op"] == "norm":
        x = d["x"]
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + 1e-5) * d["weight"] + d["bias"]
    else:
        y = _act64(torch.addmm(d["bias"], d["x"], d["weight"].t()), case["act"])
        if "residual" in d:
            y = y + d["residual"]
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, wrt, d["dy"])]


def _distill64(st, d, case):
    T, some = case["temperature"], (st["index"] >= 0).any(1)
    count = max(1, int(some.sum()))
    losses, grads = [], []
    most = max(1, (1 << 27) // case["vocab"])  # rows at a time
    for r in range(0, case["rows"], most):
        index, z = st["index"][r:r + most], d["logits"][r:r + most].detach().requires_grad_()
        keep = index >= 0
        p = torch.softmax((d["top"][r:r + most] / T).masked_fill(~keep, -1e300), 1) * keep
        logq = torch.log_softmax(z / T, 1).gather(1, index.clamp(min=0))
        row = T * T * (torch.special.xlogy(p, p) - p * logq).sum(1)
        losses.append(row.detach())
        if case["train"]:
            grads.append(torch.autograd.grad(row.sum() * case["scale"] / count, z)[0])
    loss = torch.cat(losses)
    return [loss.sum() / count, torch.cat(grads)] if case["train"] else loss

"""The operators at the end of a training step, as cases that can be timed and compared.

Three families, each entered the way a program enters it:

  norm      `row_norm_forward` / `row_norm_backward`: LayerNorm or RMSNorm with a learned gain (and shift), its
            statistics kept, and its gradient with the sums over the rows for gain and shift
  xent      `linear_cross_entropy` / `linear_cross_entropy_backward`: softmax cross entropy of hidden states against a
            vocabulary head, without the logits in memory
  distill   `linear_distillation` / `linear_distillation_backward`: the same head against a teacher's top logits

A case with mode "train" is a forward and a backward call, as a training step makes them; mode "loss" the forward alone,
as scoring a text or a validation pass does.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100


def _norm(name, rows, cols, kind, dtype="bf16", mode="train", shift=False, param="same"):
    return {"name": name, "family": "norm", "rows": rows, "cols": cols, "kind": kind, "dtype": dtype, "mode": mode, "shift": shift,
            "param": param}


def _xent(name, rows, hidden, vocab, dtype="bf16", mode="train", bias=False, ignored=0.0, weight="vd"):
    return {"name": name, "family": "xent", "rows": rows, "hidden": hidden, "vocab": vocab, "dtype": dtype, "mode": mode, "bias": bias,
            "ignored": ignored, "weight": weight}


def _distill(name, rows, hidden, vocab, k, dtype="bf16", mode="train", bias=False, ignored=0.0, weight="vd", temperature=2.0):
    return {"name": name, "family": "distill", "rows": rows, "hidden": hidden, "vocab": vocab, "k": k, "dtype": dtype, "mode": mode,
            "bias": bias, "ignored": ignored, "weight": weight, "temperature": temperature}


def listed():
    return [
        # LayerNorm of the GPT-J-shaped block (width 4096), four sequences of 2048 tokens, in a training step
        _norm("norm_layer_8192x4096", 8192, 4096, "layer", shift=True),
        # RMSNorm of heads or of a narrow model, many short rows, parameters kept in 32 bits
        _norm("norm_rms_65536x256", 65536, 256, "rms", param="fp32"),
        # one short sequence: the call's latency
        _norm("norm_rms_64x4096", 64, 4096, "rms"),
        # a batch of uneven prompts through a width that no vector load divides
        _norm("norm_layer_odd", 1371, 2047, "layer", dtype="fp16", shift=True),
        # scoring sixteen candidate tokens: one stream of the head's weights
        _xent("xent_score_16", 16, 4096, 51200, mode="loss"),
        # one training sequence on the GPT-J-shaped width, whose head has a bias
        _xent("xent_train_2048", 2048, 4096, 51200, bias=True),
        # fine-tuning on instructions: half of the tokens are prompt and carry no loss; a vocabulary of 256 thousand
        _xent("xent_train_tuning", 8192, 2048, 256000, ignored=0.5),
        # a few ragged rows in fp16, odd vocabulary
        _xent("xent_train_ragged", 777, 1000, 32003, dtype="fp16", ignored=0.2),
        # a small model: the calls' latency
        _xent("xent_train_small", 48, 512, 4000, weight="dv"),
        # distillation of one batch from a teacher's 64 best logits
        _distill("distill_train_4096", 4096, 4096, 51200, 64),
        # a large vocabulary, few entries, padding in some sequences
        _distill("distill_train_wide", 2048, 2048, 256000, 16, ignored=0.25),
        # a validation pass over a ragged batch
        _distill("distill_loss_ragged", 301, 1504, 32003, 100, dtype="fp16", mode="loss", bias=True),
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, int(round(v / multiple)) * multiple)


def draw(rng):
    """One more case of the same ranges; none costs more than the largest listed one."""
    family = rng.choice(["norm", "norm", "xent", "xent", "xent", "distill", "distill"])
    if family == "norm":
        cols = _log_int(rng, 64, 12288, rng.choice([1, 8, 8]))
        rows = min(_log_int(rng, 1, 65536), int(6e7 / cols))
        kind = rng.choice(["layer", "rms"])
        c = _norm("", max(rows, 1), cols, kind, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["train", "train", "loss"]),
                  kind == "layer", rng.choice(["same", "fp32"]))
    else:
        hidden = _log_int(rng, 128, 4096, 8)
        vocab = _log_int(rng, 500, 256000)
        weight = rng.choice(["vd", "vd", "dv"])
        if weight == "dv":
            vocab = (vocab + 7) // 8 * 8
        rows = max(1, min(_log_int(rng, 1, 8192), int(4.2e12 / (hidden * vocab))))
        common = (rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["train", "train", "loss"]), rng.random() < 0.3,
                  rng.choice([0.0, 0.0, 0.1, 0.3, 0.6]), weight)
        if family == "xent":
            c = _xent("", rows, hidden, vocab, *common)
        else:
            c = _distill("", rows, hidden, vocab, _log_int(rng, 1, 128), *common, temperature=rng.choice([1.0, 2.0, 4.0]))
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------- preparation

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    # (made in the tensor's own type: a head's weights are half a billion numbers)
    t = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    return t.mul_(scale) if scale != 1.0 else t


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def prepare(case, seed):
    """What the program holds when it makes the call."""
    c, g, dt = case, _generator(seed), DTYPES[case["dtype"]]
    if c["family"] == "norm":
        R, C = c["rows"], c["cols"]
        pt = torch.float32 if c["param"] == "fp32" else dt
        s = {"case": c, "eps": 1e-5 if c["kind"] == "layer" else 1e-6}
        # residual streams: every row has its own size, some channels stand out
        rows = (_randn(g, R, 1) * 0.5).exp_()
        s["x"] = (_randn(g, R, C) * rows * (1.0 + 3.0 * (_rand(g, C) < 0.01)) + 0.2).to(dt)
        s["offset"] = 1.0 if c["kind"] == "rms" else 0.0        # (1 + w) for RMSNorm, w for LayerNorm
        s["gain"] = (_randn(g, C, scale=0.1) + (1.0 - s["offset"])).to(pt)
        s["shift"] = _randn(g, C, scale=0.1).to(pt) if c["shift"] else None
        s["grad_out"] = (_randn(g, R, C) * rows).to(dt) if c["mode"] == "train" else None
        return s
    N, D, V = c["rows"], c["hidden"], c["vocab"]
    w = _randn(g, V, D, dtype=dt, scale=0.02) if c["weight"] == "vd" else _randn(g, D, V, dtype=dt, scale=0.02).t()
    s = {"case": c, "w": w, "bias": _randn(g, V, scale=0.1).to(dt) if c["bias"] else None}
    best = torch.randint(0, V, (N,), generator=g, device="cuda")
    # a model that has learned something: the right token's logit stands 4 to 12 above the others'
    lift = (4.0 + 8.0 * _rand(g, N, 1)) / (4e-4 * D)
    s["x"] = (_randn(g, N, D) + lift * w[best].float()).to(dt)
    ignored = torch.zeros(N, dtype=torch.bool, device="cuda")
    ignored[torch.randperm(N, generator=g, device="cuda")[:int(c["ignored"] * N)]] = True
    if c["family"] == "xent":
        s["labels"] = torch.where(ignored, IGNORE, best)
    else:
        # the teacher's best entries, in its order: distinct tokens, logits falling off from the first
        K = c["k"]
        steps = torch.randint(1, max(V // K, 2), (N, K), generator=g, device="cuda")
        steps[:, 0] = 0
        index = (best[:, None] + steps.cumsum(1)) % V
        logits = 12.0 - 6.0 * _rand(g, N, K).sort(1).values - 2.0 * (torch.arange(K, device="cuda") > 0)
        s["index"] = torch.where(ignored[:, None], -1, index)
        s["teacher"] = logits.to(dt)
    active = max(N - int(c["ignored"] * N), 1)
    # mean over the tokens that count; fp16 training scales its loss
    s["grad_loss"] = torch.full((N,), (4096.0 if c["dtype"] == "fp16" else 1.0) / active, device="cuda")
    return s


# ------------------------------------------------------------------------------------- one pass

def _package():
    import importlib
    return importlib.import_module("intel-extension-for-openxla_b200")


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ixk, c = _package(), s["case"]
    if c["family"] == "norm":
        kind = ixk.NORM_LAYER if c["kind"] == "layer" else ixk.NORM_RMS
        y, mean, rstd = ixk.row_norm_forward(s["x"], kind=kind, eps=s["eps"], gain=s["gain"], gain_offset=s["offset"], shift=s["shift"])
        out = {"y": y}
        if c["mode"] == "train":
            out["dx"], out["dgain"], dshift = ixk.row_norm_backward(
                s["grad_out"], s["x"], mean, rstd, kind=kind, gain=s["gain"], gain_offset=s["offset"], with_shift=c["shift"])
            if c["shift"]:
                out["dshift"] = dshift
        return out
    if c["family"] == "xent":
        loss, lse = ixk.linear_cross_entropy(s["x"], s["w"], s["labels"], bias=s["bias"], ignore_index=IGNORE)
        out = {"loss": loss, "lse": lse}
        if c["mode"] == "train":
            grads = ixk.linear_cross_entropy_backward(s["x"], s["w"], s["labels"], lse, s["grad_loss"], bias=s["bias"],
                                                      ignore_index=IGNORE)
    else:
        loss, lse = ixk.linear_distillation(s["x"], s["w"], s["index"], s["teacher"], bias=s["bias"], temperature=c["temperature"])
        out = {"loss": loss, "lse": lse}
        if c["mode"] == "train":
            grads = ixk.linear_distillation_backward(s["x"], s["w"], s["index"], s["teacher"], lse, s["grad_loss"], bias=s["bias"],
                                                     temperature=c["temperature"])
    if c["mode"] == "train":
        out["dx"], out["dw"] = grads[0], grads[1]
        if c["bias"]:
            out["dbias"] = grads[2]
    return out


def _run_plain(s):
    c = s["case"]
    dt = s["x"].dtype
    if c["family"] == "norm":
        x, scale = s["x"].float(), s["gain"].float() + s["offset"]
        xc = x - x.mean(1, keepdim=True) if c["kind"] == "layer" else x
        rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + s["eps"])
        xh = xc * rstd
        y = xh * scale
        if c["shift"]:
            y = y + s["shift"].float()
        out = {"y": y.to(dt)}
        if c["mode"] == "train":
            gy = s["grad_out"].float()
            h = gy * scale
            d = h - xh * (h * xh).mean(1, keepdim=True)
            if c["kind"] == "layer":
                d = d - h.mean(1, keepdim=True)
            out["dx"] = (d * rstd).to(dt)
            out["dgain"] = (gy * xh).sum(0).to(s["gain"].dtype)
            if c["shift"]:
                out["dshift"] = gy.sum(0).to(s["gain"].dtype)
        return out
    V = c["vocab"]
    w = s["w"].float()
    if c["family"] == "xent":
        active = (s["labels"] != IGNORE) & (s["labels"] >= 0) & (s["labels"] < V)
        index, q, scale, factor = torch.where(active, s["labels"], 0)[:, None], active[:, None].float(), 1.0, 1.0
    else:
        T = c["temperature"]
        present = (s["index"] >= 0) & (s["index"] < V)
        t = torch.where(present, s["teacher"].float() / T, -math.inf)
        active = present.any(1)
        top = torch.where(active, t.max(1).values, 0.0)[:, None]
        e = torch.exp(t - top)
        q = e / torch.where(active, e.sum(1), 1.0)[:, None]
        index, scale, factor = torch.where(present, s["index"], 0), 1.0 / T, T * T
    x = torch.where(active[:, None], s["x"].float(), 0.0)
    z = x @ w.t()
    if s["bias"] is not None:
        z += s["bias"].float()
    if scale != 1.0:
        z *= scale
    top = z.max(1, keepdim=True).values
    at_targets = z.gather(1, index)
    p = z.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    lse = (top + total.log()).squeeze(1)
    entropy = torch.where(q > 0, q * torch.log(torch.where(q > 0, q, 1.0)), 0.0).sum(1)
    loss = factor * (entropy - (q * at_targets).sum(1) + q.sum(1) * lse)
    out = {"loss": torch.where(active, loss, 0.0), "lse": torch.where(active, lse, 0.0)}
    if c["mode"] == "train":
        g = torch.where(active, s["grad_loss"] * (factor * scale), 0.0)[:, None]
        p.mul_(g / total)
        p.scatter_add_(1, index, -g * q)
        out["dx"] = (p @ w).to(dt)
        out["dw"] = (p.t() @ x).to(dt) if c["weight"] == "vd" else (x.t() @ p).to(dt).t()
        if c["bias"]:
            out["dbias"] = p.sum(0).to(dt)
    return out


# ------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The definitions in 64 bits, the head's a block of rows at a time."""
    c, s = case, prepare(case, seed)
    f64 = torch.float64
    if c["family"] == "norm":
        x, w = s["x"].to(f64), s["gain"].to(f64) + s["offset"]
        n = x.shape[1]
        mu = x.sum(1, keepdim=True) / n if c["kind"] == "layer" else torch.zeros_like(x[:, :1])
        sigma = ((x - mu).square().sum(1, keepdim=True) / n + s["eps"]).sqrt()
        u = (x - mu) / sigma
        out = {"y": u * w + (s["shift"].to(f64) if c["shift"] else 0.0)}
        if c["mode"] == "train":
            gy = s["grad_out"].to(f64)
            # projected off the directions that the norm takes out: u, and the constant for LayerNorm
            h = gy * w
            h = h - u * ((h * u).sum(1, keepdim=True) / n) - (h.sum(1, keepdim=True) / n if c["kind"] == "layer" else 0.0)
            out["dx"] = h / sigma
            out["dgain"] = torch.einsum("rc,rc->c", gy, u)
            if c["shift"]:
                out["dshift"] = gy.sum(0)
        return out
    N, D, V, train = c["rows"], c["hidden"], c["vocab"], c["mode"] == "train"
    w = s["w"].to(f64)
    b = s["bias"].to(f64) if c["bias"] else 0.0
    loss, lse = torch.zeros(N, dtype=f64, device="cuda"), torch.zeros(N, dtype=f64, device="cuda")
    if train:
        dx = torch.zeros(N, D, dtype=f64, device="cuda")
        dw = torch.zeros(V, D, dtype=f64, device="cuda")
        db = torch.zeros(V, dtype=f64, device="cuda")
    T = c.get("temperature", 1.0)
    if c["family"] == "xent":
        entries, weights = s["labels"][:, None], None
    else:
        entries = s["index"]
        weights = torch.softmax(s["teacher"].to(f64) / T, 1)     # (a row has all of its entries, or none)
    rows = torch.nonzero((entries >= 0).any(1)).squeeze(1)
    for part in rows.split(max(1, int(4e8 / V))):
        x = s["x"][part].to(f64)
        z = (x @ w.t() + b) / T
        log_z = torch.logsumexp(z, 1)
        lse[part] = log_z
        q = torch.ones(len(part), 1, dtype=f64, device="cuda") if weights is None else weights[part]
        log_p = z.gather(1, entries[part]) - log_z[:, None]
        loss[part] = T * T * (torch.special.xlogy(q, q) - q * log_p).sum(1)
        if train:
            grad = torch.exp(z - log_z[:, None])
            grad.scatter_add_(1, entries[part], -q)
            grad *= (s["grad_loss"][part].to(f64) * T)[:, None]
            dx[part] = grad @ w
            dw += grad.t() @ x
            db += grad.sum(0)
    out = {"loss": loss, "lse": lse}
    if train:
        out["dx"], out["dw"] = dx, dw if c["weight"] == "vd" else dw.t().contiguous().t()
        if c["bias"]:
            out["dbias"] = db
    return out


# ------------------------------------------------------------------------------------- what it takes

def work(case):
    """Each input once, each output once; the products that have to be made.  A head's training pass is three products of
    the rows that count; that a path which keeps no logits makes the first of them twice is not counted."""
    c = case
    e = 4.0 if c["dtype"] == "fp32" else 2.0
    if c["family"] == "norm":
        R, C = c["rows"], c["cols"]
        train = c["mode"] == "train"
        pe = 4.0 if c["param"] == "fp32" else e
        params = (2 if c["shift"] else 1) * C * pe
        return {"bytes": R * C * e * (4 if train else 2) + params * (2 if train else 1), "flops": R * C * (16.0 if train else 6.0)}
    N, D, V = c["rows"], c["hidden"], c["vocab"]
    active = N - int(c["ignored"] * N)
    train = c["mode"] == "train"
    nbytes = e * (active * D + V * D + (V if c["bias"] else 0)) + 8.0 * N
    nbytes += 8.0 * N if c["family"] == "xent" else (8.0 + e) * N * c["k"]
    if train:
        nbytes += e * (N * D + V * D + (V if c["bias"] else 0)) + 4.0 * N
    return {"bytes": nbytes, "flops": (6.0 if train else 2.0) * active * D * V}

"""Operators of a residual network's block and head, as measured work.

Three operators, forward alone ("fwd") or forward and backward ("step"):

  norm      layer norm over the last axis, with the residual sum in front of it
  linear    x W^T + b, an activation, and a residual added behind it
  logprobs  log probability of a target per row of logits, the row's entropy
            and its top alternatives

``run`` computes them in plain torch operations in 32 bits, or, where ``own``
is true, through cpd_amd's public entry points.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16,
          "float16": torch.float16}
EPS = 1e-5
IGNORE = -100


def listed():
    return [
        # one token of a sequence that is being generated: latency
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 4096,
         "dtype": "bfloat16", "residual": True, "mode": "fwd"},
        # many short, odd rows in full precision (per-head or per-patch norms)
        {"name": "norm_ragged", "op": "norm", "rows": 20011, "cols": 257,
         "dtype": "float32", "residual": False, "mode": "step"},
        # a training step's norm in front of a block, with the residual stream
        {"name": "norm_block", "op": "norm", "rows": 8192, "cols": 4096,
         "dtype": "bfloat16", "residual": True, "mode": "step"},
        # one token through a widening layer: bound by reading the weight
        {"name": "linear_token", "op": "linear", "m": 1, "k": 4096,
         "n": 16384, "dtype": "bfloat16", "act": "gelu", "residual": False,
         "mode": "fwd"},
        # a small batch of tokens through a narrowing layer and its residual
        {"name": "linear_batch", "op": "linear", "m": 48, "k": 16384,
         "n": 4096, "dtype": "bfloat16", "act": "none", "residual": True,
         "mode": "fwd"},
        # a training step of the widening layer
        {"name": "linear_up", "op": "linear", "m": 8192, "k": 4096,
         "n": 16384, "dtype": "bfloat16", "act": "gelu", "residual": False,
         "mode": "step"},
        # a training step of odd sizes in half precision, all of the epilogue
        {"name": "linear_ragged", "op": "linear", "m": 1023, "k": 5000,
         "n": 2050, "dtype": "float16", "act": "silu", "residual": True,
         "mode": "step"},
        # an image classifier's head in full precision: 2048 features, 1000
        # classes
        {"name": "linear_head", "op": "linear", "m": 512, "k": 2048,
         "n": 1000, "dtype": "float32", "act": "none", "residual": False,
         "mode": "step"},
        # the logits of one generated token, with alternatives
        {"name": "logprobs_token", "op": "logprobs", "rows": 1,
         "vocab": 128000, "dtype": "bfloat16", "top_k": 8, "mode": "fwd"},
        # a validation batch of ten classes: loss, top-1 and top-5 of images
        {"name": "logprobs_images", "op": "logprobs", "rows": 512,
         "vocab": 10, "dtype": "float32", "top_k": 5, "mode": "fwd"},
        # a training step's loss over an odd vocabulary, with the gradient of
        # an entropy term
        {"name": "logprobs_train", "op": "logprobs", "rows": 4096,
         "vocab": 50021, "dtype": "bfloat16", "top_k": 0, "mode": "step"},
        # scoring given texts, with alternatives at every place
        {"name": "logprobs_score", "op": "logprobs", "rows": 2048,
         "vocab": 131072, "dtype": "float16", "top_k": 16, "mode": "fwd"},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, even over its logarithm; half are odd or
    ragged, half multiples of 64 where they are that large."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if n >= 128 and rng.random() < 0.5:
        n = n // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["norm", "linear", "logprobs"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    mode = rng.choice(["fwd", "step"])
    if op == "norm":
        cols = _size(rng, 8, 16384)
        rows = _size(rng, 1, min(65536, 33554432 // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype,
                "residual": rng.random() < 0.5, "mode": mode}
    if op == "linear":
        k, n = _size(rng, 8, 16384), _size(rng, 8, 16384)
        most = 40_000_000_000 if dtype == "float32" else 400_000_000_000
        m = _size(rng, 1, max(1, min(16384, most // (k * n))))
        # relu's slope jumps at zero, and two orders of a sum may fall on both
        # sides of it: in 32 bits it is compared forward only
        acts = ["none", "gelu", "silu"]
        if dtype != "float32" or mode == "fwd":
            acts.append("relu")
        return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype,
                "act": rng.choice(acts),
                "residual": rng.random() < 0.5, "mode": mode}
    vocab = _size(rng, 16, 131072)
    rows = _size(rng, 1, min(16384, 201326592 // vocab))
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype,
            "top_k": rng.choice([0, 1, 5, 8, 16]), "mode": mode}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    step = case["mode"] == "step"

    def normal(*shape, scale=1.0, shift=0.0):
        t = torch.randn(*shape, device="cuda", generator=g)
        return t.mul_(scale).add_(shift).to(dt)

    s = {"case": case}
    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        # a residual stream: some features much larger than the others, and
        # a mean that is not zero
        loud = torch.rand(c, device="cuda", generator=g) < 0.01
        x = torch.randn(r, c, device="cuda", generator=g)
        s["x"] = (x * torch.where(loud, 12.0, 1.0) + 0.25).to(dt)
        s["res"] = normal(r, c, scale=0.5) if case["residual"] else None
        s["w"] = normal(c, scale=0.2, shift=1.0)
        s["b"] = normal(c, scale=0.1)
        if step:
            s["dy"] = normal(r, c, scale=0.05)
            s["ds"] = normal(r, c, scale=0.05) if case["residual"] else None
        learned = ["x", "res", "w", "b"]
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k)
        s["w"] = normal(n, k, scale=k ** -0.5)
        s["b"] = normal(n, scale=0.2)
        s["res"] = normal(m, n) if case["residual"] else None
        if step:
            s["dy"] = normal(m, n, scale=0.05)
        learned = ["x", "w", "b", "res"]
    else:
        r, v = case["rows"], case["vocab"]
        x = torch.randn(r, v, device="cuda", generator=g).mul_(2.0)
        # rows of every sharpness; the last entries of the vocabulary are
        # padding that no row may choose; some targets are to be passed over
        x *= torch.rand(r, 1, device="cuda", generator=g) * 2 + 0.25
        real = max(1, v - v // 40)
        x[:, real:] = -math.inf
        s["x"] = x.to(dt)
        t = torch.randint(0, real, (r,), device="cuda", generator=g)
        skip = torch.rand(r, device="cuda", generator=g) < 0.1
        s["t"] = torch.where(skip, torch.full_like(t, IGNORE), t) \
            if r > 1 else t
        if step:
            s["glp"] = torch.randn(r, device="cuda", generator=g)
            s["gent"] = torch.randn(r, device="cuda", generator=g) * 0.1
        learned = ["x"]
    if step:
        for name in learned:
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear,
                "logprobs": _own_logprobs}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "linear": _plain_linear,
                "logprobs": _plain_logprobs}[op](state)


# -- the framework's calls ---------------------------------------------------

def _own_norm(s):
    from cpd_amd.models import fused_layer_norm
    out = fused_layer_norm(s["x"], s["w"], s["b"], eps=EPS, residual=s["res"])
    y, total = out if s["res"] is not None else (out, None)
    if s["case"]["mode"] == "fwd":
        return {"y": y, "s": total}
    if total is None:
        dx, dw, db = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    dx, dres, dw, db = torch.autograd.grad(
        [y, total], [s["x"], s["res"], s["w"], s["b"]], [s["dy"], s["ds"]])
    return {"y": y.detach(), "s": total.detach(), "dx": dx, "dres": dres,
            "dw": dw, "db": db}


def _own_linear(s):
    from cpd_amd.models import fused_linear
    act = s["case"]["act"]
    y = fused_linear(s["x"], s["w"], s["b"],
                     activation=None if act == "none" else act,
                     residual=s["res"])
    if s["case"]["mode"] == "fwd":
        return {"y": y}
    leaves = [s["x"], s["w"], s["b"]] + ([s["res"]] if s["case"]["residual"]
                                         else [])
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y.detach(),
            **dict(zip(["dx", "dw", "db", "dres"], grads))}


def _own_logprobs(s):
    from cpd_amd.utils import token_logprobs
    out = token_logprobs(s["x"], s["t"], top_k=s["case"]["top_k"],
                         ignore_index=IGNORE)
    got = {"logprobs": out.logprobs, "entropy": out.entropy,
           "top_ids": out.top_ids, "top_logprobs": out.top_logprobs}
    if s["case"]["mode"] == "step":
        got["dx"] = torch.autograd.grad(
            [out.logprobs, out.entropy], s["x"], [s["glp"], s["gent"]])[0]
        got = {k: v if v is None else v.detach() for k, v in got.items()}
    return got


# -- plain forms -------------------------------------------------------------

def _plain_norm(s):
    dt = s["x"].dtype
    total = s["x"].float()
    if s["res"] is not None:
        # the sum is an output of its own; the norm is of what it holds
        total = (total + s["res"].float()).to(dt).float()
    w, b = s["w"].float(), s["b"].float()
    centred = total - total.mean(-1, keepdim=True)
    rstd = (centred.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hat = centred * rstd
    y = (hat * w + b).to(dt)
    got = {"y": y, "s": total.to(dt) if s["res"] is not None else None}
    if s["case"]["mode"] == "fwd":
        return got
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True)
                 - hat * (g * hat).mean(-1, keepdim=True))
    if s["res"] is not None:
        dx = dx + s["ds"].float()
    dx = dx.to(dt)
    got.update(dx=dx, dw=(dy * hat).sum(0).to(dt), db=dy.sum(0).to(dt))
    if s["res"] is not None:
        got["dres"] = dx.clone()
    return got


def _act(z, act):
    """The activation's value and its derivative."""
    if act == "relu":
        return z.clamp_min(0), (z > 0).float()
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(
            2 * math.pi)
    if act == "silu":
        sig = torch.sigmoid(z)
        return z * sig, sig * (1 + z * (1 - sig))
    return z, None


def _plain_linear(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t() + s["b"].float()
    a, slope = _act(z, s["case"]["act"])
    if s["res"] is not None:
        a = a + s["res"].float()
    got = {"y": a.to(dt)}
    if s["case"]["mode"] == "fwd":
        return got
    dz = s["dy"].float()
    if slope is not None:
        dz = dz * slope
    got.update(dx=(dz @ w).to(dt), dw=(dz.t() @ x).to(dt),
               db=dz.sum(0).to(dt))
    if s["res"] is not None:
        got["dres"] = s["dy"].clone()
    return got


def _plain_logprobs(s):
    x, k = s["x"].float(), s["case"]["top_k"]
    kept = s["t"] != IGNORE
    t = torch.where(kept, s["t"], 0)
    shifted = x - x.amax(-1, keepdim=True)
    e = shifted.exp()
    total = e.sum(-1, keepdim=True)
    p = e / total
    logp = shifted - total.log()
    safe = torch.where(p > 0, logp, 0.0)
    entropy = -(p * safe).sum(-1)
    chosen = logp.gather(-1, t[:, None])[:, 0]
    got = {"logprobs": torch.where(kept, chosen, 0.0),
           "entropy": torch.where(kept, entropy, 0.0),
           "top_ids": None, "top_logprobs": None}
    if k:
        # equal values: the lowest index first
        ids = torch.sort(x, dim=-1, descending=True,
                         stable=True)[1][:, :k]
        got["top_ids"] = torch.where(kept[:, None], ids, -1)
        got["top_logprobs"] = torch.where(kept[:, None], logp.gather(-1, ids),
                                          -math.inf)
    if s["case"]["mode"] == "step":
        glp = torch.where(kept, s["glp"], 0.0)[:, None]
        gent = torch.where(kept, s["gent"], 0.0)[:, None]
        dx = -p * (glp + gent * (safe + entropy[:, None]))
        dx.scatter_add_(-1, t[:, None], glp)
        got["dx"] = dx.to(s["x"].dtype)
    return got


# -- what one pass cannot do without -----------------------------------------

def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    step = case["mode"] == "step"
    if case["op"] == "norm":
        n, c = case["rows"] * case["cols"], case["cols"]
        through = 4 if case["residual"] else 2      # x, y, and res, s
        vectors = 2 * c
        if step:
            through += 4 if case["residual"] else 2  # dy, dx, and ds, dres
            vectors += 2 * c
        return {"bytes": size * (through * n + vectors),
                "flops": (24 if step else 9) * n}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        res = m * n if case["residual"] else 0
        values = m * k + n * k + n + m * n + res
        if step:
            values += m * n + m * k + n * k + n + res
        return {"bytes": size * values,
                "flops": (6 if step else 2) * m * n * k}
    r, v, top = case["rows"], case["vocab"], case["top_k"]
    moved = size * r * v * (2 if step else 1) + r * (8 + 4 + 4 + 12 * top)
    return {"bytes": moved + (8 * r if step else 0),
            "flops": (12 if step else 5) * r * v}


# -- 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    leaf = {k: v.detach().double() for k, v in s.items()
            if isinstance(v, torch.Tensor) and v.is_floating_point()}
    step = case["mode"] == "step"
    names = {"norm": ["x", "w", "b"], "linear": ["x", "w", "b"],
             "logprobs": ["x"]}[case["op"]]
    if step:
        for name in names:
            leaf[name].requires_grad_(True)
    with torch.set_grad_enabled(step):
        if case["op"] == "norm":
            total = leaf["x"]
            if s["res"] is not None:
                # the operator normalises the sum as it is stored; rounding
                # is passed through unchanged by the gradient
                held = (total + leaf["res"]).to(s["x"].dtype).double()
                total = total + (held - total).detach()
            var, mean = torch.var_mean(total, -1, correction=0, keepdim=True)
            y = (total - mean) / torch.sqrt(var + EPS) * leaf["w"] + leaf["b"]
            got = {"y": y, "s": total if s["res"] is not None else None}
            if step:
                loss = (y * leaf["dy"]).sum()
                if s["res"] is not None:
                    loss = loss + (total * leaf["ds"]).sum()
        elif case["op"] == "linear":
            z = torch.addmm(leaf["b"], leaf["x"], leaf["w"].t())
            a = {"none": lambda v: v, "relu": torch.relu,
                 "gelu": torch.nn.functional.gelu,
                 "silu": torch.nn.functional.silu}[case["act"]](z)
            got = {"y": a + leaf["res"] if s["res"] is not None else a}
            if step:
                loss = (got["y"] * leaf["dy"]).sum()
        else:
            kept = s["t"] >= 0
            lp = torch.log_softmax(leaf["x"], -1)
            finite = torch.where(torch.isinf(lp), torch.zeros_like(lp), lp)
            chosen = lp[torch.arange(case["rows"], device=lp.device),
                        s["t"].clamp_min(0)]
            ent = -(torch.exp(lp) * finite).sum(-1)
            zero = torch.zeros_like(ent)
            got = {"logprobs": torch.where(kept, chosen, zero),
                   "entropy": torch.where(kept, ent, zero),
                   "top_ids": None, "top_logprobs": None}
            if case["top_k"]:
                top = torch.topk(lp.detach(), case["top_k"], -1)[0]
                got["top_logprobs"] = torch.where(
                    kept[:, None], top, torch.full_like(top, -math.inf))
            if step:
                loss = (got["logprobs"] * leaf["glp"]
                        + got["entropy"] * leaf["gent"]).sum()
    if step:
        grads = torch.autograd.grad(loss, [leaf[n] for n in names])
        got.update(zip(["dx", "dw", "db"], grads))
        if s.get("res") is not None:
            got["dres"] = got["dx"] if case["op"] == "norm" else leaf["dy"]
        got = {k: v if v is None else v.detach() for k, v in got.items()}
    return got

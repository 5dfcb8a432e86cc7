"""Measured cases of the sequence operators: the linear / gated recurrence and
its gradient, the embedding lookup and its gradient, clipping by the global
norm.  ``run`` computes them in plain torch operations where ``own`` is false
and calls this repository's operators where it is true; ``exact`` evaluates
their definitions in 64 bits."""

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "f32": torch.float32, "f64": torch.float64}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one token of each of 32 running sequences: latency of a decode step
        {"name": "step_f16", "op": "rec", "dtype": "f16", "gated": True, "batch": 32, "steps": 1, "width": 2048,
         "packed": True, "h0": True},
        # a training batch; gate and candidate are the halves of one projection's output
        {"name": "train_f16", "op": "rec", "dtype": "f16", "gated": True, "batch": 8, "steps": 2048, "width": 2048,
         "packed": True, "h0": False},
        # one long document through a layer of odd width, as its prompt is read in
        {"name": "long_f32", "op": "rec", "dtype": "f32", "gated": False, "batch": 1, "steps": 65521, "width": 1000,
         "packed": False, "h0": True},
        # a ragged double-precision batch: the numerics check a user runs beside a model
        {"name": "ragged_f64", "op": "rec", "dtype": "f64", "gated": True, "batch": 3, "steps": 1001, "width": 257,
         "packed": False, "h0": True},
        # the backward pass of the training batch
        {"name": "train_grad_f16", "op": "rec_grad", "dtype": "f16", "gated": True, "batch": 8, "steps": 2048,
         "width": 2048, "packed": True, "h0": False},
        # the backward pass over long sequences cut for truncated backpropagation (state and its gradient passed on)
        {"name": "long_grad_f32", "op": "rec_grad", "dtype": "f32", "gated": False, "batch": 2, "steps": 16383,
         "width": 1536, "packed": False, "h0": True},
        # the tokens of one decode step
        {"name": "tokens_f16", "op": "emb", "dtype": "f16", "tokens": 32, "rows": 32000, "width": 2048,
         "ids": "int64"},
        # the tokens of a training batch, a large vocabulary
        {"name": "batch_f32", "op": "emb", "dtype": "f32", "tokens": 16384, "rows": 128000, "width": 1024,
         "ids": "int32"},
        # a small vocabulary and batch: latency of the sorted gradient
        {"name": "tokens_grad_f32", "op": "emb_grad", "dtype": "f32", "tokens": 512, "rows": 8192, "width": 768,
         "ids": "int64"},
        # the training batch's gradient over the whole vocabulary
        {"name": "batch_grad_f16", "op": "emb_grad", "dtype": "f16", "tokens": 16384, "rows": 50257, "width": 2048,
         "ids": "int64"},
        # the gradients of a toy model: latency over many small arrays
        {"name": "clip_small", "op": "clip", "dtype": "f32", "layers": 2, "width": 128, "rows": 1000},
        # the gradients of a model of some 350 million weights, matrices in half and vectors in single precision
        {"name": "clip_large", "op": "clip", "dtype": "mixed", "layers": 24, "width": 1024, "rows": 50257},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rec", "rec", "rec_grad", "rec_grad", "emb", "emb_grad", "emb_grad", "clip"])
    if op in ("rec", "rec_grad"):
        dtype = rng.choice(["f16", "f16", "f32", "f32", "f64"])
        most = (1 << 25) // (2 if op == "rec_grad" else 1) // (2 if dtype == "f64" else 1)
        width = _log(rng, 64, 4096)
        steps = min(_log(rng, 1, 65536), most // width)
        return {"op": op, "dtype": dtype, "gated": rng.random() < 0.5,
                "batch": min(_log(rng, 1, 64), most // (width * steps)), "steps": steps, "width": width,
                "packed": rng.random() < 0.5, "h0": rng.random() < 0.5}
    if op in ("emb", "emb_grad"):
        rows, width = _log(rng, 256, 131072), _log(rng, 64, 4096)
        return {"op": op, "dtype": rng.choice(["f16", "f32"]), "tokens": _log(rng, 1, 32768),
                "rows": min(rows, (1 << 27) // width), "width": width, "ids": rng.choice(["int32", "int64"])}
    return {"op": op, "dtype": rng.choice(["f16", "f32", "mixed"]), "layers": rng.randint(1, 16),
            "width": _log(rng, 64, 1024), "rows": _log(rng, 256, 50257)}


# ------------------------------------------------------------------ inputs

def _name(dtype):
    return str(dtype).replace("torch.", "")


def _acc(dtype):
    """The type sums and states are held in."""
    return torch.float64 if dtype == torch.float64 else torch.float32


def _shapes(case):
    """The weight shapes of a stack of layers: four square matrices, two wide
    ones and their vectors in each, and one table of rows."""
    d = case["width"]
    layer = [(d, d)] * 4 + [(4 * d, d), (d, 4 * d)] + [(d,)] * 5 + [(4 * d,)]
    return [(case["rows"], d)] + layer * case["layers"] + [(d,)]


def _ids(case, gen, n):
    """Token ids as frequent as a text's words: P(id) falls as 1 / (id + 1)."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(case["rows"] + 1)) - 1).long().clamp_(0, case["rows"] - 1).to(
        getattr(torch, case["ids"]))


def _inputs(case, seed):
    """The inputs as torch tensors, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, mean=0.0, std=1.0):
        t = torch.empty(shape, dtype=torch.float64 if dtype == torch.float64 else torch.float32, device="cuda")
        return t.normal_(mean, std, generator=gen).to(dtype)

    op = case["op"]
    if op in ("rec", "rec_grad"):
        dt = DTYPES[case["dtype"]]
        shape = (case["batch"], case["steps"], case["width"])
        # gates are logits that remember some tens to hundreds of steps; plain decays lie in (0.5, 1)
        a = normal(shape, dt, 3.0, 1.5) if case["gated"] else torch.sigmoid(normal(shape, torch.float32, 3.0, 1.5)).to(dt)
        x = normal(shape, dt)
        s = {}
        if case["packed"]:
            s["packed"] = torch.cat([a, x], -1)
            a, x = s["packed"][..., :case["width"]], s["packed"][..., case["width"]:]
        s["a"], s["x"] = a, x
        state = (case["batch"], case["width"])
        if case["h0"]:
            s["h0"] = normal(state, _acc(dt))
        if op == "rec_grad":
            s["h"] = _recurrence(case, s)["h"]
            s["grad"] = normal(shape, dt)
            if case["h0"]:
                s["grad_state"] = normal(state, _acc(dt))
        return s
    if op == "emb":
        return {"weight": normal((case["rows"], case["width"]), DTYPES[case["dtype"]], 0.0, 0.02),
                "ids": _ids(case, gen, case["tokens"]), "scale": math.sqrt(case["width"])}
    if op == "emb_grad":
        return {"ids": _ids(case, gen, case["tokens"]), "scale": math.sqrt(case["width"]),
                "grad": normal((case["tokens"], case["width"]), DTYPES[case["dtype"]], 0.0, 0.1)}
    kind = case["dtype"]
    dts = [DTYPES[kind] if kind != "mixed" else torch.float16 if len(sh) == 2 else torch.float32
           for sh in _shapes(case)]
    return {"grads": [normal(sh, dt, 0.0, 0.01) for sh, dt in zip(_shapes(case), dts)], "max_norm": 1.0}


def _flat(case, grads, new):
    """One buffer per dtype, made by ``new(n, dtype)``, and each array's place
    in it: the clipped gradients lie there one after another, each from a
    multiple of 128 elements on."""
    sizes, places = {}, []
    for g in grads:
        at = sizes.get(g.dtype, 0)
        places.append((g.dtype, at, g.numel(), tuple(g.shape)))
        sizes[g.dtype] = at + -(-g.numel() // 128) * 128
    flats = {dt: new(n, dt) for dt, n in sizes.items()}
    return flats, [flats[dt][at:at + n].reshape(shape) for dt, at, n, shape in places]


def _own_arrays(case, s):
    """The same inputs as arrays of this package, which is what its user holds,
    with the output arrays that a loop over steps uses again."""
    import macmetalpy_b200 as cp

    arrays, views = {}, {}

    def wrap(t):
        a = cp.empty(tuple(t.shape), dtype=_name(t.dtype))
        cp.synchronize()
        torch.as_tensor(a, device="cuda").copy_(t)
        return a

    def output(name, shape, dtype):
        a = arrays[name] = cp.empty(tuple(shape), dtype=_name(dtype))
        views[name] = torch.as_tensor(a, device="cuda")

    for k, v in s.items():
        if isinstance(v, torch.Tensor) and not ("packed" in s and k in ("a", "x")):
            arrays[k] = wrap(v)
        elif isinstance(v, list):
            arrays[k] = [wrap(t) for t in v]
        elif not isinstance(v, torch.Tensor):
            arrays[k] = v
    if "packed" in s:
        w = case["width"]
        arrays["a"], arrays["x"] = arrays["packed"][..., :w], arrays["packed"][..., w:]
    op = case["op"]
    if op in ("rec", "rec_grad"):
        shape, dt = s["x"].shape, s["x"].dtype
        state = (shape[0], shape[2])
        if op == "rec":
            output("out_h", shape, dt)
            output("out_state", state, _acc(dt))
        else:
            output("out_a", shape, dt)
            output("out_x", shape, dt)
            if case["h0"]:
                output("out_h0", state, _acc(dt))
    elif op == "emb":
        output("out", (case["tokens"], case["width"]), s["weight"].dtype)
    elif op == "emb_grad":
        output("out", (case["rows"], case["width"]), s["grad"].dtype)
    else:
        flats, arrays["outs"] = _flat(case, s["grads"], lambda n, dt: cp.zeros(n, dtype=_name(dt)))
        arrays["norm"] = cp.empty((), dtype="float32")
        views["grads"] = {_name(dt): torch.as_tensor(f, device="cuda") for dt, f in flats.items()}
        views["norm"] = torch.as_tensor(arrays["norm"], device="cuda")
    cp.synchronize()
    return {"case": case, "arrays": arrays, "views": views}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # arrays of this package instead of torch tensors
        return _own_arrays(case, s)
    if case["op"] == "clip":
        s["flats"], s["outs"] = _flat(case, s["grads"], lambda n, dt: torch.zeros(n, dtype=dt, device="cuda"))
    s["case"] = case
    return s


# ------------------------------------------------------------------ plain forms

def _scan(f, u):
    """h_t = f_t h_{t-1} + u_t from h = 0 along axis 1, by doubling: after the
    step of width n, each entry stands for its last 2 n steps."""
    n, steps = 1, u.shape[1]
    while n < steps:
        u = torch.cat([u[:, :n], u[:, n:] + f[:, n:] * u[:, :-n]], 1)
        if 2 * n < steps:
            f = torch.cat([f[:, :n], f[:, n:] * f[:, :-n]], 1)
        n *= 2
    return u


def _gates(case, s):
    """(f, 1 - f) of the recurrence, in the type that sums are held in."""
    a = s["a"].to(_acc(s["a"].dtype))
    return (torch.sigmoid(a), torch.sigmoid(-a)) if case["gated"] else (a, None)


def _recurrence(case, s):
    f, rest = _gates(case, s)
    x = s["x"].to(f.dtype)
    u = rest * x if case["gated"] else x
    if "h0" in s:
        u = torch.cat([u[:, :1] + f[:, :1] * s["h0"][:, None], u[:, 1:]], 1)
    h = _scan(f, u)
    return {"h": h.to(s["x"].dtype), "state": h[:, -1].clone()}


def _recurrence_grad(case, s):
    f, rest = _gates(case, s)
    dh, h = s["grad"].to(f.dtype), s["h"].to(f.dtype)
    first = s["h0"][:, None] if "h0" in s else torch.zeros_like(h[:, :1])
    before = torch.cat([first, h[:, :-1]], 1)
    if "grad_state" in s:
        dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["grad_state"][:, None]], 1)
    # g_t = dh_t + f_{t+1} g_{t+1}, from the last step to the first
    after = torch.cat([torch.zeros_like(f[:, :1]), f.flip(1)[:, :-1]], 1)
    g = _scan(after, dh.flip(1)).flip(1)
    if case["gated"]:
        da, dx = g * (before - s["x"].to(f.dtype)) * f * rest, g * rest
    else:
        da, dx = g * before, g
    out = {"da": da.to(s["a"].dtype), "dx": dx.to(s["x"].dtype)}
    if case["h0"]:
        out["dh0"] = f[:, 0] * g[:, 0]
    return out


def _embedding(case, s):
    return {"out": (s["weight"][s["ids"].long()].float() * s["scale"]).to(s["weight"].dtype)}


def _embedding_grad(case, s):
    rows = torch.zeros(case["rows"], case["width"], device="cuda", dtype=torch.float32)
    rows.index_add_(0, s["ids"].long(), s["grad"].float())
    return {"grad": (rows * s["scale"]).to(s["grad"].dtype)}


def _clip(case, s):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = torch.where(norm <= s["max_norm"], torch.ones_like(norm), s["max_norm"] / norm).float()
    _ = [out.copy_(g.float() * coef) for out, g in zip(s["outs"], s["grads"])]
    return {"grads": {_name(dt): f for dt, f in s["flats"].items()}, "norm": norm.float()}


# ------------------------------------------------------------------ one pass

def _run_own(state):
    import macmetalpy_b200 as cp

    case, a, v = state["case"], state["arrays"], state["views"]
    op = case["op"]
    if op == "rec":
        cp.linear_recurrence(a["a"], a["x"], a.get("h0"), gated=case["gated"], out=a["out_h"],
                             state_out=a["out_state"])
        return {"h": v["out_h"], "state": v["out_state"]}
    if op == "rec_grad":
        outs = (a["out_a"], a["out_x"]) + ((a["out_h0"],) if case["h0"] else ())
        cp.linear_recurrence_grad(a["a"], a["x"], a["h"], a["grad"], a.get("h0"), gated=case["gated"],
                                  grad_state=a.get("grad_state"), out=outs)
        return {"da": v["out_a"], "dx": v["out_x"], **({"dh0": v["out_h0"]} if case["h0"] else {})}
    if op == "emb":
        cp.embedding(a["weight"], a["ids"], a["scale"], out=a["out"])
        return {"out": v["out"]}
    if op == "emb_grad":
        cp.embedding_grad(a["ids"], a["grad"], case["rows"], a["scale"], out=a["out"])
        return {"grad": v["out"]}
    cp.clip_by_global_norm(a["grads"], a["max_norm"], out=a["outs"], norm_out=a["norm"])
    return {"grads": v["grads"], "norm": v["norm"]}


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    return {"rec": _recurrence, "rec_grad": _recurrence_grad, "emb": _embedding, "emb_grad": _embedding_grad,
            "clip": _clip}[case["op"]](case, state)


# ------------------------------------------------------------------ floors and definitions

def work(case):
    op = case["op"]
    if op in ("rec", "rec_grad"):
        e = {"f16": 2, "f32": 4, "f64": 8}[case["dtype"]]
        chains = case["batch"] * case["width"]
        n, state = chains * case["steps"], chains * max(e, 4)
        if op == "rec":  # a, x and the first state in; h and the last state out
            return {"bytes": 3 * n * e + state * (1 + case["h0"]), "flops": n * (8 if case["gated"] else 2)}
        # a, h, grad (x where gated) in; the gradients of a and x out; three states where there are states
        return {"bytes": (6 if case["gated"] else 5) * n * e + 3 * state * case["h0"],
                "flops": n * (12 if case["gated"] else 4)}
    if op in ("emb", "emb_grad"):
        e = 2 if case["dtype"] == "f16" else 4
        n, v = case["tokens"], case["rows"]
        # of ids as frequent as 1 / (id + 1), the expected number of distinct ones: a lookup reads each row once
        rank = torch.arange(1, v + 1, dtype=torch.float64)
        p = torch.log((rank + 1) / rank) / math.log(v + 1)
        rows = float((1 - (1 - p) ** n).sum()) if op == "emb" else v
        return {"bytes": (n + rows) * case["width"] * e + n * (8 if case["ids"] == "int64" else 4),
                "flops": n * case["width"]}
    n = [math.prod(sh) * (2 if case["dtype"] == "f16" or case["dtype"] == "mixed" and len(sh) == 2 else 4)
         for sh in _shapes(case)]
    return {"bytes": 2 * sum(n), "flops": 3 * sum(math.prod(sh) for sh in _shapes(case))}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("rec", "rec_grad"):
        f = s["a"].double()
        if case["gated"]:
            f = 1 / (1 + torch.exp(-f))
        x = s["x"].double()
        h0 = s["h0"].double() if case["h0"] else torch.zeros_like(x[:, 0])
        steps = case["steps"]
        if op == "rec":  # step by step
            h, out = h0, torch.empty_like(x)
            for t in range(steps):
                u = (1 - f[:, t]) * x[:, t] if case["gated"] else x[:, t]
                h = torch.addcmul(u, f[:, t], h)
                out[:, t] = h
            return {"h": out, "state": h}
        dh, h = s["grad"].double(), s["h"].double()
        c = s["grad_state"].double() if case["h0"] else torch.zeros_like(h0)
        da, dx = torch.empty_like(x), torch.empty_like(x)
        for t in range(steps - 1, -1, -1):
            g = dh[:, t] + c
            h1 = h[:, t - 1] if t else h0
            if case["gated"]:
                rest = 1 - f[:, t]
                da[:, t] = g * (h1 - x[:, t]) * f[:, t] * rest
                dx[:, t] = g * rest
            else:
                da[:, t] = g * h1
                dx[:, t] = g
            c = f[:, t] * g
        return {"da": da, "dx": dx, **({"dh0": c} if case["h0"] else {})}
    if op == "emb":
        return {"out": torch.index_select(s["weight"], 0, s["ids"].long()).double() * s["scale"]}
    if op == "emb_grad":  # differences of a running sum over the sorted tokens
        ids, order = torch.sort(s["ids"].long(), stable=True)
        total = torch.cumsum(s["grad"][order].double(), 0)
        last = torch.nonzero(torch.cat([ids[1:] != ids[:-1], torch.ones_like(ids[:1], dtype=torch.bool)]))[:, 0]
        ends = total[last]
        rows = torch.zeros(case["rows"], case["width"], device="cuda", dtype=torch.float64)
        rows[ids[last]] = (ends - torch.cat([torch.zeros_like(ends[:1]), ends[:-1]])) * s["scale"]
        return {"grad": rows}
    norm = math.sqrt(math.fsum(float(torch.dot(g.double().reshape(-1), g.double().reshape(-1))) for g in s["grads"]))
    coef = 1.0 if norm <= s["max_norm"] else s["max_norm"] / norm
    flats, places = _flat(case, s["grads"], lambda n, dt: torch.zeros(n, dtype=torch.float64, device="cuda"))
    for place, g in zip(places, s["grads"]):
        place.copy_(g.double() * coef)
    return {"grads": {_name(dt): f for dt, f in flats.items()}, "norm": norm}

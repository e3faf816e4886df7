"""The operators of a typed residual block and of its training step, as they are measured.

    grouped products   y_i = W_{t(i)} x_i + b_{t(i)}: rows sorted by type (node type, tissue, donor ...), one weight per type
    residual norm      r = x + scale * act(gate) * norm_post(f),  h = norm_pre(r): what stands between two blocks
    gradient clipping  the global norm of many gradient tensors and their scaling

``own`` selects the framework's kernels; otherwise the same values come from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # 16 cells of 8 tissues through one typed layer (scDeepSort's 400 -> 200): a single small request, latency is what counts
        dict(name="grouped_request", op="grouped", dir="fwd", dtype="f32", rows=16, types=8, skew=0.0, k=400, n=200),
        # a mini-batch of 500 cells of 17 tissues, forward and all gradients
        dict(name="grouped_batch500", op="grouped", dir="train", dtype="f32", rows=500, types=17, skew=1.0, k=400, n=200),
        # a full-batch hidden layer, very unequal types
        dict(name="grouped_hidden", op="grouped", dir="train", dtype="f32", rows=20011, types=12, skew=1.5, k=512, n=256),
        # many types with a handful of rows each (one weight per cluster): the weights are what is read
        dict(name="grouped_many_types", op="grouped", dir="fwd", dtype="bf16", rows=4099, types=700, skew=0.3, k=200, n=64),
        # the first layer over an atlas: 2000 genes -> 512, bf16 storage, forward and all gradients
        dict(name="grouped_atlas", op="grouped", dir="train", dtype="bf16", rows=200003, types=9, skew=1.0, k=2000, n=512),
        # the norm around a block for one mini-batch of 128 cells, forward only
        dict(name="norm_batch128", op="norm", dir="fwd", dtype="f32", rows=128, d=200, kind="layer", gate="scalar", gate_act="sigmoid",
             post=True, pre=True),
        # 50 principal components per spot (rows that are no multiple of 16 bytes), element gates, forward and all gradients
        dict(name="norm_spots", op="norm", dir="train", dtype="f32", rows=20001, d=50, kind="layer", gate="full", gate_act="sigmoid",
             post=True, pre=True),
        # few wide rows: one value per gene, a gate per row
        dict(name="norm_genes", op="norm", dir="train", dtype="bf16", rows=4099, d=2000, kind="rms", gate="row", gate_act="none", post=True,
             pre=True),
        # the hidden width over an atlas
        dict(name="norm_atlas", op="norm", dir="train", dtype="bf16", rows=200003, d=512, kind="layer", gate="channel", gate_act="none",
             post=True, pre=True),
        # the gradients of a graph-attention auto-encoder 2000 -> 512 -> 30 (STAGATE)
        dict(name="clip_stagate", op="clip", dtype="f32", out="same", layers="2000,512,30", copies=1, norm="2", clipped=True),
        # an auto-encoder's many small tensors, bf16 gradients into fp32 ones
        dict(name="clip_small_tensors", op="clip", dtype="bf16", out="f32", layers="200,64,32,16,7", copies=40, norm="2", clipped=True),
        # 330 million parameters
        dict(name="clip_large", op="clip", dtype="f32", out="same", layers="20000,2000,512,2000,20000", copies=4, norm="2", clipped=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["grouped", "norm", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "grouped":
        k, n = _log_int(rng, 8, 2000), _log_int(rng, 8, 600)
        rows = _log_int(rng, 1, 200000)
        rows = max(1, min(rows, int((1e11 if dtype == "bf16" else 1e10) / (k * n))))
        types = _log_int(rng, 1, max(2, min(700, int(2e8 / (k * n)))))
        return dict(op=op, dir=rng.choice(["fwd", "train"]), dtype=dtype, rows=rows, types=types, skew=rng.uniform(0.0, 2.0), k=k, n=n)
    if op == "norm":
        d = _log_int(rng, 16, 8192)
        rows = max(1, min(_log_int(rng, 1, 400000), int(1e8 / d)))
        post, pre = rng.choice([(True, True), (True, False), (False, True)])
        return dict(op=op, dir=rng.choice(["fwd", "train"]), dtype=dtype, rows=rows, d=d, kind=rng.choice(["layer", "rms"]),
                    gate=rng.choice(["none", "scalar", "channel", "row", "full"]), gate_act=rng.choice(["none", "sigmoid"]), post=post, pre=pre)
    layers = [_log_int(rng, 4, 3000) for _ in range(rng.randint(1, 5))]
    copies = _log_int(rng, 1, 60)
    while copies > 1 and copies * sum(a * b for a, b in zip(layers, layers[1:])) > 1e8:
        copies //= 2
    return dict(op=op, dtype=dtype, out=rng.choice(["same", "f32"]), layers=",".join(map(str, layers)), copies=copies, norm=rng.choice(["2", "2", "2", "inf", "1"]),
                clipped=rng.random() < 0.8)


# ---- inputs --------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _group_ptr(case, seed):
    """Row bounds of the types: multinomial sizes with weights 1 / (t + 1)^skew, types left empty by chance among them."""
    g = torch.Generator().manual_seed(int(seed) + 17)
    weights = (torch.arange(case["types"], dtype=torch.float64) + 1.0).pow(-case["skew"])
    weights = weights[torch.randperm(case["types"], generator=g)]
    ids = torch.multinomial(weights, case["rows"], replacement=True, generator=g)
    sizes = torch.bincount(ids, minlength=case["types"])
    return [0] + torch.cumsum(sizes, 0).tolist()


def _clip_shapes(case):
    layers, shapes = [int(v) for v in case["layers"].split(",")], []
    for _ in range(case["copies"]):
        for a, b in zip(layers, layers[1:]):
            shapes += [(a, b), (b, )]
        if len(layers) == 1:
            shapes.append((layers[0], ))
    return shapes


def prepare(case, seed):
    g, dt = _generator(seed), _DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    if case["op"] == "grouped":
        ptr = _group_ptr(case, seed)
        m, k, n, t = case["rows"], case["k"], case["n"], case["types"]
        st = dict(case=case, ptr_host=ptr, ptr=torch.tensor(ptr, dtype=torch.int32, device="cuda"),
                  x=torch.relu(randn(m, k)).to(dt), w=(randn(t, n, k) / math.sqrt(k)).to(dt), b=0.1 * randn(t, n))
        if case["dir"] == "train":
            st["dy"] = randn(m, n).to(dt)
            for key in ("x", "w", "b"):
                st[key].requires_grad_(True)
        return st
    if case["op"] == "norm":
        m, d = case["rows"], case["d"]
        st = dict(case=case, f=(0.3 + 1.5 * randn(m, d)).to(dt), x=randn(m, d).to(dt), gate=None, scale=0.5, eps=1e-5, w1=None, b1=None,
                  w2=None, b2=None)
        if case["gate"] != "none":
            shape = {"scalar": (1, ), "channel": (d, ), "row": (m, 1), "full": (m, d)}[case["gate"]]
            st["gate"] = 0.7 + 0.5 * randn(*shape)
            if case["gate"] in ("row", "full"):
                st["gate"] = st["gate"].to(dt)
        for i, on in (("1", case["post"]), ("2", case["pre"])):
            if on:
                st["w" + i] = 1.0 + 0.2 * randn(d)
                st["b" + i] = 0.1 * randn(d) if case["kind"] == "layer" else None
        if case["dir"] == "train":
            st["dr"] = randn(m, d).to(dt)
            st["dh"] = randn(m, d).to(dt) if case["pre"] else None
            for key in ("f", "x", "gate", "w1", "b1", "w2", "b2"):
                if st[key] is not None:
                    st[key].requires_grad_(True)
        return st
    grads = [(0.02 * randn(*s)).to(dt) for s in _clip_shapes(case)]
    out_dt = torch.float32 if case["out"] == "f32" else dt
    total = sum(t.numel() for t in grads)
    p = math.inf if case["norm"] == "inf" else float(case["norm"])
    typical = 0.06 if p == math.inf else 0.02 * (total if p == 1 else math.sqrt(total))
    # the optimiser's gradient buffer: one flat tensor, the parameters' views of it tightly packed
    flat = torch.empty(total, dtype=out_dt, device="cuda")
    out, at = [], 0
    for t in grads:
        out.append(flat[at:at + t.numel()].view(t.shape))
        at += t.numel()
    return dict(case=case, grads=grads, flat=flat, out=out, norm_type=p, max_norm=typical * (0.3 if case["clipped"] else 30.0))


# ---- one pass ------------------------------------------------------------------------------------------------------
def _grouped_own(st):
    from dance_amd import autograd, kernels
    if st["case"]["dir"] == "fwd":
        return [kernels.gemm_grouped(st["x"], st["w"], st["ptr"], trans_b=True, bias=st["b"])]
    y = autograd.grouped_linear(st["x"], st["w"], st["ptr"], st["b"])
    return [y.detach(), *torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"])]


def _grouped_plain(st):
    ptr, dt = st["ptr_host"], st["x"].dtype
    x, w, b = st["x"].detach().float(), st["w"].detach().float(), st["b"].detach()
    train = st["case"]["dir"] == "train"
    y = torch.zeros(x.shape[0], w.shape[1], device=x.device)
    if train:
        dy = st["dy"].float()
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for t in range(w.shape[0]):
        i, j = ptr[t], ptr[t + 1]
        if i == j:
            continue
        y[i:j] = torch.mm(x[i:j], w[t].t()) + b[t]
        if train:
            dx[i:j] = torch.mm(dy[i:j], w[t])
            dw[t] = torch.mm(dy[i:j].t(), x[i:j])
            db[t] = dy[i:j].sum(0)
    return [y.to(dt), dx.to(dt), dw.to(dt), db] if train else [y.to(dt)]


def _norm_own(st):
    from dance_amd import autograd
    c = st["case"]
    post = (st["w1"], st["b1"]) if c["post"] else None
    pre = (st["w2"], st["b2"]) if c["pre"] else None
    r, h = autograd.residual_norm(st["f"], st["x"], post=post, gate=st["gate"], gate_act=c["gate_act"], scale=st["scale"], pre=pre,
                                  kind=c["kind"], eps=st["eps"])
    outs = [r] if h is None else [r, h]
    if c["dir"] == "fwd":
        return outs
    leaves = [st[key] for key in ("f", "x", "gate", "w1", "b1", "w2", "b2") if st[key] is not None]
    grads = torch.autograd.grad(outs, leaves, [st["dr"]] if h is None else [st["dr"], st["dh"]])
    return [o.detach() for o in outs] + list(grads)


def _norm_stats(v, kind, eps):
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    rstd = 1.0 / torch.sqrt((v - mean).square().mean(1, keepdim=True) + eps)
    return (v - mean) * rstd, rstd


def _norm_backward(vhat, rstd, w, dout, kind):
    u = dout * w
    c1 = (u * vhat).mean(1, keepdim=True)
    c0 = u.mean(1, keepdim=True) if kind == "layer" else 0.0
    return rstd * (u - c0 - vhat * c1)


def _norm_plain(st):
    c, dt = st["case"], st["f"].dtype
    kind, eps, scale = c["kind"], st["eps"], st["scale"]
    val = {key: None if st[key] is None else st[key].detach().float() for key in ("f", "x", "gate", "w1", "b1", "w2", "b2")}
    f, x = val["f"], val["x"]
    n = f
    if c["post"]:
        fhat, rstd1 = _norm_stats(f, kind, eps)
        n = fhat * val["w1"] + (0.0 if val["b1"] is None else val["b1"])
    gate = 1.0 if val["gate"] is None else val["gate"]
    if val["gate"] is not None and c["gate_act"] == "sigmoid":
        gate = 1.0 / (1.0 + torch.exp(-gate))
    r = x + scale * gate * n
    outs = [r.to(dt)]
    if c["pre"]:
        rhat, rstd2 = _norm_stats(r, kind, eps)
        outs.append((rhat * val["w2"] + (0.0 if val["b2"] is None else val["b2"])).to(dt))
    if c["dir"] == "fwd":
        return outs
    dr = st["dr"].float()
    tail = []
    if c["pre"]:
        dh = st["dh"].float()
        dr = dr + _norm_backward(rhat, rstd2, val["w2"], dh, kind)
        tail = [(dh * rhat).sum(0)] + ([dh.sum(0)] if val["b2"] is not None else [])
    dn = scale * gate * dr
    middle = []
    if val["gate"] is not None:
        dg = scale * dr * n
        if c["gate_act"] == "sigmoid":
            dg = dg * gate * (1.0 - gate)
        dims = {"scalar": (0, 1), "channel": (0, ), "row": (1, ), "full": ()}[c["gate"]]
        dg = dg.sum(dims).reshape(st["gate"].shape) if dims else dg
        middle.append(dg.to(st["gate"].dtype))
    df = dn
    if c["post"]:
        middle += [(dn * fhat).sum(0)] + ([dn.sum(0)] if val["b1"] is not None else [])
        df = _norm_backward(fhat, rstd1, val["w1"], dn, kind)
    return outs + [df.to(dt), dr.to(dt)] + middle + tail


def _clip_own(st):
    from dance_amd import kernels
    norm = kernels.clip_grads(st["grads"], st["max_norm"], norm_type=st["norm_type"], out=st["out"])
    return [norm, st["flat"]]


def _clip_plain(st):
    p = st["norm_type"]
    if p == math.inf:
        norm = torch.stack([t.float().abs().max() for t in st["grads"]]).max()
    elif p == 1.0:
        norm = torch.stack([t.float().abs().sum(dtype=torch.float64) for t in st["grads"]]).sum()
    else:
        norm = torch.stack([t.float().square().sum(dtype=torch.float64) for t in st["grads"]]).sum().sqrt()
    factor = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0).float()
    for t, o in zip(st["grads"], st["out"]):
        o.copy_(t.float() * factor)
    return [norm.float(), st["flat"]]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"grouped": _grouped_own, "norm": _norm_own, "clip": _clip_own}[op](state)
    with torch.no_grad():
        return {"grouped": _grouped_plain, "norm": _norm_plain, "clip": _clip_plain}[op](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    s = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "grouped":
        m, k, n, t = case["rows"], case["k"], case["n"], min(case["types"], case["rows"])
        fwd_bytes = s * (m * k + t * n * k + m * n) + 4 * t * n
        if case["dir"] == "fwd":
            return {"bytes": fwd_bytes, "flops": 2 * m * n * k}
        # forward: x, w, b in, y out; backward: dy in beside the kept x and w, dx, dw, db out
        return {"bytes": fwd_bytes + s * (m * n + m * k + case["types"] * n * k) + 4 * case["types"] * n, "flops": 6 * m * n * k}
    if case["op"] == "norm":
        m, d = case["rows"], case["d"]
        gate = m * d if case["gate"] == "full" else m if case["gate"] == "row" else 0
        outs = 1 + int(case["pre"])
        fwd = s * (2 * m * d + gate + outs * m * d)
        if case["dir"] == "fwd":
            return {"bytes": fwd, "flops": 20 * m * d}
        return {"bytes": fwd + s * (2 * m * d + 2 * gate + outs * m * d + 2 * m * d), "flops": 60 * m * d}
    total = sum(math.prod(shape) for shape in _clip_shapes(case))
    # the scaling cannot start before the norm is known: what the caches do not hold is read twice; counted once here
    return {"bytes": total * (s + (4 if case["out"] == "f32" else s)), "flops": 3 * total}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    wide = lambda t: None if t is None else t.detach().double()
    if case["op"] == "grouped":
        ptr = st["ptr_host"]
        leaves = [wide(st[key]).requires_grad_(case["dir"] == "train") for key in ("x", "w", "b")]
        x, w, b = leaves
        parts = [torch.nn.functional.linear(x[i:j], w[t], b[t]) for t, (i, j) in enumerate(zip(ptr, ptr[1:])) if j > i]
        y = torch.cat(parts)
        if case["dir"] == "fwd":
            return [y]
        return [y.detach(), *torch.autograd.grad(y, leaves, wide(st["dy"]))]
    if case["op"] == "norm":
        keys = [key for key in ("f", "x", "gate", "w1", "b1", "w2", "b2") if st[key] is not None]
        v = {key: wide(st[key]).requires_grad_(case["dir"] == "train") for key in keys}

        def norm(t, i):
            if case["kind"] == "layer":
                return torch.nn.functional.layer_norm(t, (case["d"], ), v["w" + i], v["b" + i], st["eps"])
            return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + st["eps"]) * v["w" + i]

        n = norm(v["f"], "1") if case["post"] else v["f"]
        if "gate" in v:
            n = n * (torch.sigmoid(v["gate"]) if case["gate_act"] == "sigmoid" else v["gate"])
        outs = [v["x"] + st["scale"] * n]
        if case["pre"]:
            outs.append(norm(outs[0], "2"))
        if case["dir"] == "fwd":
            return outs
        ups = [wide(st["dr"])] + ([wide(st["dh"])] if case["pre"] else [])
        grads = torch.autograd.grad(outs, [v[key] for key in keys], ups)
        return [o.detach() for o in outs] + list(grads)
    flat = torch.cat([t.reshape(-1) for t in st["grads"]])
    norm = torch.linalg.vector_norm(flat, ord=st["norm_type"], dtype=torch.float64)
    factor = min(1.0, st["max_norm"] / (float(norm) + 1e-6))
    return [norm, flat.double() * factor]

"""GPU: the fused norms / gate / residual (dh_residual_norm_forward / _backward, autograd.residual_norm) against float64.

Tolerance, element by element: each output is compared within C 2^-24 times the sum of the magnitudes of the terms it is built from, where
every intermediate that is itself a rounded sum enters with its own terms' magnitudes (``_reference`` carries such a magnitude beside every
value).  C counts the roundings on the longest path: a row sum is at most 8 additions in a lane, 6 across lanes and 8 across waves (22);
mean, variance, 1 / sqrt and the affine map of a norm are two such sums and 8 more operations (52); a forward has two norms and the gate,
whose sigmoid is 4 operations and an exponential of 2 ulp: 120.  The backward recomputes them and adds two rounds of row sums: 256.
Column sums add one rounding per row.  A bf16 result adds half a step of its own, 2^-8 of the value."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0**-24
C_FWD, C_BWD = 120, 256


def _inputs(M, D, dtype, gate, kind, seed=0, post=True, pre=True, x=True):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=gen)
    v = dict(f=(0.3 + 1.5 * mk(M, D)).to(dtype), x=mk(M, D).to(dtype) if x else None, gate=None, w1=None, b1=None, w2=None, b2=None,
             dr=mk(M, D).to(dtype), dh=mk(M, D).to(dtype) if pre else None)
    if gate != "none":
        g = 0.7 + 0.5 * mk(*{"scalar": (1, ), "channel": (D, ), "row": (M, 1), "full": (M, D)}[gate])
        v["gate"] = g.to(dtype) if gate in ("row", "full") else g
    if post:
        v["w1"], v["b1"] = 1 + 0.2 * mk(D), (0.1 * mk(D) if kind == "layer" else None)
    if pre:
        v["w2"], v["b2"] = 1 + 0.2 * mk(D), (0.1 * mk(D) if kind == "layer" else None)
    return {k: None if t is None else t.to(DEV) for k, t in v.items()}


class V:
    """A value with the magnitude of the terms it was summed from."""

    def __init__(self, v, m=None):
        self.v, self.m = v, v.abs() if m is None else m

    def __add__(self, o):
        return V(self.v + o.v, self.m + o.m)

    def __sub__(self, o):
        return V(self.v - o.v, self.m + o.m)

    def __mul__(self, o):
        if not isinstance(o, V):
            return V(self.v * o, self.m * abs(o))
        return V(self.v * o.v, self.m * o.v.abs() + self.v.abs() * o.m)

    def mean(self):
        return V(self.v.mean(1, keepdim=True), self.m.mean(1, keepdim=True))

    def sum(self, dims):
        return V(self.v.sum(dims), self.m.sum(dims)) if dims else self


def _normalise(t, kind, eps):
    mean = t.mean() if kind == "layer" else V(torch.zeros_like(t.v[:, :1]))
    c = t - mean
    var = c.v.square().mean(1, keepdim=True) + eps
    rstd = V(var.rsqrt(), 0.5 * var.pow(-1.5) * (2 * (c.v.abs() * c.m).mean(1, keepdim=True) + eps) + var.rsqrt())
    return c * rstd, rstd


def _norm_grad(hat, rstd, w, dout, kind):
    u = dout * w
    t = u - hat * (u * hat).mean()
    if kind == "layer":
        t = t - u.mean()
    return t * rstd


def _reference(v, gate, gate_act, kind, scale, eps, dr=True, dh=True):
    val = {k: None if t is None else V(t.cpu().double()) for k, t in v.items()}
    M, D = v["f"].shape
    one = V(torch.ones(D, dtype=torch.float64))
    zero = V(torch.zeros(M, D, dtype=torch.float64))
    f, x = val["f"], val["x"] or zero
    w1, b1, w2, b2 = (val[k] or (one if k[0] == "w" else V(torch.zeros(D, dtype=torch.float64))) for k in ("w1", "b1", "w2", "b2"))
    post, pre = v["w1"] is not None, v["w2"] is not None
    n = f
    if post:
        fhat, rstd1 = _normalise(f, kind, eps)
        n = fhat * w1 + b1
    g = val["gate"] or V(torch.ones(1, dtype=torch.float64))
    dact = V(torch.ones_like(g.v))
    if gate_act == "sigmoid" and val["gate"] is not None:
        s = torch.sigmoid(g.v)
        g, dact = V(s, 2 * s), V(s * (1 - s), 6 * s * (1 - s) + 2 * s * s)
    r = x + g * n * scale
    out = {"r": r}
    if pre:
        rhat, rstd2 = _normalise(r, kind, eps)
        out["h"] = rhat * w2 + b2
    d = val["dr"] if dr else zero
    if pre and dh:
        d = d + _norm_grad(rhat, rstd2, w2, val["dh"], kind)
        out["w2"], out["b2"] = (val["dh"] * rhat).sum((0, )), val["dh"].sum((0, ))
    elif pre:
        out["w2"] = out["b2"] = V(torch.zeros(D, dtype=torch.float64))
    out["x"] = d
    dn = g * d * scale
    if val["gate"] is not None:
        out["gate"] = (d * n * scale * dact).sum({"scalar": (0, 1), "channel": (0, ), "row": (1, ), "full": ()}[gate])
    out["f"] = dn
    if post:
        out["w1"], out["b1"] = (dn * fhat).sum((0, )), dn.sum((0, ))
        out["f"] = _norm_grad(fhat, rstd1, w1, dn, kind)
    return out


def _check(got, ref, c, what):
    want, mag = ref.v.reshape(got.shape), ref.m.reshape(got.shape)
    tol = c * U * mag
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0**-8 * (want.abs() + tol)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (what, float((err / tol.clamp(min=1e-300)).max()))


def _run(M, D, dtype, gate, gate_act="none", kind="layer", post=True, pre=True, x=True, dr=True, dh=True, scale=0.5, eps=1e-5, seed=0, v=None):
    from dance_amd.autograd import residual_norm
    v = v or _inputs(M, D, dtype, gate, kind, seed, post, pre, x)
    leaves = {k: v[k] for k in ("f", "x", "gate", "w1", "b1", "w2", "b2") if v[k] is not None}
    for t in leaves.values():
        t.requires_grad_(True)
    r, h = residual_norm(v["f"], v["x"], post=(v["w1"], v["b1"]) if post else None, gate=v["gate"], gate_act=gate_act, scale=scale,
                         pre=(v["w2"], v["b2"]) if pre else None, kind=kind, eps=eps)
    ref = _reference({k: None if t is None else t.detach() for k, t in v.items()}, gate, gate_act, kind, scale, eps, dr, dh)
    _check(r.detach(), ref["r"], C_FWD, "r")
    assert (h is None) == (not pre)
    if pre:
        _check(h.detach(), ref["h"], C_FWD, "h")
    outs, ups = ([r], [v["dr"]]) if dr else ([], [])
    if pre and dh:
        outs, ups = outs + [h], ups + [v["dh"]]
    grads = torch.autograd.grad(outs, list(leaves.values()), ups, allow_unused=True)
    for (k, leaf), g in zip(leaves.items(), grads):
        assert g.shape == leaf.shape and g.dtype == leaf.dtype
        _check(g, ref[k], C_BWD + (M if k in ("w1", "b1", "w2", "b2") or gate in ("scalar", "channel") and k == "gate" else 0), k)
    return r.detach(), h, grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,D", [(1, 16), (37, 50), (5, 200), (9, 512), (3, 513), (130, 31), (3, 2000), (2, 4096), (3, 4095), (2, 1030), (3, 2700)])
@pytest.mark.parametrize("gate", ["none", "scalar", "channel", "row", "full"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_shapes(cuda_device, dtype, M, D, gate, kind):
    _run(M, D, dtype, gate, "sigmoid" if (M + D) % 2 else "none", kind)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("post,pre,x,dr,dh", [c for c in itertools.product([True, False], repeat=5) if (c[3] or (c[1] and c[4])) and (c[1] or c[4])])
def test_parts(cuda_device, dtype, post, pre, x, dr, dh):
    """Every combination of norms, residual and upstream gradients."""
    for gate, kind in (("full", "layer"), ("row", "rms"), ("none", "layer")):
        _run(21, 72, dtype, gate, "sigmoid", kind, post, pre, x, dr, dh)


@pytest.mark.parametrize("D", [1, 2, 3, 5, 7, 8, 9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_narrow_rows(cuda_device, D, dtype, kind):
    """Rows shorter than one 16-byte access, and one element longer.  (Two equal-ish values make a layer norm ill-conditioned: the
    magnitudes that the reference carries contain the 1 / sigma of it.)"""
    _run(300, D, dtype, "channel" if D > 1 else "scalar", "none", kind)
    _run(300, D, dtype, "full", "sigmoid", kind)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(cuda_device, dtype):
    """More rows than one pass of the grid: every workgroup walks several."""
    _run(20011, 48, dtype, "channel", "sigmoid", "layer")
    r, h, grads = _run(9000, 520, dtype, "scalar", "sigmoid", "rms")
    r2, h2, grads2 = _run(9000, 520, dtype, "scalar", "sigmoid", "rms")
    assert torch.equal(r, r2) and torch.equal(h, h2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))  # fixed order


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows(cuda_device, dtype):
    """Rows inside wider buffers that start at odd elements; expanded residuals and upstream gradients."""
    from dance_amd import kernels
    from dance_amd.autograd import residual_norm
    M, D = 33, 75
    v = _inputs(M, D, dtype, "full", "layer")
    wide = {k: torch.full((M, D + 9), float("nan"), dtype=dtype, device=DEV) for k in ("f", "x", "gate", "dr", "dh")}
    for i, k in enumerate(wide):
        wide[k][:, i + 1:i + 1 + D] = v[k]
        v[k] = wide[k][:, i + 1:i + 1 + D]
    r, h, stats = kernels.residual_norm_forward(v["f"], v["x"], post=(v["w1"], v["b1"]), gate=v["gate"], gate_sigmoid=True, scale=0.5,
                                                pre=(v["w2"], v["b2"]), want_stats=True)
    ref = _reference(v, "full", "sigmoid", "layer", 0.5, 1e-5)
    _check(r, ref["r"], C_FWD, "r")
    _check(h, ref["h"], C_FWD, "h")
    g = kernels.residual_norm_backward(v["dr"], v["dh"], v["f"], v["x"], stats, post=(v["w1"], v["b1"]), gate=v["gate"], gate_sigmoid=True, scale=0.5,
                                       pre=(v["w2"], v["b2"]))
    for k in ("f", "x", "gate", "w1", "b1", "w2", "b2"):
        _check(g[k], ref[k], C_BWD + M, k)
    # one residual row for all rows, a sum as the loss
    row = v["x"][:1].clone().requires_grad_(True)
    r, _ = residual_norm(v["f"], row.expand(M, D), post=(v["w1"], v["b1"]))
    r.sum().backward()
    assert torch.equal(row.grad, torch.full_like(row, M))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_do_not_touch_each_other(cuda_device, dtype):
    """A NaN or an infinity reaches its own row only; an all-zero and a constant row are finite."""
    from dance_amd import kernels
    M, D = 70, 50
    v = _inputs(M, D, dtype, "none", "layer")
    opts = dict(post=(v["w1"], v["b1"]), pre=(v["w2"], v["b2"]), want_stats=True)
    clean = kernels.residual_norm_forward(v["f"], v["x"], **opts)
    f = v["f"].clone()
    f[3, 49], f[40, 0], f[41] = float("nan"), float("inf"), 0.0
    f[42] = 2.5
    r, h, stats = kernels.residual_norm_forward(f, v["x"], **opts)
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[[3, 40, 41, 42]] = False
    assert torch.equal(r[keep], clean[0][keep]) and torch.equal(h[keep], clean[1][keep])
    assert bool(r[3].isnan().all()) and bool(h[3].isnan().all()) and bool(h[40].isnan().all())
    assert bool(r[41:43].isfinite().all()) and bool(h[41:43].isfinite().all())
    back = dict(post=opts["post"], pre=opts["pre"], want=("f", "x"))
    g0 = kernels.residual_norm_backward(v["dr"], v["dh"], v["f"], v["x"], clean[2], **back)
    g = kernels.residual_norm_backward(v["dr"], v["dh"], f, v["x"], stats, **back)
    assert all(torch.equal(g[k][keep], g0[k][keep]) and bool(g[k][41:43].isfinite().all()) for k in ("f", "x"))
    zero = torch.zeros(4, D, dtype=dtype, device=DEV)
    r, h, _ = kernels.residual_norm_forward(zero, zero, post=(None, None), pre=(None, None), kind=kernels.NORM_RMS)
    assert not bool(r.any()) and not bool(h.any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [3, 20, 23, 64, 300, 513, 2050])
def test_infinity_and_row_gate(cuda_device, D, dtype):
    """An infinite element makes its row's gate gradient infinite, not NaN, wherever in the row it lies: nothing behind a row's end enters."""
    from dance_amd import kernels
    for at in {0, D // 2, D - 1}:
        f, x = torch.ones(5, D, dtype=dtype, device=DEV), torch.ones(5, D, dtype=dtype, device=DEV)
        dr = torch.ones(5, D, dtype=dtype, device=DEV)
        f[2, at], f[3, at] = float("inf"), float("-inf")
        gate = torch.full((5, 1), 0.5, dtype=dtype, device=DEV)
        r, _, stats = kernels.residual_norm_forward(f, x, gate=gate, want_stats=True)
        g = kernels.residual_norm_backward(dr, None, f, x, stats, gate=gate, want=("f", "gate"))
        want = f.double().sum(1, keepdim=True)  # D itself in the finite rows: exact in fp32, one rounding in bf16
        assert torch.equal(g["gate"], want.to(dtype)) and torch.equal(g["f"], dr * 0.5)
        assert torch.equal(r, x + f * 0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_row_gate_of_any_stride(cuda_device, dtype):
    """A [M, 1] gate is contiguous whatever its last stride: the transpose of a row."""
    from dance_amd.autograd import residual_norm
    v = _inputs(33, 40, dtype, "none", "layer")
    row = torch.randn(1, 33, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
    gates = [row.reshape(33, 1).clone().requires_grad_(), row.t().detach().requires_grad_()]
    assert gates[0].stride() != gates[1].stride()
    results = []
    for gate in gates:
        r, h = residual_norm(v["f"], v["x"], gate=gate, pre=(v["w2"], v["b2"]))
        torch.autograd.backward((r, h), (v["dr"], v["dh"]))
        results.append((r, h, gate.grad))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("D", [40, 512, 2000])
def test_offset_rows(cuda_device, D):
    """Rows of a large common offset and small differences: the differences are what the norm sees.  mean carries 22 roundings of the row's
    magnitude, the subtraction is exact to a rounding: |error| <= 32 2^-24 |offset| rstd + 120 2^-24 |value|."""
    from dance_amd import kernels
    gen = torch.Generator().manual_seed(0)
    f = (1000.0 + torch.randn(30, D, generator=gen)).to(DEV)
    f[7] = 1234.5678                                              # constant: nothing but the bias may come out
    r, _, _ = kernels.residual_norm_forward(f, post=(None, None))
    ref = torch.nn.functional.layer_norm(f.double(), (D, ))
    rstd = (f.double().var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    assert bool(((r.double() - ref).abs() <= 32 * U * f.double().abs() * rstd + 120 * U * ref.abs()).all())


def test_gradient_against_differences(cuda_device):
    """<grad, d> against the central difference of L = <r, dr> + <h, dh> along d, L evaluated by the float64 reference (which the forward is
    held to above): the truncation error is O(step^2) = 1e-8 of a third derivative of order one."""
    M, D = 12, 40
    v = _inputs(M, D, torch.float32, "channel", "layer")

    def loss(**change):
        u = dict(v, **change)
        ref = _reference(u, "channel", "sigmoid", "layer", 0.5, 1e-5)
        return float((ref["r"].v * v["dr"].cpu().double()).sum() + (ref["h"].v * v["dh"].cpu().double()).sum())

    from dance_amd.autograd import residual_norm
    keys = ("f", "x", "gate", "w1", "b1", "w2", "b2")
    leaves = [v[k].clone().requires_grad_(True) for k in keys]
    a = dict(zip(keys, leaves))
    r, h = residual_norm(a["f"], a["x"], post=(a["w1"], a["b1"]), gate=a["gate"], gate_act="sigmoid", scale=0.5, pre=(a["w2"], a["b2"]))
    grads = torch.autograd.grad([r, h], leaves, [v["dr"], v["dh"]])
    gen = torch.Generator().manual_seed(4)
    for k, g in zip(keys, grads):
        d = torch.randn(v[k].shape, generator=gen, dtype=torch.float64)
        step = 1e-4
        base = v[k].cpu().double()
        quotient = (loss(**{k: base + step * d}) - loss(**{k: base - step * d})) / (2 * step)
        slope = float((g.cpu().double() * d).sum())
        size = float((g.cpu().double() * d).abs().sum())
        assert abs(quotient - slope) <= 1e-5 * max(size, 1.0), k


def test_refusals(cuda_device):
    from dance_amd import _lib, kernels
    from dance_amd.autograd import residual_norm
    v = _inputs(6, 40, torch.float32, "none", "layer")
    f, x, w = v["f"], v["x"], v["w1"]
    for call in (lambda: residual_norm(f, x, kind="batch"), lambda: residual_norm(f, x, gate_act="tanh"), lambda: residual_norm(f, x[:3]),
                 lambda: residual_norm(f, x.bfloat16()), lambda: residual_norm(f, x, post=(w[:5], None)), lambda: residual_norm(f, x, eps=-1.0),
                 lambda: residual_norm(f, x, gate=torch.zeros(6, device=DEV)), lambda: residual_norm(torch.zeros(2, 4097, device=DEV)),
                 lambda: residual_norm(torch.zeros(2, 0, device=DEV)), lambda: kernels.residual_norm_forward(f.t()),
                 lambda: kernels.residual_norm_forward(f, x[:1].expand(6, 40)), lambda: kernels.residual_norm_backward(None, None, f, x, f[:, :4])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: residual_norm(f.half(), None), lambda: residual_norm(f, x, post=(w.bfloat16(), None)),
                 lambda: residual_norm(f, x, gate=torch.zeros(40, device=DEV, dtype=torch.bfloat16)),
                 lambda: residual_norm(f, x, gate=torch.zeros(6, 1, device=DEV, dtype=torch.bfloat16))):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(_lib.DanceHipError):
        residual_norm(f, x.cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows(cuda_device, dtype):
    from dance_amd.autograd import residual_norm
    f = torch.zeros(0, 40, dtype=dtype, device=DEV, requires_grad=True)
    w, b, g = (torch.ones(40, device=DEV, requires_grad=True) for _ in range(3))
    r, h = residual_norm(f, None, post=(w, b), gate=g, pre=(w, None))
    assert r.shape == h.shape == (0, 40)
    (r.sum() + h.sum()).backward()
    assert not bool(w.grad.any()) and not bool(b.grad.any()) and not bool(g.grad.any())

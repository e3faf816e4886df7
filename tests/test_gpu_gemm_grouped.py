"""GPU: products grouped by row type (dh_gemm_grouped, dh_gemm_grouped_wgrad, autograd.grouped_linear) against float64.

Tolerance, element by element: an output is a sum of at most n products (n = K, or the rows of the group), each product and each addition
rounded once in fp32.  Counting a whole step of 2^-23 for each (the matrix cores do not document how they round inside an instruction),
|error| <= (n + 3) 2^-23 sum |terms|; a bf16 output adds half a step of its own, 2^-8 of the value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U32, HALF_BF16 = 2.0**-23, 2.0**-8

# name: (rows, group sizes, rows before the first group)
LAYOUTS = {
    "one_row": (1, [1], 0),
    "one_group": (77, [77], 0),
    "empty_groups": (70, [0, 33, 0, 0, 37, 0], 0),
    "gaps": (90, [5, 0, 40], 13),                     # 13 rows in front and 32 behind belong to no group
    "all_empty": (9, [0, 0, 0], 4),
    "mostly_empty": (7, [0] * 300 + [3] + [0] * 700 + [4] + [0] * 100, 0),
    "ragged": (611, [1, 128, 129, 127, 3, 0, 200, 23], 0),
    "many": (700, [i % 5 for i in range(350)], 0),    # more groups than one 64-wide probe
    "long": (3700, [2500, 1100], 60),                 # the large tile
    "chunks": (1900, [700, 0, 256, 257, 1, 686], 0),  # groups of several weight-gradient chunks beside groups of one
}


def _ptr(sizes, lead):
    return torch.tensor(np.concatenate(([lead], lead + np.cumsum(sizes))), dtype=torch.int32, device=DEV)


def _operands(name, K, N, dtype, seed=0, trans_b=True):
    rows, sizes, lead = LAYOUTS[name]
    gen = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=gen).to(dtype)
    x, dy = mk(rows, K), mk(rows, N)
    w = mk(len(sizes), N, K) if trans_b else mk(len(sizes), K, N)
    return x.to(DEV), w.to(DEV), torch.randn(len(sizes), N, generator=gen).to(DEV), dy.to(DEV), _ptr(sizes, lead)


def _reference(x, w, b, ptr, trans_b=True):
    """y and the sum of its terms' magnitudes, float64 on the CPU; rows of no group are zero."""
    x, w, ptr = x.cpu().double(), w.cpu().double(), ptr.tolist()
    N = w.shape[1] if trans_b else w.shape[2]
    y, mag = torch.zeros(x.shape[0], N, dtype=torch.float64), torch.zeros(x.shape[0], N, dtype=torch.float64)
    for g in range(w.shape[0]):
        i, j = ptr[g], ptr[g + 1]
        wt = w[g].t() if trans_b else w[g]
        y[i:j], mag[i:j] = x[i:j] @ wt, x[i:j].abs() @ wt.abs()
        if b is not None:
            y[i:j] += b[g].cpu().double()
            mag[i:j] += b[g].cpu().double().abs()
    return y, mag


def _check(got, ref, mag, n, out_bf16=False):
    err = (got.cpu().double() - ref).abs()
    tol = (n + 3) * U32 * mag + (HALF_BF16 * (ref.abs() + (n + 3) * U32 * mag) if out_bf16 else 0.0)
    assert got.shape == ref.shape and bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,N", [(40, 24), (33, 17), (1, 1), (200, 136), (64, 256), (136, 264), (320, 40)])
@pytest.mark.parametrize("trans_b", [True, False])
def test_forward(cuda_device, layout, dtype, K, N, trans_b):
    from dance_amd import kernels
    x, w, b, _, ptr = _operands(layout, K, N, dtype, trans_b=trans_b)
    ref, mag = _reference(x, w, b, ptr, trans_b)
    y = kernels.gemm_grouped(x, w, ptr, trans_b=trans_b, bias=b)
    assert y.dtype == dtype
    _check(y, ref, mag, K, dtype == torch.bfloat16)
    y32 = kernels.gemm_grouped(x, w, ptr, trans_b=trans_b, out_dtype=torch.float32)
    _check(y32, *_reference(x, w, None, ptr, trans_b), K)
    if dtype == torch.bfloat16:  # one nearest-even rounding of the same fp32 value
        assert torch.equal(kernels.gemm_grouped(x, w, ptr, trans_b=trans_b), y32.to(dtype))


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,N", [(40, 24), (33, 17), (1, 1), (136, 200), (264, 520)])
def test_weight_gradient(cuda_device, layout, dtype, K, N):
    from dance_amd import kernels
    x, w, b, dy, ptr = _operands(layout, K, N, dtype)
    dw, db = kernels.gemm_grouped_wgrad(dy, x, ptr, want_bias=True)
    dw32 = kernels.gemm_grouped_wgrad(dy, x, ptr, out_dtype=torch.float32)
    assert dw.dtype == dtype and db.dtype == torch.float32
    p, xd, yd = ptr.tolist(), x.cpu().double(), dy.cpu().double()
    for g in range(w.shape[0]):
        i, j = p[g], p[g + 1]
        ref, mag = yd[i:j].t() @ xd[i:j], yd[i:j].abs().t() @ xd[i:j].abs()
        _check(dw[g], ref, mag, j - i, dtype == torch.bfloat16)
        _check(dw32[g], ref, mag, j - i)
        _check(db[g], yd[i:j].sum(0), yd[i:j].abs().sum(0), j - i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,K,N", [(5000, 512, 260), (130, 2000, 512), (3, 400, 200), (5000, 511, 331), (52000, 37, 12), (60000, 3, 5), (52000, 24, 16)])
def test_larger(cuda_device, dtype, rows, K, N):
    from dance_amd import kernels
    gen = torch.Generator().manual_seed(rows)
    sizes = torch.multinomial(torch.rand(11, generator=gen), rows, replacement=True, generator=gen).bincount(minlength=11).tolist()
    LAYOUTS["tmp"] = (rows, sizes, 0)
    try:
        x, w, b, dy, ptr = _operands("tmp", K, N, dtype, seed=1)
    finally:
        del LAYOUTS["tmp"]
    bf = dtype == torch.bfloat16
    _check(kernels.gemm_grouped(x, w, ptr, bias=b), *_reference(x, w, b, ptr), K, bf)
    _check(kernels.gemm_grouped(dy, w, ptr, trans_b=False), *_reference(dy, w, None, ptr, False), N, bf)
    dw, db = kernels.gemm_grouped_wgrad(dy, x, ptr, want_bias=True)
    p, xd, yd = ptr.tolist(), x.cpu().double(), dy.cpu().double()
    for g in range(11):
        i, j = p[g], p[g + 1]
        _check(dw[g], yd[i:j].t() @ xd[i:j], yd[i:j].abs().t() @ xd[i:j].abs(), j - i, bf)
        _check(db[g], yd[i:j].sum(0), yd[i:j].abs().sum(0), j - i)
    # the same call gives the same bits
    dw2, db2 = kernels.gemm_grouped_wgrad(dy, x, ptr, want_bias=True)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(cuda_device, dtype):
    """Rows inside wider buffers, starting at odd elements; weights that are a view of a larger stack; an output that is a column window:
    what lies beside it stays as it was, and so do rows of no group."""
    from dance_amd import kernels
    rows, sizes, lead = LAYOUTS["gaps"]
    ptr, K, N = _ptr(sizes, lead), 37, 29
    gen = torch.Generator().manual_seed(5)
    xb = torch.randn(rows, K + 8, generator=gen).to(dtype).to(DEV)
    wb = torch.randn(len(sizes), N + 3, K + 5, generator=gen).to(dtype).to(DEV)
    dyb = torch.randn(rows, N + 4, generator=gen).to(dtype).to(DEV)
    x, w, dy = xb[:, 3:3 + K], wb[:, 1:1 + N, 2:2 + K], dyb[:, 1:1 + N]
    big = torch.full((rows, N + 6), 7.0, dtype=dtype, device=DEV)
    out = big[:, 5:5 + N]
    assert kernels.gemm_grouped(x, w, ptr, out=out) is out
    ref, mag = _reference(x, w, None, ptr)
    inside = slice(lead, lead + sum(sizes))
    _check(out[inside], ref[inside], mag[inside], K, dtype == torch.bfloat16)
    assert bool((out[:lead] == 7).all()) and bool((out[inside.stop:] == 7).all()) and bool((big[:, :5] == 7).all()) and bool((big[:, 5 + N:] == 7).all())
    _check(kernels.gemm_grouped(dy, w, ptr, trans_b=False), *_reference(dy, w, None, ptr, False), N, dtype == torch.bfloat16)
    dw = kernels.gemm_grouped_wgrad(dy, x, ptr, out_dtype=torch.float32)
    p = ptr.tolist()
    for g in range(len(sizes)):
        i, j = p[g], p[g + 1]
        yd, xd = dy[i:j].cpu().double(), x[i:j].cpu().double()
        _check(dw[g], yd.t() @ xd, yd.abs().t() @ xd.abs(), j - i)


def test_values_outside_the_group_do_not_enter(cuda_device):
    """Infinities and NaN in rows of other groups, in rows of no group and behind a window's columns change nothing: the same bits as with
    ones there.  (The clean side lies in a buffer of the same strides: the alignment of the rows chooses the kernel, and with it the order
    in which the bias gradient's rows are added.)"""
    from dance_amd import kernels
    for dtype in (torch.float32, torch.bfloat16):
        for K, N in ((40, 24), (33, 17)):
            x, w, b, dy, ptr = _operands("gaps", K, N, dtype)
            xw, dyw = torch.full((x.shape[0], K + 3), float("nan"), dtype=dtype, device=DEV), torch.full((x.shape[0], N + 3), float("inf"), dtype=dtype, device=DEV)
            xw[:, :K], dyw[:, :N] = x, dy
            bad = torch.arange(x.shape[0], device=DEV)
            bad = (bad < 13) | (bad >= 58)
            xw[bad], dyw[bad] = float("nan"), float("nan")
            xc, dyc = torch.ones_like(xw), torch.ones_like(dyw)
            xc[:, :K], dyc[:, :N] = x, dy
            xp, dyp, x, dy = xw[:, :K], dyw[:, :N], xc[:, :K], dyc[:, :N]
            assert torch.equal(kernels.gemm_grouped(xp, w, ptr, bias=b), kernels.gemm_grouped(x, w, ptr, bias=b))
            assert torch.equal(kernels.gemm_grouped(dyp, w, ptr, trans_b=False), kernels.gemm_grouped(dy, w, ptr, trans_b=False))
            for a, c in zip(kernels.gemm_grouped_wgrad(dyp, xp, ptr, want_bias=True), kernels.gemm_grouped_wgrad(dy, x, ptr, want_bias=True)):
                assert torch.equal(a, c)
    # and inside a group they reach exactly the rows that hold them
    x, w, b, dy, ptr = _operands("empty_groups", 40, 24, torch.float32)
    clean = kernels.gemm_grouped(x, w, ptr, bias=b, act=kernels.ACT_RELU)
    x2 = x.clone()
    x2[5, 3], x2[40, 0] = float("nan"), float("inf")
    y = kernels.gemm_grouped(x2, w, ptr, bias=b, act=kernels.ACT_RELU)
    keep = torch.ones(70, dtype=torch.bool, device=DEV)
    keep[5] = keep[40] = False
    assert torch.equal(y[keep], clean[keep]) and bool(y[5].isnan().all()) and not bool(y[40].isfinite().all())


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_grouped_linear_gradients(cuda_device, relu, dtype, wdtype):
    from dance_amd.autograd import grouped_linear
    x, w, b, dy, ptr = _operands("gaps", 40, 24, dtype)
    w = w.to(wdtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = grouped_linear(leaves[0], leaves[1], ptr, leaves[2], relu=relu)
    gx, gw, gb = torch.autograd.grad(y, leaves, dy)
    assert gx.dtype == dtype and gw.dtype == wdtype and gb.dtype == torch.float32
    p = ptr.tolist()
    ref, mag = _reference(x, w, b, ptr)
    bf = dtype == torch.bfloat16
    _check(y, ref.clamp(min=0) if relu else ref, mag, 40, bf)
    dyd = dy.cpu().double() * ((y.cpu() > 0) if relu else 1)
    rx, mx = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    for g in range(w.shape[0]):
        i, j = p[g], p[g + 1]
        wd, xd = w[g].cpu().double(), x[i:j].cpu().double()
        rx[i:j], mx[i:j] = dyd[i:j] @ wd, dyd[i:j].abs() @ wd.abs()
        _check(gw[g], dyd[i:j].t() @ xd, dyd[i:j].abs().t() @ xd.abs(), j - i, wdtype == torch.bfloat16)
        _check(gb[g], dyd[i:j].sum(0), dyd[i:j].abs().sum(0), j - i)
    _check(gx, rx, mx, 24, bf)


def test_gradient_against_differences(cuda_device):
    """<dL/dv, d> against the central difference of L along d, L = <y, c> computed from the fp32 kernel: y is bilinear, so the difference
    quotient has no truncation error; each y carries (K + 3) 2^-23 of its terms, divided by the step."""
    from dance_amd.autograd import grouped_linear
    x, w, b, dy, ptr = _operands("ragged", 40, 24, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(grouped_linear(leaves[0], leaves[1], ptr, leaves[2]), leaves, dy)
    gen = torch.Generator().manual_seed(9)
    for i, (v, g) in enumerate(zip((x, w, b), grads)):
        d = torch.randn(v.shape, generator=gen).to(DEV)
        h, vals, mags = 0.5, [], []
        for s in (h, -h):
            args = [x, w, b]
            args[i] = v + s * d
            vals.append((grouped_linear(args[0], args[1], ptr, args[2]).double() * dy.double()).sum())
            mags.append((_reference(args[0], args[1], args[2], ptr)[1].to(DEV) * dy.double().abs()).sum())
        quotient = float((vals[0] - vals[1]) / (2 * h))
        slope = float((g.double() * d.double()).sum())
        # the perturbed argument itself is rounded to fp32 (2^-24 of it), which moves y by that share of its terms
        tol = (40 + 5) * U32 * float(mags[0] + mags[1]) / (2 * h) + (611 + 3) * U32 * float((g.abs().double() * d.abs().double()).sum())
        assert abs(quotient - slope) <= tol


def test_expanded_and_partial_gradients(cuda_device):
    from dance_amd.autograd import grouped_linear
    x, w, b, _, ptr = _operands("ragged", 40, 24, torch.float32)
    row = torch.randn(1, 40, device=DEV, requires_grad=True)
    y = grouped_linear(row.expand(x.shape[0], 40), w, ptr, b)
    y.sum().backward()                                            # an expanded upstream gradient, a broadcast input
    p = ptr.tolist()
    ref = sum((p[g + 1] - p[g]) * w[g].double().sum(0) for g in range(w.shape[0]))
    mag = sum((p[g + 1] - p[g]) * w[g].double().abs().sum(0) for g in range(w.shape[0]))
    assert bool(((row.grad[0].double() - ref).abs() <= (24 + 611 + 3) * U32 * mag).all())
    only_w = w.clone().requires_grad_(True)
    grouped_linear(x, only_w, ptr).sum().backward()
    assert only_w.grad is not None
    only_b = b.clone().requires_grad_(True)
    grouped_linear(x, w, ptr, only_b).sum().backward()
    sizes = (ptr[1:] - ptr[:-1]).double()
    assert torch.equal(only_b.grad.double(), sizes[:, None].expand(-1, 24))


def test_refusals(cuda_device):
    from dance_amd import _lib, kernels
    x, w, b, dy, ptr = _operands("gaps", 40, 24, torch.float32)
    ok = lambda **kw: kernels.gemm_grouped(*[kw.pop(n, d) for n, d in (("x", x), ("w", w), ("ptr", ptr))], **kw)
    ok()
    with pytest.raises(TypeError):
        ok(ptr=ptr.long())
    with pytest.raises(TypeError):
        ok(x=x.half())
    with pytest.raises(TypeError):
        ok(w=w.bfloat16())
    with pytest.raises(TypeError):
        ok(bias=b.bfloat16())
    with pytest.raises(TypeError):
        ok(out_dtype=torch.float16)
    with pytest.raises(_lib.DanceHipError):
        ok(ptr=ptr.cpu())
    for kw in (dict(ptr=ptr[:-1]), dict(x=x[:, :39]), dict(bias=b[:, :5]), dict(w=w[0]), dict(x=x[0]), dict(act=5), dict(x=x.t()), dict(out=x), dict(out=torch.zeros(90, 64, device=DEV)[:, :24], x=torch.zeros(90, 40, device=DEV).t()),
               dict(x=x[:1].expand(90, 40)), dict(ptr=ptr[None])):
        with pytest.raises(ValueError):
            ok(**kw)
    with pytest.raises(ValueError):
        kernels.gemm_grouped_wgrad(dy[:5], x, ptr)
    shared = torch.zeros(90, 64, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        kernels.gemm_grouped(shared[:, :40], w, ptr, out=shared[:, 40:])
    with pytest.raises(ValueError):
        kernels.gemm_grouped_wgrad(dy.t(), x, ptr)


def test_nothing_to_multiply(cuda_device):
    from dance_amd import kernels
    for dtype in (torch.float32, torch.bfloat16):
        p0 = torch.zeros(4, dtype=torch.int32, device=DEV)
        z = lambda *s: torch.zeros(*s, dtype=dtype, device=DEV)
        assert kernels.gemm_grouped(z(0, 8), z(3, 5, 8), p0).shape == (0, 5)
        dw, db = kernels.gemm_grouped_wgrad(z(0, 5), z(0, 8), p0, want_bias=True)
        assert dw.shape == (3, 5, 8) and not bool(dw.any()) and not bool(db.any())
        y = kernels.gemm_grouped(z(6, 8) + 1, z(0, 5, 8), p0[:1])  # no groups: every row is outside
        assert y.shape == (6, 5) and not bool(y.any())
        b = torch.randn(1, 5, device=DEV)
        y = kernels.gemm_grouped(z(6, 0), z(1, 5, 0), torch.tensor([0, 6], dtype=torch.int32, device=DEV), bias=b, out_dtype=torch.float32)
        assert torch.equal(y, b.expand(6, 5))  # no columns: the bias


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,K,N", [(6000, 333, 331), (52000, 35, 13), (60000, 5, 3), (70, 37, 21)])
def test_nothing_behind_a_row_enters(cuda_device, dtype, rows, K, N):
    """NaN behind every row of every operand (up to three columns), in the rows of no group and in front of the first."""
    from dance_amd import kernels
    gen = torch.Generator().manual_seed(K)
    nan = float("nan")

    def padded(*shape):
        buf = torch.full((*shape[:-1], shape[-1] + 3), nan)
        buf[..., :shape[-1]] = torch.randn(*shape, generator=gen)
        return buf.to(dtype).to(DEV)[..., :shape[-1]]

    sizes, lead = [rows // 3, 0, 1, rows // 2], 9
    ptr = _ptr(sizes, lead)
    x, dy, w = padded(rows, K), padded(rows, N), padded(4, N, K)
    outside = torch.ones(rows, dtype=torch.bool)
    outside[lead:lead + sum(sizes)] = False
    x[outside.to(DEV)], dy[outside.to(DEV)] = nan, nan
    bf = dtype == torch.bfloat16
    clean = [t.cpu().nan_to_num(0.0) for t in (x, dy)]
    _check(kernels.gemm_grouped(x, w, ptr), *_reference(clean[0], w, None, ptr), K, bf)
    _check(kernels.gemm_grouped(dy, w, ptr, trans_b=False), *_reference(clean[1], w, None, ptr, False), N, bf)
    dw, db = kernels.gemm_grouped_wgrad(dy, x, ptr, want_bias=True)
    p, xd, yd = ptr.tolist(), clean[0].double(), clean[1].double()
    for g in range(4):
        i, j = p[g], p[g + 1]
        _check(dw[g], yd[i:j].t() @ xd[i:j], yd[i:j].abs().t() @ xd[i:j].abs(), j - i, bf)
        _check(db[g], yd[i:j].sum(0), yd[i:j].abs().sum(0), j - i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_single_columns_of_any_stride(cuda_device, dtype):
    """A matrix of one column is contiguous whatever that dimension's stride: transposes of a row."""
    from dance_amd.autograd import grouped_linear
    ptr = torch.tensor([0, 7, 20, 33], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(3)
    draw = lambda *shape: torch.randn(*shape, generator=g).to(DEV, dtype)
    for K, N in ((1, 5), (24, 1), (1, 1)):
        odd = lambda t: t.as_strided(t.shape, (*t.stride()[:-1], 7)) if t.shape[-1] == 1 else t
        x, w, b, dy = draw(33, K), draw(3, N, K), draw(3, N).float(), draw(33, N)
        results = []
        for change in (lambda t: t, odd):
            leaves = [change(t).detach().requires_grad_() for t in (x, w, b)]
            y = grouped_linear(leaves[0], leaves[1], ptr, leaves[2])
            y.backward(change(dy))
            results.append([y] + [t.grad for t in leaves])
        assert odd(x).stride() != x.stride() or odd(b).stride() != b.stride()
        assert all(torch.equal(a, c) for a, c in zip(*results))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bias_gradient_without_input_columns(cuda_device, dtype):
    from dance_amd.autograd import grouped_linear
    ptr = torch.tensor([1, 3, 3, 6], dtype=torch.int32, device=DEV)
    x = torch.zeros(7, 0, dtype=dtype, device=DEV, requires_grad=True)
    w = torch.zeros(3, 4, 0, dtype=dtype, device=DEV, requires_grad=True)
    b = torch.ones(3, 4, device=DEV, requires_grad=True)
    y = grouped_linear(x, w, ptr, b)
    dy = torch.arange(28, device=DEV).reshape(7, 4).to(dtype)
    y.backward(dy)
    d = dy.float()
    assert torch.equal(b.grad, torch.stack([d[1:3].sum(0), torch.zeros(4, device=DEV), d[3:6].sum(0)]))  # (small integers: exact)
    assert w.grad.shape == (3, 4, 0) and x.grad.shape == (7, 0)

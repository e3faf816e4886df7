"""GPU: the residual norm on rows of 4097 to 8192 columns (dh_residual_norm_wide_forward / _backward) against float64.

Tolerance as for the narrower rows (test_gpu_residual_norm.py), with the longer row sums counted: 16 additions in a lane, 6 across lanes, 8
across waves (30).  A norm is two such sums and 8 more operations (68); a forward two norms, the gate and the residual (152).  The backward
recomputes it and adds, for each norm, two row sums and 10 operations: 152 + 2 (60 + 10) = 292 (300).  Column sums add one rounding per row."""
import itertools

import pytest
import torch

import test_gpu_residual_norm as narrow

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def longer_sums(monkeypatch):
    monkeypatch.setattr(narrow, "C_FWD", 152)
    monkeypatch.setattr(narrow, "C_BWD", 300)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,D", [(1, 4097), (3, 8192), (5, 6000), (2, 8191), (3, 5004), (2, 7170)])
@pytest.mark.parametrize("gate", ["none", "scalar", "channel", "row", "full"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_shapes(cuda_device, dtype, M, D, gate, kind):
    narrow._run(M, D, dtype, gate, "sigmoid" if (M + D) % 2 else "none", kind)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("post,pre,x,dr,dh", [c for c in itertools.product([True, False], repeat=5) if (c[0] or c[1]) and (c[3] or (c[1] and c[4])) and (c[1] or c[4])])
def test_parts(cuda_device, dtype, post, pre, x, dr, dh):
    for gate, kind in (("full", "layer"), ("row", "rms"), ("channel", "layer")):
        narrow._run(4, 4105, dtype, gate, "sigmoid", kind, post, pre, x, dr, dh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(cuda_device, dtype):
    """Several rows in every chunk of the column gradients, a last chunk that is not full; the same bits every time."""
    for gate, act in (("channel", "sigmoid"), ("scalar", "none")):
        first = narrow._run(1030, 4100, dtype, gate, act, "layer")
        again = narrow._run(1030, 4100, dtype, gate, act, "layer")
        for a, b in zip(itertools.chain(first[:2], first[2]), itertools.chain(again[:2], again[2])):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows_and_single_gradients(cuda_device, dtype):
    """Rows inside wider buffers of NaN that start at odd elements; each gradient asked for alone is the one that comes with all the others."""
    from dance_amd import kernels
    M, D = 7, 4109
    v = narrow._inputs(M, D, dtype, "full", "layer")
    for i, k in enumerate(("f", "x", "gate", "dr", "dh")):
        wide = torch.full((M, D + 9), float("nan"), dtype=dtype, device=DEV)
        wide[:, i + 1:i + 1 + D] = v[k]
        v[k] = wide[:, i + 1:i + 1 + D]
    opts = dict(post=(v["w1"], v["b1"]), gate=v["gate"], gate_sigmoid=True, scale=0.5, pre=(v["w2"], v["b2"]))
    r, h, stats = kernels.residual_norm_forward(v["f"], v["x"], want_stats=True, **opts)
    ref = narrow._reference(v, "full", "sigmoid", "layer", 0.5, 1e-5)
    narrow._check(r, ref["r"], narrow.C_FWD, "r")
    narrow._check(h, ref["h"], narrow.C_FWD, "h")
    g = kernels.residual_norm_backward(v["dr"], v["dh"], v["f"], v["x"], stats, **opts)
    for k in ("f", "x", "gate", "w1", "b1", "w2", "b2"):
        narrow._check(g[k], ref[k], narrow.C_BWD + M, k)
        alone = kernels.residual_norm_backward(v["dr"], v["dh"], v["f"], v["x"], stats, want=(k, ), **opts)
        assert list(alone) == [k] and torch.equal(alone[k], g[k])


def test_rows_do_not_touch_each_other(cuda_device):
    from dance_amd import kernels
    M, D = 6, 5003
    for dtype in (torch.float32, torch.bfloat16):
        v = narrow._inputs(M, D, dtype, "none", "layer")
        opts = dict(post=(v["w1"], v["b1"]), pre=(v["w2"], v["b2"]))
        clean = kernels.residual_norm_forward(v["f"], v["x"], want_stats=True, **opts)
        f = v["f"].clone()
        f[1, D - 1], f[4, 0] = float("nan"), float("inf")
        r, h, stats = kernels.residual_norm_forward(f, v["x"], want_stats=True, **opts)
        g0 = kernels.residual_norm_backward(v["dr"], v["dh"], v["f"], v["x"], clean[2], want=("f", "x"), **opts)
        g = kernels.residual_norm_backward(v["dr"], v["dh"], f, v["x"], stats, want=("f", "x"), **opts)
        keep = [0, 2, 3, 5]
        for a, b in ((r, clean[0]), (h, clean[1]), (g["f"], g0["f"]), (g["x"], g0["x"])):
            assert torch.equal(a[keep], b[keep]) and not bool(a[1].isfinite().any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured(cuda_device, dtype):
    from dance_amd import kernels
    sets = [narrow._inputs(300, 4200, dtype, "channel", "layer", seed=s) for s in (1, 2, 3)]

    def step(v):
        opts = dict(post=(v["w1"], v["b1"]), gate=v["gate"], gate_sigmoid=True, scale=0.5, pre=(v["w2"], v["b2"]))
        r, h, stats = kernels.residual_norm_forward(v["f"], v["x"], want_stats=True, **opts)
        return [r, h, *kernels.residual_norm_backward(v["dr"], v["dh"], v["f"], v["x"], stats, **opts).values()]

    eager = [[t.clone() for t in step(v)] for v in sets]
    static = {k: None if t is None else t.clone() for k, t in sets[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for turn in (0, 1, 2, 0, 1):
        for k, t in sets[turn].items():
            if t is not None:
                static[k].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager[turn]))
        assert all(torch.equal(a, b) for a, b in zip(step(sets[turn]), eager[turn]))


def test_layers_take_wide_rows(cuda_device):
    from dance_amd.nn import GatedResidualNorm, RowNorm
    x = torch.randn(4, 6001, device=DEV, requires_grad=True)
    y = RowNorm(6001, kind="rms").to(DEV)(x)
    r, h = GatedResidualNorm(6001).to(DEV)(y, x)
    (r.sum() + h.square().sum()).backward()
    assert r.shape == h.shape == x.grad.shape == (4, 6001) and bool(x.grad.isfinite().all())


def test_no_rows_and_refusals(cuda_device):
    from dance_amd.autograd import residual_norm
    f = torch.zeros(0, 5000, device=DEV, requires_grad=True)
    w, b = (torch.ones(5000, device=DEV, requires_grad=True) for _ in range(2))
    r, h = residual_norm(f, None, post=(w, b), pre=(None, None))
    (r.sum() + h.sum()).backward()
    assert r.shape == (0, 5000) and not bool(w.grad.any()) and not bool(b.grad.any())
    with pytest.raises(ValueError, match="8192"):
        residual_norm(torch.zeros(2, 8193, device=DEV), post=(None, None))
    with pytest.raises(ValueError, match="4096"):
        residual_norm(torch.zeros(2, 5000, device=DEV), torch.zeros(2, 5000, device=DEV), gate=torch.zeros(2, 1, device=DEV))


def test_more_rows_than_one_grid_dimension(cuda_device):
    """The rows of the backward lie on two grid dimensions of 2^20 workgroups in the first: rows on both sides of that border."""
    from dance_amd import kernels
    M, D = 2**20 + 3, 4097
    gen = torch.Generator(device=DEV).manual_seed(1)
    f = torch.empty(M, D, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    dr = torch.empty_like(f).normal_(generator=gen)
    gate = torch.full((M, 1), 0.5, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(D, device=DEV)
    r, _, stats = kernels.residual_norm_forward(f, post=(w, None), gate=gate, want_stats=True)
    g = kernels.residual_norm_backward(dr, None, f, None, stats, post=(w, None), gate=gate, want=("f", "gate"))
    rows = torch.tensor([0, 1, 500_000, 2**20 - 1, 2**20, 2**20 + 1, 2**20 + 2], device=DEV)
    v = dict(f=f[rows], x=None, gate=gate[rows], w1=w, b1=None, w2=None, b2=None, dr=dr[rows], dh=None)
    ref = narrow._reference(v, "row", "none", "layer", 1.0, 1e-5)
    narrow._check(r[rows], ref["r"], narrow.C_FWD, "r")
    for k in ("f", "gate"):
        narrow._check(g[k][rows], ref[k], narrow.C_BWD, k)

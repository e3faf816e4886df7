"""GPU: the global norm of many tensors and their scaling (dh_grad_norm, dh_grad_clip, kernels.clip_grad_norm_) against float64.

Tolerance: the sums are double (relative error far below 2^-24), so the fp32 norm is off by its own rounding, half a step = 2^-24 (counted
as 1.01 x 2^-24 for the double part); a scaled value by the rounding of the factor and of the product, 2 x 2^-24 (2.01), and a bf16 result
by half a step of its own, 2^-8."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0**-24

SETS = {
    "one": [(1, )],
    "small": [(7, ), (3, 5), (), (64, 64), (1, 1)],
    "empty": [(0, ), (5, ), (0, 3), (4096, ), (4097, ), (4095, )],
    "many": [(1 + (i * 37) % 90, ) for i in range(300)],           # three launches
    "long": [(2000, 512), (512, ), (512, 30), (3, 4096 * 3 + 1)],
    "huge": [(5_000_000, ), (17, )],                                # more chunks than workgroups
}


def _make(name, dtype, seed=0, scale=0.1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [(scale * torch.randn(s, generator=gen, device=DEV)).to(dtype) for s in SETS[name]]


def _norm64(ts, p):
    flat = torch.cat([t.reshape(-1).double().cpu() for t in ts])
    return float(torch.linalg.vector_norm(flat, ord=p)) if flat.numel() else 0.0


def _check(got, ref, factor):
    want = ref.double() * factor
    rel = 2.01 * U + (2.0**-8 * (1 + 2.01 * U) if got.dtype == torch.bfloat16 else 0.0)
    # below the smallest normal number a step is a fixed 2^-149 (fp32) or 2^-133 (bf16)
    assert bool(((got.double() - want).abs() <= rel * want.abs() + 2.0**-133).all())


@pytest.mark.parametrize("name", sorted(SETS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_norm_and_clip(cuda_device, name, dtype, p):
    from dance_amd import kernels
    ts = _make(name, dtype)
    ref = [t.clone() for t in ts]
    norm = _norm64(ts, p)
    assert abs(float(kernels.global_norm(ts, p)) - norm) <= 1.01 * U * norm
    for max_norm in (0.25 * norm, 4 * norm, 0.0):
        for out_dtype in (torch.float32, torch.bfloat16):
            out = [torch.full(t.shape, 9.0, dtype=out_dtype, device=DEV) for t in ts]
            got = kernels.clip_grads(ts, max_norm, norm_type=p, out=out)
            assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - norm) <= 1.01 * U * norm
            factor = min(1.0, max_norm / (norm + 1e-6))
            for o, r, t in zip(out, ref, ts):
                assert torch.equal(t, r)
                _check(o, r, factor)
        mine = [t.clone() for t in ts]
        kernels.clip_grads(mine, max_norm, norm_type=p)
        for m, r in zip(mine, ref):
            if factor == 1.0:
                assert torch.equal(m, r)
            else:
                _check(m, r, factor)


def test_mixed_types_and_flat_views(cuda_device):
    """fp32 and bf16 tensors in one call, as views of flat buffers that start at every residue of 16 bytes; the bytes between stay."""
    from dance_amd import kernels
    gen = torch.Generator(device=DEV).manual_seed(3)
    ts, flats = [], []
    for dtype in (torch.float32, torch.bfloat16):
        flat = torch.randn(60000, generator=gen, device=DEV).to(dtype)
        at = 1
        for n in (1, 2, 5, 8, 4096, 4099, 9000, 3, 20000):
            ts.append(flat[at:at + n])
            at += n + 1
        flats.append(flat)
    before = [f.clone() for f in flats]
    refs = [t.clone() for t in ts]
    norm = _norm64(ts, 2.0)
    got = kernels.clip_grads(ts, 0.5 * norm)
    assert abs(float(got) - norm) <= 1.01 * U * norm
    for t, r in zip(ts, refs):
        _check(t, r, 0.5 * norm / (norm + 1e-6))
    touched = sum(t.numel() for t in ts)
    assert sum(int((f != b).sum()) for f, b in zip(flats, before)) <= touched
    for f, b in zip(flats, before):
        at = 1
        for n in (1, 2, 5, 8, 4096, 4099, 9000, 3, 20000):
            assert torch.equal(f[at - 1:at], b[at - 1:at])
            at += n + 1


def test_layouts(cuda_device):
    """Transposed gradients are scaled where they lie, column slices through copies; what lies beside a slice stays."""
    from dance_amd import kernels
    base = torch.randn(40, 30, device=DEV)
    trans, wide = base.t(), torch.randn(50, 20, device=DEV)
    cols = wide[:, 3:9]
    ref_t, ref_w = base.clone(), wide.clone()
    norm = _norm64([trans, cols], 2.0)
    kernels.clip_grads([trans, cols], 0.3 * norm)
    factor = 0.3 * norm / (norm + 1e-6)
    _check(base, ref_t, factor)
    _check(cols, ref_w[:, 3:9], factor)
    assert torch.equal(wide[:, :3], ref_w[:, :3]) and torch.equal(wide[:, 9:], ref_w[:, 9:])
    out = [torch.zeros(40, 30, device=DEV).t(), torch.zeros(50, 20, device=DEV)[:, 2:8]]  # outputs in those layouts
    src = [torch.randn(30, 40, device=DEV), torch.randn(50, 6, device=DEV)]
    norm = _norm64(src, 2.0)
    kernels.clip_grads(src, 0.5 * norm, out=out)
    for o, s in zip(out, src):
        _check(o, s, 0.5 * norm / (norm + 1e-6))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_extreme_values(cuda_device, dtype):
    from dance_amd import kernels
    big = [torch.full((5000, ), 3e38, dtype=dtype, device=DEV), torch.full((5, ), -2e38, dtype=dtype, device=DEV)]
    norm = _norm64(big, 2.0)
    ref = [t.clone() for t in big]
    got = kernels.clip_grads(big, 1.0)  # the sum of squares is far outside fp32, and so is the norm: the scaling is still right
    assert float(got) == math.inf and norm > 3.4e38
    for t, r in zip(big, ref):
        _check(t, r, 1.0 / norm)
    tiny = [torch.full((4096, ), 1e-30, dtype=dtype, device=DEV)]
    norm = _norm64(tiny, 2.0)
    assert abs(float(kernels.global_norm(tiny)) - norm) <= 1.01 * U * norm
    zero = [torch.zeros(100, dtype=dtype, device=DEV)]
    assert float(kernels.clip_grads(zero, 1.0)) == 0.0 and not bool(zero[0].any())
    for p in (1.0, 2.0, math.inf):
        ts = _make("small", dtype)
        ts[3][5, 7] = float("nan")
        ref = [t.clone() for t in ts]
        assert math.isnan(float(kernels.clip_grads(ts, 1.0, norm_type=p)))
        assert all(bool(t.isnan().all()) for t in ts)                     # as torch: min(1, nan) is nan
        ts = ref
        ts[3][5, 7] = float("-inf")
        finite = [t.isfinite() for t in ts]
        assert float(kernels.clip_grads(ts, 1.0, norm_type=p)) == math.inf
        assert all(bool((t[f] == 0).all()) for t, f in zip(ts, finite)) and bool(ts[3][5, 7].isnan())


def test_clip_grad_norm_matches_torch(cuda_device):
    from dance_amd import kernels
    torch.manual_seed(0)
    for max_norm in (0.1, 100.0):
        a = torch.nn.Sequential(torch.nn.Linear(50, 70), torch.nn.ReLU(), torch.nn.Linear(70, 9)).to(DEV)
        a[0].weight.requires_grad_(False)  # a parameter without a gradient
        x = torch.randn(33, 50, device=DEV)
        a(x).square().sum().backward()
        ref = [p.grad.clone() for p in a.parameters() if p.grad is not None]
        norm = _norm64(ref, 2.0)
        version = a[0].bias.grad._version
        got = kernels.clip_grad_norm_(a.parameters(), max_norm)
        assert a[0].bias.grad._version > version
        assert abs(float(got) - norm) <= 1.01 * U * norm
        grads = [p.grad for p in a.parameters() if p.grad is not None]
        for g, r in zip(grads, ref):
            _check(g, r, min(1.0, max_norm / (norm + 1e-6)))
    p = torch.nn.Parameter(torch.zeros(3, device=DEV))
    p.grad = torch.tensor([1.0, float("inf"), 2.0], device=DEV)
    with pytest.raises(RuntimeError, match="non-finite"):
        kernels.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert p.grad.tolist() == [1.0, math.inf, 2.0]


def test_refusals(cuda_device):
    from dance_amd import _lib, kernels
    t = torch.ones(8, 8, device=DEV)
    for call in (lambda: kernels.clip_grads([t, t], 1.0), lambda: kernels.clip_grads([t, t[2:3]], 1.0), lambda: kernels.clip_grads([t], -1.0),
                 lambda: kernels.clip_grads([t], float("nan")), lambda: kernels.clip_grads([t], 1.0, norm_type=3), lambda: kernels.clip_grads([], 1.0),
                 lambda: kernels.global_norm([]), lambda: kernels.clip_grads([t], 1.0, out=[t[:4]]), lambda: kernels.clip_grads([t], 1.0, out=[t, t]),
                 lambda: kernels.clip_grads([t[:4], t[4:]], 1.0, out=[t[4:], t[:4]]),
                 lambda: kernels.clip_grads([torch.ones(1, device=DEV).expand(5)], 1.0)):
        with pytest.raises(ValueError):
            call()
    for bad in (t.half(), t.double(), t.to_sparse()):
        with pytest.raises(TypeError):
            kernels.clip_grads([bad], 1.0)
    with pytest.raises(TypeError):
        kernels.clip_grads([None], 1.0)
    with pytest.raises(_lib.DanceHipError):
        kernels.clip_grads([t, t.cpu()], 1.0)
    assert bool((t == 1).all())
    assert kernels.global_norm([t, t]).item() == pytest.approx(math.sqrt(128.0), rel=1e-6)  # reading one twice is counted twice

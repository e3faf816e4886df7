"""GPU: the grouped products at sizes where the large tiles take them.

Operands are small integers: every product, every partial sum and every result is a whole number below 2^24, so fp32 holds all of them
exactly in whatever order they are added, and the results have to be the float64 ones to the last bit (a bf16 result: that value rounded once).

Which kernel a size takes (gemm_grouped.hip: forward_pick, wgrad_plan): bf16 100003 x 1032 -> 520 both ways over the 256 x 256 tile (at least
256 rows a type and 768 tiles), its weight gradient too (5913 positions a chunk); fp32 30011 x 1036 -> 1028 over the 128 x 128 tile (5056
positions a chunk); rows that are no multiple of 16 bytes over the tiles staged through registers."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

LEAD = 13
SIZES = {100003: [0, 61, 50000, 0, 7, 30001, 0, 257, 19600], 30011: [300, 0, 17000, 1, 12600, 0]}  # 64 and 97 rows behind the last type


def _case(rows, K, N, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    whole = lambda *s: torch.randint(-3, 4, s, generator=g, device=DEV).to(dtype)
    sizes = SIZES[rows]
    bounds = [LEAD]
    for n in sizes:
        bounds.append(bounds[-1] + n)
    return whole(rows, K), whole(rows, N), bounds, torch.tensor(bounds, dtype=torch.int32, device=DEV), whole


@pytest.mark.parametrize("rows,K,N,dtype", [(100003, 1032, 520, torch.bfloat16), (100003, 1031, 519, torch.bfloat16), (30011, 1036, 1028, torch.float32),
                                            (30011, 1035, 1027, torch.float32)])
def test_exact(cuda_device, rows, K, N, dtype):
    from dance_amd import kernels
    x, dy, bounds, ptr, whole = _case(rows, K, N, dtype, K)
    G = len(bounds) - 1
    w, wt, b = whole(G, N, K), whole(G, K, N), whole(G, N).float()
    spans = list(zip(bounds, bounds[1:]))
    y32 = kernels.gemm_grouped(x, w, ptr, bias=b, act=kernels.ACT_RELU, out_dtype=torch.float32)
    y = kernels.gemm_grouped(x, w, ptr, bias=b, act=kernels.ACT_RELU)
    other = kernels.gemm_grouped(x, wt, ptr, trans_b=False, out_dtype=torch.float32)
    dx = kernels.gemm_grouped(dy, w, ptr, trans_b=False)
    dw, db = kernels.gemm_grouped_wgrad(dy, x, ptr, out_dtype=torch.float32, want_bias=True)
    dw_rounded = kernels.gemm_grouped_wgrad(dy, x, ptr)
    outside = [slice(0, bounds[0]), slice(bounds[-1], rows)]
    for t in (y32, y, other, dx):
        assert not any(bool(t[s].any()) for s in outside)
    for g, (i, j) in enumerate(spans):
        xd, yd = x[i:j].double(), dy[i:j].double()
        want = torch.mm(xd, w[g].double().t().contiguous()) + b[g].double()
        want.clamp_(min=0)
        assert torch.equal(y32[i:j].double(), want), g
        assert torch.equal(y[i:j], want.to(dtype)), g
        assert torch.equal(other[i:j].double(), torch.mm(xd, wt[g].double())), g
        assert torch.equal(dx[i:j], torch.mm(yd, w[g].double()).to(dtype)), g
        want = torch.mm(yd.t().contiguous(), xd)
        assert torch.equal(dw[g].double(), want), g
        assert torch.equal(dw_rounded[g], want.to(dtype)), g
        assert torch.equal(db[g].double(), yd.sum(0)), g


def test_repeats(cuda_device):
    """A persistent tile's next operands are requested while it is stored: many passes over different inputs, interleaved, give each its own bits."""
    from dance_amd import kernels
    for rows, K, N, dtype in ((100003, 520, 328, torch.bfloat16), (30011, 268, 516, torch.float32)):
        cases = [_case(rows, K, N, dtype, s) for s in (1, 2)]
        weights = [c[4](len(c[2]) - 1, N, K) for c in cases]
        first = [kernels.gemm_grouped(c[0], w, c[3]) for c, w in zip(cases, weights)]
        for turn in range(4):
            for c, w, f in zip(cases, weights, first):
                assert torch.equal(kernels.gemm_grouped(c[0], w, c[3]), f)
        c, w = cases[0], weights[0]
        for g, (i, j) in enumerate(zip(c[2], c[2][1:])):
            assert torch.equal(first[0][i:j], torch.mm(c[0][i:j].double(), w[g].double().t().contiguous()).to(dtype)), g

"""GPU: what lies behind a row's last whole access stays out of the row's sums, however large the values of a channel gate are; the forward
without the residual stream as an output."""
import pytest
import torch

import test_gpu_residual_norm as narrow

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [9, 15, 20, 23, 65, 300, 511, 513, 1001, 2050, 4095, 4097, 8191])
def test_channel_gate_of_the_lowest_value(cuda_device, dtype, D):
    """A channel whose feature is zero everywhere may carry any gate, the type's lowest value among them: 0 x gate is 0, r and h are finite, and
    so are all gradients but that channel's own."""
    from dance_amd import kernels
    M, scale = 5, 0.5
    for at in (D - 1, D - 2, 0):
        v = narrow._inputs(M, D, dtype, "channel", "layer", post=False)
        v["f"][:, :] = 4.0 * v["f"].sign()
        v["f"][:, at] = 0.0
        v["gate"][at] = torch.finfo(torch.float32).min
        opts = dict(gate=v["gate"], scale=scale, pre=(v["w2"], v["b2"]))
        r, h, stats = kernels.residual_norm_forward(v["f"], v["x"], want_stats=True, **opts)
        assert bool(r.isfinite().all()) and bool(h.isfinite().all())
        g = kernels.residual_norm_backward(v["dr"], v["dh"], v["f"], v["x"], stats, **opts)
        ref = narrow._reference(v, "channel", "none", "layer", scale, 1e-5)
        wide = 44 if D > 4096 else 0  # (the longer row sums of wide rows: 300 in place of 256)
        for k in ("x", "gate", "w2", "b2"):
            narrow._check(g[k], ref[k], narrow.C_BWD + wide + M, k)
        others = [c for c in range(D) if c != at]
        narrow._check(g["f"][:, others], narrow.V(ref["f"].v[:, others], ref["f"].m[:, others]), narrow.C_BWD + wide, "f")


def test_forward_without_the_stream(cuda_device):
    """The C entry with r = NULL: h alone, the same bits."""
    from dance_amd import _lib, kernels
    lib = _lib.load()
    for dtype in (torch.float32, torch.bfloat16):
        for D in (50, 512, 2000, 5000):
            v = narrow._inputs(9, D, dtype, "none", "layer")
            _, h, _ = kernels.residual_norm_forward(v["f"], v["x"], post=(v["w1"], v["b1"]), pre=(v["w2"], v["b2"]))
            alone = torch.zeros_like(h)
            entry = lib.dh_residual_norm_forward if D <= 4096 else lib.dh_residual_norm_wide_forward
            p = {k: None if t is None else t.data_ptr() for k, t in v.items()}
            rc = entry(9, D, 0 if dtype == torch.float32 else 1, p["f"], D, p["x"], D, None, 0, 0, 0, 1.0, 0, 1e-5, 1, p["w1"], p["b1"], 1, p["w2"], p["b2"],
                       None, 0, alone.data_ptr(), D, None, torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and torch.equal(alone, h)

"""GPU: clipping refuses tensors that share memory whatever their layout, and takes those that only interleave."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _clip(grads, max_norm, out=None):
    from dance_amd import kernels
    return kernels.clip_grads(grads, max_norm, out=out)


def test_shared_windows_are_refused(cuda_device):
    wide = torch.randn(50, 20, device=DEV)
    cube = torch.randn(6, 7, 8, device=DEV)
    dense = torch.randn(50, 6, device=DEV)
    room = torch.zeros(50, 20, device=DEV)
    before = [t.clone() for t in (wide, cube, dense, room)]
    bad = [
        ([wide[:, :6], wide[:, 3:9]], None),                          # overlapping columns
        ([wide[:, 3:9], wide[:, 3:9]], None),                         # the same slice twice
        ([wide[:, 3:9], wide[2]], None),                              # a row across a column slice
        ([wide[::2, 3:9], wide[:, 8:12]], None),                      # every second row of it
        ([wide[:, 3:9], wide.t()[5:7]], None),
        ([cube[:, 2:4], cube[2:3, :, 1]], None),
        ([cube[..., 1], cube[:, 3]], None),
        ([dense, dense.clone()], [room[:, :6], room[:, 3:9]]),        # outputs that overlap
        ([dense], [dense.as_strided((50, 6), (5, 1))]),               # an output whose own rows overlap
        ([wide[:, :6]], [wide[:, 3:9]]),                              # an output across its gradient
        ([wide[:, :6], dense], [room[:, :6], wide[:, 5:11]]),         # ... across another gradient
        ([wide[:, :6].bfloat16().float()[:, :5], wide[:, 5:9]], [room[:, :5], room.view(torch.bfloat16)[:, 9:13]]),  # in bytes: 0 .. 20 and 18 .. 26
    ]
    for grads, out in bad:
        with pytest.raises(ValueError):
            _clip(grads, 0.5, out)
    assert all(torch.equal(a, b) for a, b in zip((wide, cube, dense, room), before))


def test_interleaved_windows_are_taken(cuda_device):
    wide = torch.randn(50, 20, device=DEV)
    cube = torch.randn(6, 7, 8, device=DEV)
    sets = [
        [wide[:, :6], wide[:, 6:9], wide[:, 9:]],
        [wide[:, 0::2], wide[:, 1::2]],
        [wide[0::2, 3:9], wide[1::2, 3:9], wide[:, 9:11]],
        [cube[:, 0:2], cube[:, 2:7, 0:3], cube[:, 2:7, 3:]],
        [cube[..., 1], cube[..., 2], cube[0::3, :, 4:], cube[1::3, :, 4:]],
        [wide[:, 3:9], cube.permute(2, 0, 1), wide[:, :3]],
    ]
    for ts in sets:
        ref = [t.clone() for t in ts]
        norm = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
        whole = [wide.clone(), cube.clone()]
        got = float(_clip(ts, 0.25 * norm))
        assert abs(got - norm) <= 1.01 * 2.0**-24 * norm
        factor = 0.25 * norm / (norm + 1e-6)
        for t, r in zip(ts, ref):
            assert bool(((t.double() - r.double() * factor).abs() <= 2.01 * 2.0**-24 * r.double().abs() + 2.0**-140).all())
        moved = sum(int((a != b).sum()) for a, b in zip((wide, cube), whole))
        assert moved <= sum(t.numel() for t in ts)  # what lies between stays
    # one gradient expanded over many rows may be read: it is written into an output of its own
    row, out = torch.randn(1, 6, device=DEV), torch.zeros(50, 20, device=DEV)
    _clip([row.expand(50, 6), wide[:, :3]], 1e9, [out[:, :6], out[:, 6:9]])
    assert torch.equal(out[:, :6], row.expand(50, 6)) and torch.equal(out[:, 6:9], wide[:, :3]) and not bool(out[:, 9:].any())

"""CPU: which tensors share memory (kernels._refuse_shared_windows), against the sets of the bytes that they hold."""
import numpy as np
import pytest
import torch

from dance_amd import kernels


def _bytes_of(t):
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at.unsqueeze(-1) + torch.arange(n) * s
    size = t.element_size()
    base = t.data_ptr() + at.reshape(-1).numpy() * size
    return set((base[:, None] + np.arange(size)).reshape(-1).tolist())


def _refused(ts):
    try:
        kernels._refuse_shared_windows(ts)
        return False
    except ValueError:
        return True


@pytest.mark.parametrize("seed", range(300))
def test_pairs_of_views(seed):
    """Random slices, steps, transposes and casts of one buffer: refused exactly where they hold a common byte."""
    rng = np.random.default_rng(seed)
    shape = [(60, ), (9, 14), (4, 5, 6), (3, 4, 2, 5)][seed % 4]
    buf = torch.zeros(shape)

    def view():
        v = buf
        if rng.random() < 0.2 and v.shape[-1] % 2 == 0:
            v = v.view(torch.bfloat16) if rng.random() < 0.5 else v.view(-1)
        for d in range(v.dim()):
            if rng.random() < 0.7:
                lo = int(rng.integers(0, v.shape[d]))
                v = v[(slice(None), ) * d + (slice(lo, int(rng.integers(lo, v.shape[d])) + 1, int(rng.integers(1, 4))), )]
        return v.permute(*rng.permutation(v.dim()).tolist())

    ts = [view() for _ in range(int(rng.integers(2, 4)))]
    held = [_bytes_of(t) for t in ts]
    meet = any(held[i] & held[j] for i in range(len(ts)) for j in range(i))
    assert _refused(ts) == meet


def test_many_rows_of_different_strides():
    buf = torch.zeros(4_000_000)
    a, b = buf.view(200_000, 20)[:, :6], buf.view(160_000, 25)[:, 20:24]
    assert _refused([a, b])
    even, odd = buf.view(2_000_000, 2)[:, 0], buf.view(1_000_000, 4)[:, 1]
    assert not _refused([even, odd]) and _refused([even, buf.view(1_000_000, 4)[:, 2]])


def test_empty_and_scalar():
    buf = torch.zeros(8)
    assert not _refused([buf, buf[3:3], torch.zeros(()), buf.view(2, 4)[:, :0]]) and _refused([buf, buf[5]])

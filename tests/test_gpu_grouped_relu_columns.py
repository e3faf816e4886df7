"""GPU: a fused ReLU over a single output column, whose gradient may come with any stride of that column (the transpose of a row)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [1, 24])
def test_grouped_linear(cuda_device, dtype, K):
    from dance_amd.autograd import grouped_linear
    ptr = torch.tensor([0, 7, 20, 33], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(K)
    draw = lambda *shape: torch.randn(*shape, generator=g).to(DEV, dtype)
    x, w, b, dy = draw(33, K), draw(3, 1, K), draw(3, 1).float(), draw(33, 1)
    results = []
    for stride in (1, 33, 7):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = grouped_linear(leaves[0], leaves[1], ptr, leaves[2], relu=True)
        up = dy.as_strided(dy.shape, (1, stride))
        assert up.is_contiguous()
        y.backward(up)
        results.append([y.detach()] + [t.grad for t in leaves])
    assert all(torch.equal(a, c) for other in results[1:] for a, c in zip(results[0], other))
    assert bool((results[0][0] > 0).any()) and bool((results[0][0] == 0).any())


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_transposed_output(cuda_device, dtype, relu):
    """The transpose of a [M, 1] output, as a loss meets it; the untyped layer beside the typed one."""
    from dance_amd.autograd import grouped_linear, linear
    g = torch.Generator().manual_seed(1)
    x = torch.randn(9, 8, generator=g).to(DEV, dtype)
    w = torch.randn(1, 8, generator=g).to(DEV)
    c = torch.randn(1, 9, generator=g).to(DEV, dtype)
    ptr = torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    for layer in (lambda xx, ww: grouped_linear(xx, ww[None], ptr, relu=relu), lambda xx, ww: linear(xx, ww, relu=relu)):
        grads = []
        for transposed in (True, False):
            leaves = [t.clone().requires_grad_() for t in (x, w)]
            y = layer(*leaves)
            ((y.t() * c) if transposed else (y * c.t().contiguous())).sum().backward()
            grads.append([t.grad for t in leaves])
        assert all(torch.equal(a, b) for a, b in zip(*grads))

"""GPU: a typed residual block and its training step as they are used together — TypedLinear, GatedResidualNorm / RowNorm, clip_grad_norm_ —
eagerly, captured and replayed, on other streams, from two threads, and beyond 2^31 elements.  Every kernel sums in a fixed order, so the
comparisons between ways of running the same step are exact."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0**-24


class Block(torch.nn.Module):

    def __init__(self, dim, hidden, types, seed=0):
        super().__init__()
        from dance_amd.nn import GatedResidualNorm, TypedLinear
        torch.manual_seed(seed)
        self.up, self.down = TypedLinear(dim, hidden, types), TypedLinear(hidden, dim, types)
        self.join = GatedResidualNorm(dim, gate="channel", gate_act="sigmoid", scale=0.5)

    def forward(self, x, ptr):
        return self.join(self.down(self.up(x, ptr, fuse_relu=True), ptr), x)


def _data(rows=700, dim=72, types=5, dtype=torch.float32, seed=1):
    gen = torch.Generator().manual_seed(seed)
    from dance_amd.nn import group_rows
    kind = torch.randint(0, types, (rows, ), generator=gen)
    order, ptr = group_rows(kind.to(DEV), types)
    x = torch.randn(rows, dim, generator=gen).to(DEV)[order].to(dtype)
    ups = [torch.randn(rows, dim, generator=gen).to(DEV).to(dtype) for _ in range(2)]
    return x, ptr, ups


def _step(block, x, ptr, ups, max_norm=1.0):
    """(outputs, clipped gradients, norm) of one pass, without touching .grad."""
    from dance_amd import kernels
    params = list(block.parameters())
    r, h = block(x, ptr)
    grads = [g.contiguous() for g in torch.autograd.grad([r, h], params, ups)]
    norm = kernels.clip_grads(grads, max_norm)
    return [r.detach(), h.detach(), *grads, norm]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_is_its_operators(cuda_device, dtype):
    """The module's outputs and gradients are, bit for bit, those of the operators called one after the other (each of them is held to
    float64 in its own tests), and the clipped gradients are the unclipped ones times the factor."""
    from dance_amd import kernels
    x, ptr, (ur, uh) = _data(dtype=dtype)
    block = Block(72, 96, 5).to(DEV)
    j = block.join
    w1, w2 = (m.weight.detach().to(dtype) for m in (block.up, block.down))
    a = kernels.gemm_grouped(x, w1, ptr, bias=block.up.bias.detach(), act=kernels.ACT_RELU)
    f = kernels.gemm_grouped(a, w2, ptr, bias=block.down.bias.detach())
    post, pre = (j.post_weight.detach(), j.post_bias.detach()), (j.pre_weight.detach(), j.pre_bias.detach())
    opts = dict(post=post, gate=j.gate.detach(), gate_sigmoid=True, scale=0.5, pre=pre)
    r, h, stats = kernels.residual_norm_forward(f, x, want_stats=True, **opts)
    g = kernels.residual_norm_backward(ur, uh, f, x, stats, **opts)
    dw2, db2 = kernels.gemm_grouped_wgrad(g["f"], a, ptr, out_dtype=torch.float32, want_bias=True)
    da = kernels.gemm_grouped(g["f"], w2, ptr, trans_b=False)
    da = da * (a > 0)
    dw1, db1 = kernels.gemm_grouped_wgrad(da, x, ptr, out_dtype=torch.float32, want_bias=True)
    want = {"up.weight": dw1, "up.bias": db1, "down.weight": dw2, "down.bias": db2, "join.post_weight": g["w1"], "join.post_bias": g["b1"],
            "join.pre_weight": g["w2"], "join.pre_bias": g["b2"], "join.gate": g["gate"]}
    mr, mh = block(x, ptr)
    assert torch.equal(mr.detach(), r) and torch.equal(mh.detach(), h)
    torch.autograd.backward([mr, mh], [ur, uh])
    for name, p in block.named_parameters():
        assert torch.equal(p.grad, want[name]), name
    before = [p.grad.clone() for p in block.parameters()]
    norm = kernels.clip_grad_norm_(block.parameters(), 0.5)
    ref = float(torch.cat([b.reshape(-1).double() for b in before]).norm())
    assert abs(float(norm) - ref) <= 1.01 * U * ref
    for p, b in zip(block.parameters(), before):
        want_g = b.double() * (0.5 / (ref + 1e-6))
        assert bool(((p.grad.double() - want_g).abs() <= 2.01 * U * want_g.abs() + 2.0**-140).all())


def test_training_runs(cuda_device):
    """A few clipped Adam steps on a random task: everything stays finite and every parameter moves."""
    from dance_amd import kernels
    x, ptr, (target, _) = _data()
    block = Block(72, 96, 5).to(DEV)
    opt = torch.optim.Adam(block.parameters(), lr=1e-2)
    start = [p.detach().clone() for p in block.parameters()]
    for _ in range(5):
        opt.zero_grad()
        r, h = block(x, ptr)
        ((h - target).square().mean() + r.square().mean()).backward()
        norm = kernels.clip_grad_norm_(block.parameters(), 0.1)
        opt.step()
    assert bool(torch.isfinite(norm)) and all(bool(p.isfinite().all()) and not torch.equal(p, s) for p, s in zip(block.parameters(), start))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_step(cuda_device, dtype):
    """Forward, backward and clipping in a graph; two graphs over different inputs, replayed in turn with eager work and synchronisations in
    between: every replay gives the eager step's bits for the inputs it finds."""
    block = Block(72, 96, 5).to(DEV)
    sets = [_data(dtype=dtype, seed=s) for s in (1, 2, 3, 4)]
    eager = [[t.clone() for t in _step(block, *s)] for s in sets]
    static = [[sets[k][0].clone(), sets[k][1].clone(), [u.clone() for u in sets[k][2]]] for k in (0, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            _step(block, *s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(block, *s))
        graphs.append(graph)
    for turn in range(4):
        for k in (0, 1):
            src = (2 * turn + k) % 4
            static[k][0].copy_(sets[src][0])
            static[k][1].copy_(sets[src][1])
            for to, u in zip(static[k][2], sets[src][2]):
                to.copy_(u)
            graphs[k].replay()
            noise = torch.randn(3000, 300, device=DEV).sum()  # eager work between the replays
            if turn % 2:
                torch.cuda.synchronize()
            got = [t.clone() for t in outs[k]]
            assert all(torch.equal(g, e) for g, e in zip(got, eager[src])), (turn, k)
            assert bool(noise.isfinite())


def test_other_streams_and_threads(cuda_device):
    block = Block(72, 96, 5).to(DEV)
    data = [_data(seed=s) for s in (5, 6)]
    eager = [[t.clone() for t in _step(block, *d)] for d in data]
    torch.cuda.synchronize()
    results, errors = [None, None], []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    out = _step(block, *data[k])
            stream.synchronize()
            results[k] = out
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k, )) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(results[k], eager[k]))


def test_modules(cuda_device):
    from dance_amd.nn import GatedResidualNorm, RowNorm, TypedLinear, group_rows
    types = torch.tensor([2, 0, -1, 2, 5, 0, 3], device=DEV)
    order, ptr = group_rows(types, 4)
    layer = TypedLinear(8, 5, 4).to(DEV)
    x = torch.randn(7, 8, device=DEV)
    y = torch.empty(7, 5, device=DEV)
    y[order] = layer(x[order], ptr).detach()
    for i, t in enumerate(types.tolist()):
        want = x[i].double() @ layer.weight[t].double().t() + layer.bias[t].double() if 0 <= t < 4 else torch.zeros(5, device=DEV, dtype=torch.float64)
        mag = x[i].double().abs() @ layer.weight[t].double().abs().t() + layer.bias[t].double().abs() if 0 <= t < 4 else torch.zeros(5, device=DEV)
        assert bool(((y[i].double() - want.detach()).abs() <= 11 * 2 * U * mag.detach()).all())
    assert sorted(TypedLinear(3, 2, 2, bias=False).state_dict()) == ["weight"]
    assert sorted(GatedResidualNorm(4, kind="rms").state_dict()) == ["gate", "post_weight", "pre_weight"]
    with pytest.raises(ValueError):
        GatedResidualNorm(4, gate="row")
    with pytest.raises(ValueError):
        GatedResidualNorm(8).to(DEV)(x, x, gate=torch.ones(7, 1, device=DEV))
    r, h = GatedResidualNorm(8, gate=None, pre=False).to(DEV)(x, x, gate=torch.zeros(7, 1, device=DEV))
    assert h is None and torch.equal(r.detach(), x)
    plain = RowNorm(8, affine=False)
    assert not list(plain.parameters()) and plain(x).shape == (7, 8)


def test_row_norm_in_the_sage_layer(cuda_device):
    """The ``norm`` slot of the framework's own layer: norm(relu(Linear(h_dst))), against float64.  The layer's product carries at most
    (K + 2) 2^-23 of its terms (tests/test_gpu_gemm_grouped.py's count), the norm passes that on times rstd w and adds its own 60 roundings."""
    from dance_amd.nn import AdaptiveSAGE, RowNorm
    from test_gpu_fullsize import _cellgene_graph
    cg = _cellgene_graph(300, 50, 10, 16, seed=3)
    block = cg.cell_rows_block()
    n = block.number_of_dst_nodes()
    torch.manual_seed(0)
    h = torch.randn(cg.number_of_nodes(), 24, device=DEV)
    layer = AdaptiveSAGE(24, 40, torch.nn.Parameter(torch.ones(52, 1, device=DEV)), torch.nn.Dropout(0.0), torch.nn.ReLU(), RowNorm(40),
                         compute_neigh=False).to(DEV)
    with torch.no_grad():
        layer.layers[3].weight.copy_(1 + 0.1 * torch.randn(40))
        layer.layers[3].bias.copy_(0.1 * torch.randn(40))
    out = layer(block, h)
    off = getattr(block, "dst_offset", 0)
    lin, norm = layer.layers[1], layer.layers[3]
    x = h[off:off + n].double()
    z = torch.relu(x @ lin.weight.double().t() + lin.bias.double())
    ez = (24 + 2) * 2 * U * (x.abs() @ lin.weight.double().abs().t() + lin.bias.double().abs())
    rstd = (z.var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    zhat = (z - z.mean(1, keepdim=True)) * rstd
    want = zhat * norm.weight.double() + norm.bias.double()
    spread = (ez + ez.mean(1, keepdim=True)) * rstd
    tol = norm.weight.double().abs() * (spread + zhat.abs() * (zhat.abs() * spread).mean(1, keepdim=True)) + 60 * U * ((z.abs() + z.mean(1, keepdim=True)) * rstd + 1)
    assert bool(((out.double() - want).abs() <= tol).all())
    out.sum().backward()
    assert lin.weight.grad is not None and norm.weight.grad is not None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_relu_of_odd_and_empty_outputs(cuda_device, dtype):
    from dance_amd.autograd import grouped_linear
    for rows, n in ((0, 24), (9, 17), (9, 1)):
        x = torch.randn(rows, 12, device=DEV).to(dtype).requires_grad_(True)
        w = torch.randn(2, n, 12, device=DEV).to(dtype).requires_grad_(True)
        b = torch.randn(2, n, device=DEV, requires_grad=True)
        ptr = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=DEV)
        y = grouped_linear(x, w, ptr, b, relu=True)
        up = torch.randn(rows, n, device=DEV).to(dtype)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), up)
        assert gx.shape == x.shape and gw.shape == w.shape
        masked = (up * (y > 0)).float()
        for g, (i, j) in enumerate(((0, rows // 2), (rows // 2, rows))):
            assert bool(((gb[g] - masked[i:j].sum(0)).abs() <= 1e-6 * masked[i:j].abs().sum(0)).all())


def test_differentiated_twice_is_refused(cuda_device):
    from dance_amd.autograd import grouped_linear, residual_norm
    x = torch.randn(6, 12, device=DEV, requires_grad=True)
    w = torch.randn(1, 5, 12, device=DEV, requires_grad=True)
    ptr = torch.tensor([0, 6], dtype=torch.int32, device=DEV)
    for y in (grouped_linear(x, w, ptr), residual_norm(x, None, post=(None, None))[0]):
        (g, ) = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_beyond_32_bit_offsets(cuda_device):
    """1.1 million rows of 2000 bf16 values: element offsets up to 2.2e9.  The last rows against the same rows on their own."""
    from dance_amd import kernels
    M, K, N = 1_100_000, 2000, 24
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(M, K, device=DEV, generator=gen, dtype=torch.bfloat16)
    w = torch.randn(3, N, K, device=DEV, generator=gen).to(torch.bfloat16)
    ptr = torch.tensor([0, M // 2, M - 70, M], dtype=torch.int32, device=DEV)
    y = kernels.gemm_grouped(x, w, ptr, out_dtype=torch.float32)
    for rows, g in ((slice(M - 70, M), 2), (slice(M - 90, M - 70), 1), (slice(0, 40), 0)):
        xd, wd = x[rows].double(), w[g].double()
        assert bool(((y[rows].double() - xd @ wd.t()).abs() <= (K + 3) * 2 * U * (xd.abs() @ wd.abs().t())).all())
    dy = torch.randn(M, N, device=DEV, generator=gen).to(torch.bfloat16)
    dw = kernels.gemm_grouped_wgrad(dy, x, ptr, out_dtype=torch.float32)
    xd, yd = x[M - 70:].double(), dy[M - 70:].double()
    assert bool(((dw[2].double() - yd.t() @ xd).abs() <= 73 * 2 * U * (yd.abs().t() @ xd.abs())).all())
    back = kernels.gemm_grouped(dy, w, ptr, trans_b=False)  # the 2.2e9 values are written
    ref = dy[M - 70:].double() @ w[2].double()
    mag = dy[M - 70:].double().abs() @ w[2].double().abs()
    assert bool(((back[M - 70:].double() - ref).abs() <= (N + 3) * 2 * U * mag + 2.0**-8 * (ref.abs() + (N + 3) * 2 * U * mag)).all())
    del y, dy, dw
    r, h, stats = kernels.residual_norm_forward(x, back, post=(None, None), pre=(None, None), want_stats=True)
    tail = slice(M - 50, M)
    r2, h2, stats2 = kernels.residual_norm_forward(x[tail], back[tail], post=(None, None), pre=(None, None), want_stats=True)
    assert torch.equal(r[tail], r2) and torch.equal(h[tail], h2) and torch.equal(stats[tail], stats2)
    g = kernels.residual_norm_backward(h, r, x, back, stats, post=(None, None), pre=(None, None), want=("f", "x"))
    g2 = kernels.residual_norm_backward(h[tail], r[tail], x[tail], back[tail], stats2, post=(None, None), pre=(None, None), want=("f", "x"))
    assert torch.equal(g["f"][tail], g2["f"]) and torch.equal(g["x"][tail], g2["x"])
    del r, h, g, stats, back
    flat = x.view(-1)
    parts = [float(kernels.global_norm([flat[:flat.numel() // 2]])), float(kernels.global_norm([flat[flat.numel() // 2:]]))]
    whole = float(kernels.clip_grads([flat], 1.0))
    assert abs(whole**2 - parts[0]**2 - parts[1]**2) <= 8 * U * whole**2
    assert bool((flat[-64:].float().abs() <= 10.0 / whole).all())

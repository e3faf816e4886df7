"""CPU: the refusals of the grouped products, the residual norm and the gradient clipping at the C ABI (nothing is launched: every call
returns before it reaches the device), the closed form by which a launch finds a row slot's group, and the wrappers' host logic."""
import ctypes

import numpy as np
import pytest
import torch

from dance_amd import _lib, kernels

P = 4096  # some non-null address: no call below may get as far as using it
INVALID, WORKSPACE = -1, -3


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _grouped(lib, **kw):
    a = dict(M=8, N=4, K=4, G=2, trans_b=1, dtype=0, X=P, ldx=4, W=P, ldw=4, stride_w=16, ptr=P, bias=None, ld_bias=0, act=0, Y=P, ldy=4, y_dtype=0,
             zero=1, stream=None)
    a.update(kw)
    return lib.dh_gemm_grouped(*a.values())


@pytest.mark.parametrize("bad", [dict(M=-1), dict(N=-1), dict(K=-1), dict(G=-1), dict(M=2**31), dict(dtype=2), dict(y_dtype=-1), dict(act=7), dict(X=None),
                                 dict(W=None), dict(ptr=None), dict(Y=None), dict(ldx=3), dict(ldw=3), dict(ldy=3), dict(bias=P, ld_bias=3),
                                 dict(stride_w=-1)])
def test_grouped_refusals(lib, bad):
    assert _grouped(lib, **bad) == INVALID
    assert b"dh_gemm_grouped" in lib.dh_last_error_string()


def test_grouped_nothing_to_do(lib):
    assert _grouped(lib, M=0, X=None, Y=None) == 0 and _grouped(lib, N=0, Y=None) == 0


def _wgrad(lib, **kw):
    a = dict(M=8, N=4, K=4, G=2, dtype=0, dY=P, ldy=4, X=P, ldx=4, ptr=P, dW=P, ldw=4, stride_w=16, dw_dtype=0, db=None, ld_db=0, ws=P, ws_bytes=1 << 20,
             stream=None)
    a.update(kw)
    return lib.dh_gemm_grouped_wgrad(*a.values())


@pytest.mark.parametrize("bad", [dict(M=-1), dict(G=-1), dict(dtype=9), dict(dw_dtype=9), dict(dY=None), dict(X=None), dict(ptr=None), dict(dW=None),
                                 dict(ldy=3), dict(ldx=3), dict(ldw=3), dict(stride_w=15), dict(db=P, ld_db=3), dict(ws=P + 4), dict(K=0, db=P, ld_db=4)])
def test_grouped_wgrad_refusals(lib, bad):
    assert _wgrad(lib, **bad) == INVALID


def test_grouped_wgrad_workspace(lib):
    need = lib.dh_gemm_grouped_wgrad_workspace_bytes(8, 4, 4, 2, 0)
    assert _wgrad(lib, ws_bytes=need - 1) == WORKSPACE and _wgrad(lib, ws=None) == WORKSPACE
    for dtype in (0, 1):
        assert lib.dh_gemm_grouped_wgrad_workspace_bytes(31, 512, 2000, 1, dtype) == 16        # one chunk of rows: no partial results
        assert lib.dh_gemm_grouped_wgrad_workspace_bytes(200003, 512, 2000, 9, dtype) >= 2 * 2 * 512 * 2001 * 4


def _norm_fwd(lib, **kw):
    a = dict(M=4, D=8, dtype=0, f=P, ldf=8, x=P, ldx=8, gate=None, ldg=0, gk=0, sig=0, scale=1.0, kind=0, eps=1e-5, post=1, w1=None, b1=None, pre=1,
             w2=None, b2=None, r=P, ldr=8, h=P, ldh=8, stats=P, stream=None)
    a.update(kw)
    return lib.dh_residual_norm_forward(*a.values())


@pytest.mark.parametrize("bad", [dict(M=-1), dict(D=0), dict(D=4097, ldf=4097, ldx=4097, ldr=4097, ldh=4097), dict(dtype=3), dict(kind=2), dict(gk=5),
                                 dict(gk=-1), dict(sig=2), dict(eps=-1.0), dict(eps=float("nan")), dict(f=None), dict(gk=1), dict(ldf=7), dict(ldx=7),
                                 dict(gk=4, gate=P, ldg=7), dict(gk=3, gate=P, ldg=0), dict(h=None), dict(r=None, pre=0), dict(ldr=7), dict(ldh=7),
                                 dict(stats=P + 4)])
def test_residual_norm_forward_refusals(lib, bad):
    assert _norm_fwd(lib, **bad) == INVALID
    assert _norm_fwd(lib, M=0) == 0


def _norm_bwd(lib, **kw):
    a = dict(M=4, D=8, dtype=0, f=P, ldf=8, x=P, ldx=8, gate=None, ldg=0, gk=0, sig=0, scale=1.0, kind=0, post=1, w1=None, b1=None, pre=1, w2=None,
             stats=P, dr=P, lddr=8, dh=P, lddh=8, df=P, lddf=8, dx=P, lddx=8, dgate=None, lddg=0, dw1=None, db1=None, dw2=None, db2=None, ws=P,
             ws_bytes=1 << 20, stream=None)
    a.update(kw)
    return lib.dh_residual_norm_backward(*a.values())


@pytest.mark.parametrize("bad", [dict(D=0), dict(stats=None), dict(stats=P + 8), dict(pre=0), dict(dr=None, dh=None), dict(lddr=7), dict(lddh=7),
                                 dict(lddf=7), dict(lddx=7), dict(gk=4, gate=P, ldg=8, dgate=P, lddg=7), dict(post=0, dw1=P),
                                 dict(post=0, db1=P), dict(pre=0, dh=None, dw2=P), dict(pre=0, dh=None, db2=P), dict(dgate=P)])
def test_residual_norm_backward_refusals(lib, bad):
    assert _norm_bwd(lib, **bad) == INVALID
    assert _norm_bwd(lib, ws_bytes=lib.dh_residual_norm_backward_workspace_bytes(4, 8) - 1) == WORKSPACE


def _clip(lib, n=2, in_ptr=(P, P * 2), out_ptr=(P, P * 2), numel=(4, 4), dt=(0, 0), odt=(0, 0), norm_type=2, max_norm=1.0, norm=P, ws=P, ws_bytes=1 << 16):
    vp, i64, i32 = ctypes.c_void_p * 2, ctypes.c_int64 * 2, ctypes.c_int32 * 2
    return lib.dh_grad_clip(n, vp(*in_ptr), vp(*out_ptr), i64(*numel), i32(*dt), i32(*odt), norm_type, max_norm, norm, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(norm_type=3), dict(norm=None), dict(numel=(4, -1)), dict(in_ptr=(P, None)), dict(out_ptr=(None, P)),
                                 dict(dt=(0, 2)), dict(odt=(5, 0)), dict(dt=(1, 0)), dict(ws=P + 8)])
def test_grad_clip_refusals(lib, bad):
    assert _clip(lib, **bad) == INVALID


def test_grad_clip_workspace(lib):
    numel = (ctypes.c_int64 * 2)(4, 4)
    assert _clip(lib, ws_bytes=lib.dh_grad_norm_workspace_bytes(2, numel) - 1) == WORKSPACE
    assert lib.dh_grad_norm_workspace_bytes(2, numel) == 16 + 8 * 2
    many = (ctypes.c_int64 * 300)(*([1 << 30] * 300))
    assert lib.dh_grad_norm_workspace_bytes(300, many) >= 16 + 8 * 1024 * 3


# ---- the closed form of the row slots (gemm_grouped.hip: Groups, find_slot, the partial slots of the weight gradient) ----
def _edges(ptr, M):
    return [0] + [min(max(int(p), 0), M) for p in ptr] + [M]


def _slots(ptr, M, shift):
    """(group, begin, end, start, index) of every live slot, as find_slot computes them."""
    e, G = _edges(ptr, M), len(ptr) - 1
    keys = [(e[i] >> shift) + i for i in range(G + 2)]
    out = []
    for s in range((M >> shift) + G + 2):
        le = [i for i in range(G + 2) if keys[i] <= s]
        i = le[-1]
        a, b = e[i], e[i + 1]
        begin = a + ((s - keys[i]) << shift)
        if s >= keys[i] and begin < b:
            out.append((-1 if i in (0, G + 1) else i - 1, begin, min(b, begin + (1 << shift)), a, s - keys[i]))
    return out


@pytest.mark.parametrize("seed", range(40))
def test_row_slots_cover_every_row_once(seed):
    rng = np.random.default_rng(seed)
    M, G, shift = int(rng.integers(0, 900)), int(rng.integers(0, 90)), int(rng.integers(3, 8))
    ptr = np.sort(rng.integers(0, M + 1, G + 1)) if seed % 3 else np.sort(rng.choice([0, M // 3, M], G + 1))
    owner = np.full(M, -2)
    for group, begin, end, _, _ in _slots(ptr, M, shift):
        assert (owner[begin:end] == -2).all()
        owner[begin:end] = group
    want = np.full(M, -1)
    for g in range(G):
        want[ptr[g]:ptr[g + 1]] = g
    assert (owner == want).all()


GROUP_ROWS = 64


def _place(e, i):
    """Where group i (of those with the two of no weight) begins on the line of rows and GROUP_ROWS positions behind each group."""
    return e[i] + max(i - 1, 0) * GROUP_ROWS


def _group_at(e, s):
    return max(j for j in range(len(e) - 1) if _place(e, j) <= s)


def _row_at(e, s):
    i = _group_at(e, s)
    return min(e[i] + max(0, s - _place(e, i)), e[i + 1])


def _segments(ptr, M, chunk, c):
    """(group, begin, end, partial slot) of a chunk of positions, as Segments walks them."""
    e, G = _edges(ptr, M), len(ptr) - 1
    first, last = _row_at(e, c * chunk), _row_at(e, (c + 1) * chunk)
    out, at = [], first
    while at < last:
        lo = at
        i = max(j for j in range(G + 2) if e[j] <= lo)
        b, t = e[i], e[i + 1]
        if t <= lo:  # (bounds that decrease)
            break
        at = min(t, last)
        if i == 0:
            continue
        if i == G + 1:
            break
        out.append((i - 1, lo, at, -1 if b >= first and t <= last else 2 * c if b >= first else 2 * c + 1))
    return out


@pytest.mark.parametrize("seed", range(60))
def test_weight_gradient_segments(seed):
    """Every row of a group is in one segment, every group with rows is finished once (in place, or by the join of its parts, which reads
    exactly the slots that were written), and no slot is written twice."""
    rng = np.random.default_rng(seed)
    M, G, chunk = int(rng.integers(0, 700)), int(rng.integers(1, 60)), int(rng.choice([8, 64, 96, 1000]))
    ptr = np.sort(rng.integers(0, M + 1, G + 1)) if seed % 3 else np.sort(rng.choice([0, M // 3, M // 2, M], G + 1))
    chunks = max(1, -(-(M + (G - 1) * GROUP_ROWS) // chunk))
    owner, done, slots = np.full(M, -1), np.zeros(G, int), {}
    for c in range(chunks):
        for group, lo, hi, slot in _segments(ptr, M, chunk, c):
            assert (owner[lo:hi] == -1).all() and ptr[group] <= lo < hi <= ptr[group + 1]
            owner[lo:hi] = group
            if slot < 0:
                done[group] += 1
                assert hi - lo == ptr[group + 1] - ptr[group]
            else:
                assert slot not in slots and slot < 2 * chunks
                slots[slot] = group
    e = _edges(ptr, M)
    for c0 in range(chunks - 1):  # wgrad_join_kernel
        after = (c0 + 1) * chunk
        i = _group_at(e, after - 1)
        start, end, place = e[i], e[i + 1], _place(e, i)
        if i in (0, G + 1) or place < c0 * chunk or place > after - 1 or end - start <= after - place:
            continue
        done[i - 1] += 1
        for c in range((place + end - 1 - start) // chunk - c0 + 1):
            assert slots.pop(2 * (c0 + c) + (c > 0)) == i - 1
    assert not slots and (done == (ptr[1:] > ptr[:-1])).all()
    for g in range(G):
        assert (owner[ptr[g]:ptr[g + 1]] == g).all()


@pytest.mark.parametrize("seed", range(10))
def test_row_slots_of_a_wrong_table_stay_inside(seed):
    rng = np.random.default_rng(seed)
    M = int(rng.integers(1, 500))
    ptr = rng.integers(-2**31, 2**31, 20) if seed % 2 else rng.integers(-5, M + 5, 20)  # unsorted, out of range
    e = _edges(ptr, M)
    for shift in (5, 7):
        for i in range(len(e) - 1):  # whatever group the search ends on
            for index in range(0, (M >> shift) + 2):
                begin = e[i] + (index << shift)
                if begin < e[i + 1]:
                    assert 0 <= begin < min(e[i + 1], begin + (1 << shift)) <= M
    G, chunk = len(ptr) - 1, int(rng.choice([64, 200]))
    chunks = -(-(M + (G - 1) * GROUP_ROWS) // chunk)
    for i in range(G + 2):  # the weight gradient: rows of a chunk, and the slots that the join of a group's parts reads
        for s in range(0, chunks * chunk + 1, 17):
            assert 0 <= min(e[i] + max(0, s - _place(e, i)), e[i + 1]) <= M
        if 0 < i < G + 1 and e[i + 1] > e[i]:
            assert 0 <= (_place(e, i) + e[i + 1] - 1 - e[i]) // chunk < chunks


# ---- wrappers ----
def test_gate_kinds():
    g = kernels.residual_norm_gate_kind
    assert g(None, 5, 3) == 0 and g(torch.zeros(()), 5, 3) == 1 and g(torch.zeros(1), 5, 3) == 1 and g(torch.zeros(3), 5, 3) == 2
    assert g(torch.zeros(5, 1), 5, 3) == 3 and g(torch.zeros(5, 3), 5, 3) == 4 and g(torch.zeros(1), 5, 1) == 1
    for shape in ((5, ), (1, 3), (3, 5), (5, 3, 1)):
        with pytest.raises(ValueError):
            g(torch.zeros(shape), 5, 3)


def test_dense_and_overlap():
    t = torch.zeros(6, 8)
    assert kernels._is_dense(t) and kernels._is_dense(t.t()) and kernels._is_dense(t[1:3]) and not kernels._is_dense(t[:, :4])
    assert not kernels._is_dense(torch.zeros(1).expand(4)) and kernels._is_dense(torch.zeros(3, 1, 2).permute(2, 1, 0))
    kernels._refuse_overlap([0, 4, 8, 6], [4, 8, 8, 6])
    with pytest.raises(ValueError):
        kernels._refuse_overlap([4, 0], [8, 5])


def test_norm_types():
    assert [kernels._norm_type(p) for p in (1, 2, "inf", float("inf"), 2.0)] == [1, 2, 0, 0, 2]
    for p in (0, 3, -1, float("nan"), "x", None):
        with pytest.raises(ValueError):
            kernels._norm_type(p)


def test_clip_grad_norm_without_gradients():
    assert float(kernels.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0


def test_group_rows():
    from dance_amd.nn import group_rows
    types = torch.tensor([2, 0, -1, 2, 5, 0, 3])
    order, ptr = group_rows(types, 4)
    assert types[order].tolist() == [-1, 0, 0, 2, 2, 3, 5] and order.tolist() == [2, 1, 5, 0, 3, 6, 4]
    assert ptr.dtype == torch.int32 and ptr.tolist() == [1, 3, 3, 5, 6]
    assert group_rows(torch.zeros(0, dtype=torch.int32), 2)[1].tolist() == [0, 0, 0]
    for bad in (torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2), torch.zeros(2, dtype=torch.bool)):
        with pytest.raises(ValueError):
            group_rows(bad, 2)


@pytest.mark.skipif(torch.cuda.is_available(), reason="CPU-box behaviour")
def test_no_cpu_path():
    t = torch.zeros(4, 4)
    for call in (lambda: kernels.gemm_grouped(t, t[None], torch.tensor([0, 4], dtype=torch.int32)), lambda: kernels.residual_norm_forward(t),
                 lambda: kernels.clip_grads([t], 1.0), lambda: kernels.global_norm([t])):
        with pytest.raises(_lib.DanceHipError):
            call()

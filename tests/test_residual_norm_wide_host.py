"""CPU: refusals of the wide residual norm at the C ABI (every call returns before it reaches the device) and its workspace."""
import pytest

from dance_amd import _lib

P = 4096  # some non-null address: no call below may get as far as using it
INVALID, WORKSPACE = -1, -3
D = 5000


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _fwd(lib, **kw):
    a = dict(M=4, D=D, dtype=0, f=P, ldf=D, x=P, ldx=D, gate=None, ldg=0, gk=0, sig=0, scale=1.0, kind=0, eps=1e-5, post=1, w1=None, b1=None, pre=1,
             w2=None, b2=None, r=P, ldr=D, h=P, ldh=D, stats=P, stream=None)
    a.update(kw)
    return lib.dh_residual_norm_wide_forward(*a.values())


def _bwd(lib, **kw):
    a = dict(M=4, D=D, dtype=0, f=P, ldf=D, x=P, ldx=D, gate=None, ldg=0, gk=0, sig=0, scale=1.0, kind=0, post=1, w1=None, b1=None, pre=1, w2=None,
             stats=P, dr=P, lddr=D, dh=P, lddh=D, df=P, lddf=D, dx=P, lddx=D, dgate=None, lddg=0, dw1=None, db1=None, dw2=None, db2=None, ws=P,
             ws_bytes=1 << 24, stream=None)
    a.update(kw)
    return lib.dh_residual_norm_wide_backward(*a.values())


@pytest.mark.parametrize("bad", [dict(M=-1), dict(M=2**31), dict(D=4096), dict(D=8193, ldf=8193, ldx=8193, ldr=8193, ldh=8193), dict(post=0, pre=0), dict(dtype=2),
                                 dict(f=None), dict(ldf=D - 1), dict(gk=1), dict(gk=4, gate=P, ldg=D - 1), dict(h=None), dict(r=None, pre=0), dict(ldr=D - 1),
                                 dict(ldh=D - 1), dict(stats=P + 4), dict(eps=float("nan"))])
def test_forward_refusals(lib, bad):
    assert _fwd(lib, **bad) == INVALID
    assert b"dh_residual_norm_wide_forward" in lib.dh_last_error_string()
    assert _fwd(lib, M=0) == 0


@pytest.mark.parametrize("bad", [dict(D=4096), dict(D=8193), dict(post=0, pre=0, dh=None), dict(stats=None), dict(pre=0), dict(dr=None, dh=None), dict(lddr=D - 1),
                                 dict(lddf=D - 1), dict(post=0, dw1=P), dict(dgate=P), dict(ws=P + 8)])
def test_backward_refusals(lib, bad):
    assert _bwd(lib, **bad) == INVALID
    need = lib.dh_residual_norm_backward_workspace_bytes(4, D)
    assert _bwd(lib, ws_bytes=need - 1) == WORKSPACE and _bwd(lib, ws=None) == WORKSPACE


def test_workspace(lib):
    """Five arrays of one partial row per workgroup and one row beside them; two numbers of each row for wide ones."""
    size = lib.dh_residual_norm_backward_workspace_bytes
    assert size(4, 4096) == 21 * 4096 * 4 and size(4, D) == 21 * D * 4 + 4 * 8 and size(5000, 8191) == -(-5121 * 8191 * 4 // 16) * 16 + 5000 * 8

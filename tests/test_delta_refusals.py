"""What the C entries of the layer operators refuse, before any launch: runs without a GPU."""
import ctypes

import pytest

from vlm_training_amd import _lib

FINE = dict(q=16, k=16, v=16, a=16, b=16, a_log=16, dt_bias=16, q_tok=128, q_head=64, k_tok=128, k_head=64, v_tok=256, v_head=64, a_tok=4, b_tok=4, cu=16,
            T=64, N=1, Hk=2, Hv=4, Dk=64, Dv=64, scale=0.125, l2_norm=1)


def _args(**change):
    return ctypes.byref(_lib.DeltaArgs(**{**FINE, **change}))


@pytest.mark.parametrize("change,code,text", [
    (dict(Hv=3), -1, b"multiple of key heads"), (dict(Hk=0), -1, b"Hk=0"), (dict(T=-1), -1, b"T=-1"), (dict(Dk=136), -2, b"head dims"), (dict(Dv=12), -2, b"head dims"),
    (dict(N=0), -1, b"cu_seqlens"), (dict(cu=None), -1, b"cu_seqlens"), (dict(scale=0.0), -1, b"scale"), (dict(scale=float("nan")), -1, b"scale"), (dict(q=None), -1, b"null"),
    (dict(k_tok=12), -1, b"strides"), (dict(v=8), -1, b"16-byte"), (dict(N=1 << 28, Hv=8), -2, b"too many"),
])
def test_gated_delta_rule(change, code, text):
    lib = _lib.load()
    assert lib.dsa_delta_fwd(_args(**change), None, 16, None, 0, 16, 1 << 40, None) == code
    assert text in lib.dsa_last_error()
    assert lib.dsa_delta_bwd(_args(**change), 16, None, 16, 1 << 40, 16, 16, 16, 16, 16, 16, 16, None, 16, 1 << 40, None) == code
    assert lib.dsa_delta_workspace_bytes(_args(**change), 1) == 0 and lib.dsa_delta_scratch_bytes(_args(**change)) == 0
    if "N" not in change and "cu" not in change:
        assert lib.dsa_delta_step(_args(**change), 16, 1 << 20, 16, None) == code


def test_gated_delta_rule_buffers():
    lib = _lib.load()
    small, large = lib.dsa_delta_workspace_bytes(_args(), 0), lib.dsa_delta_workspace_bytes(_args(), 1)
    assert 0 < small < large and lib.dsa_delta_scratch_bytes(_args()) > 0
    assert lib.dsa_delta_fwd(_args(), None, 16, None, 0, 256, small - 1, None) == -3
    assert lib.dsa_delta_fwd(_args(), None, 16, None, 1, 256, small, None) == -3
    assert lib.dsa_delta_fwd(_args(), None, 16, None, 0, None, small, None) == -3
    assert lib.dsa_delta_fwd(_args(), None, None, None, 0, 256, small, None) == -1
    assert lib.dsa_delta_fwd(None, None, 16, None, 0, 256, small, None) == -1
    assert lib.dsa_delta_bwd(_args(), 16, None, 256, small, 16, 16, 16, 16, 16, 16, 16, None, 256, 1 << 40, None) == -3
    assert lib.dsa_delta_bwd(_args(), 16, None, 256, large, 16, 16, 16, 16, 16, 16, 16, None, 256, 0, None) == -3
    assert lib.dsa_delta_bwd(_args(), None, None, 256, large, 16, 16, 16, 16, 16, 16, 16, None, 256, 1 << 40, None) == -1
    assert lib.dsa_delta_step(_args(), None, 1 << 20, 16, None) == -1
    assert lib.dsa_delta_step(_args(), 8, 1 << 20, 16, None) == -1 and b"apart" in lib.dsa_last_error()
    assert lib.dsa_delta_step(_args(), 16, 64, 16, None) == -1


def test_convolution():
    lib = _lib.load()
    fwd = lambda x=16, tok=64, w=16, cu=16, T=8, N=1, C=64, W=4, y=16: lib.dsa_conv_fwd(x, tok, w, 0, None, 0, 1, cu, T, N, C, W, None, y, None, None)
    for change, code in ((dict(T=-1), -1), (dict(N=0), -1), (dict(cu=None), -1), (dict(W=1), -2), (dict(W=5), -2), (dict(C=12), -2), (dict(C=0), -2), (dict(w=None), -1),
                         (dict(x=None), -1), (dict(tok=12), -1), (dict(x=8), -1), (dict(y=None), -1), (dict(y=8), -1)):
        assert fwd(**change) == code, change
    need = lib.dsa_conv_bwd_workspace_bytes(8, 64, 4)
    assert need > 0 and lib.dsa_conv_bwd_workspace_bytes(0, 64, 4) == 0
    bwd = lambda dy=16, dx=16, dw=16, bias=None, db=None, ws=16, n=need: lib.dsa_conv_bwd(16, 64, dy, 64, 16, 0, bias, 0, 1, 16, 8, 1, 64, 4, None, dx, dw, db, ws, n, None)
    for change, code in ((dict(dy=None), -1), (dict(dx=None), -1), (dict(dw=None), -1), (dict(bias=16), -1), (dict(dy=8), -1), (dict(ws=None), -3), (dict(n=need - 1), -3)):
        assert bwd(**change) == code, change
    step = lambda state=16, stride=192, y=16, B=2: lib.dsa_conv_step(16, 64, 16, 0, None, 0, 1, B, 64, 4, state, stride, y, None)
    for change in (dict(state=None), dict(state=8), dict(stride=100), dict(stride=184), dict(y=None)):
        assert step(**change) == -1, change


def test_norms():
    lib = _lib.load()
    gn = lambda x=16, tok=64, w=16, T=4, H=1, D=64, y=16: lib.dsa_gated_norm_fwd(x, tok, 64, 16, 64, 64, w, 0, 1e-6, 0.0, T, H, D, y, None, None)
    for change, code in ((dict(T=-1), -1), (dict(H=0), -1), (dict(D=520), -2), (dict(D=12), -2), (dict(x=None), -1), (dict(w=None), -1), (dict(tok=4), -1), (dict(x=8), -1),
                         (dict(y=8), -1)):
        assert gn(**change) == code, change
    need = lib.dsa_gated_norm_bwd_workspace_bytes(4, 1, 64)
    assert lib.dsa_gated_norm_bwd(16, 16, 64, 64, 16, 64, 64, 16, 0, 0.0, 4, 1, 64, 16, 16, 16, 16, 16, need - 1, None) == -3
    assert lib.dsa_gated_norm_bwd(16, 16, 64, 64, 16, 64, 64, 16, 0, 0.0, 4, 1, 64, None, 16, 16, 16, 16, need, None) == -1
    rn = lambda x=16, y=16, w=16, T=4, C=64, xn=16: lib.dsa_residual_norm_fwd(x, 0, y, None, w, 0, None, 0, None, 0, 1e-6, 0.0, T, C, xn, 16, None, None, None)
    for change, code in ((dict(T=-1), -1), (dict(C=8200), -2), (dict(C=12), -2), (dict(x=None), -1), (dict(w=None), -1), (dict(y=8), -1), (dict(xn=8), -1)):
        assert rn(**change) == code, change
    need = lib.dsa_residual_norm_bwd_workspace_bytes(4, 64)
    bwd = lambda y=16, gate=None, post=None, dpost=None, dgate=None, ry=None, n=need: lib.dsa_residual_norm_bwd(
        16, 16, 16, 0, y, gate, 16, 0, post, 0, None, 0, 0.0, 4, 64, 16, ry, 16, 16, dgate, 16, dpost, None, 16, n, None)
    for change, code in ((dict(n=need - 1), -3), (dict(post=16), -1), (dict(post=16, dpost=16), -1), (dict(gate=16), -1), (dict(gate=16, dgate=16, y=None), -1)):
        assert bwd(**change) == code, change


def test_outputs_and_workspaces_off_their_boundaries():
    """What kernels write or read 16 bytes at a time; more rows than a run's 32-bit end can name."""
    lib = _lib.load()
    small, large = lib.dsa_delta_workspace_bytes(_args(), 0), lib.dsa_delta_workspace_bytes(_args(), 1)
    # (buffers too small on top: nothing is launched, whichever is looked at first)
    assert lib.dsa_delta_fwd(_args(), None, 24, None, 0, 256, small - 1, None) == -1 and b"16-byte" in lib.dsa_last_error()
    assert lib.dsa_delta_fwd(_args(), None, 16, None, 0, 264, small - 1, None) == -1
    good = dict(dout=16, ws=256, dq=16, dk=16, dv=16, scratch=256)
    bwd = lambda dout, ws, dq, dk, dv, scratch: lib.dsa_delta_bwd(_args(), dout, None, ws, large, dq, dk, dv, 16, 16, 16, 16, None, scratch, 0, None)
    assert bwd(**good) == -3
    for name, at in good.items():
        assert bwd(**{**good, name: at + 8}) == -1, name
        assert b"16-byte" in lib.dsa_last_error()
    assert lib.dsa_delta_step(_args(), 16, 63, 24, None) == -1
    conv = lambda T=8, ws=16, dw=16: lib.dsa_conv_bwd(16, 64, 16, 64, 16, 0, None, 0, 1, 16, T, 1, 64, 4, None, 16, dw, None, ws, 0, None)
    assert conv() == -3 and conv(ws=24) == -1
    assert conv(T=(1 << 30) + 1) == -2 and b"rows" in lib.dsa_last_error()
    assert lib.dsa_conv_fwd(16, 64, 16, 0, None, 0, 1, 16, (1 << 30) + 1, 1, 64, 4, None, 16, None, None) == -2
    assert lib.dsa_gated_norm_bwd(16, 16, 64, 64, 16, 64, 64, 16, 0, 0.0, 4, 1, 64, 16, 16, 16, 16, 24, 0, None) == -1
    assert lib.dsa_residual_norm_bwd(16, 16, 16, 0, 16, None, 16, 0, None, 0, None, 0, 0.0, 4, 64, 16, None, 16, 16, None, 16, None, None, 24, 0, None) == -1

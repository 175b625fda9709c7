"""CPU checks of the C entry points of the gated delta rule and the group norm: sizes and refusals.  None of these
calls launches a kernel."""

import ctypes

import pytest

from mamba_ssm_benchmark_b200 import _native as nat

H, V = nat.SsmHeads, nat.SsmView
P = ctypes.c_void_p(4096)
DIMS = (2, 100, 2, 4, 64, 48)


def _heads(dtype=nat.SSM_F32):
    return H(P, dtype, 0, 1 << 20, 1 << 10, 64)


def _gate(dtype=nat.SSM_F32):
    return V(P, dtype, 0, 400, 4)


def _size(dims, dtype=nat.SSM_F32, backward=0):
    n = ctypes.c_size_t(0)
    rc = nat.lib().ssm_gated_delta_workspace_size(*dims, dtype, backward, ctypes.byref(n))
    return rc, n.value


def _message():
    return nat.lib().ssm_last_error_message().decode()


def test_sizes():
    B, L, Hk, Hv, dk, dv = DIMS
    chunks = B * Hv * 2
    rc, fwd = _size(DIMS)
    assert rc == nat.SSM_OK and fwd >= chunks * 6 * 64 * 64 * 2
    rc, bwd = _size(DIMS, backward=1)
    assert rc == nat.SSM_OK and bwd >= chunks * 48 * (64 + 64) * 4
    n = ctypes.c_size_t(0)
    assert nat.lib().ssm_gated_delta_saved_size(*DIMS, nat.SSM_F32, ctypes.byref(n)) == nat.SSM_OK
    assert n.value >= fwd + chunks * 48 * (64 + 64) * 4 - 256


@pytest.mark.parametrize("dims,code,text", [
    ((0, 1, 1, 1, 1, 1), nat.SSM_ERR_INVALID, "positive"), ((1, 1, 2, 3, 1, 1), nat.SSM_ERR_INVALID, "multiple"),
    ((1, 1, 1, 1, 129, 1), nat.SSM_ERR_UNSUPPORTED, "key width"), ((70000, 1, 1, 1, 1, 1), nat.SSM_ERR_INVALID, "range"),
])
def test_refused_shapes(dims, code, text):
    rc, _ = _size(dims)
    assert rc == code and text in _message()


def test_refused_arguments():
    lib = nat.lib()

    def fwd(q=None, k=None, g=None, ws=P, wsb=1 << 40):
        return lib.ssm_gated_delta_fwd(*DIMS, q or _heads(), k or _heads(), _heads(), g or _gate(), _gate(), None, 1.0,
                                       _heads(), None, None, ws, wsb, None)

    assert _size(DIMS, dtype=7)[0] == nat.SSM_ERR_DTYPE
    assert fwd(q=H(None, 0, 0, 0, 0, 0)) == nat.SSM_ERR_INVALID and "q is required" in _message()
    assert fwd(k=_heads(nat.SSM_BF16)) == nat.SSM_ERR_DTYPE and "k must" in _message()
    assert fwd(g=_gate(nat.SSM_BF16)) == nat.SSM_ERR_DTYPE and "float32" in _message()
    assert fwd(ws=None) == nat.SSM_ERR_WORKSPACE and fwd(wsb=100) == nat.SSM_ERR_WORKSPACE
    rc = lib.ssm_gated_delta_bwd(*DIMS, _heads(), _heads(), _heads(), _gate(), _gate(), 1.0, None, _heads(), None, _heads(),
                                 _heads(), _heads(), P, P, None, P, 1 << 40, None)
    assert rc == nat.SSM_ERR_INVALID and "saved" in _message()
    rc = lib.ssm_gated_delta_state_update(2, 2, 4, 64, 48, None, _heads(), _heads(), _heads(), _gate(), _gate(), 1.0,
                                          _heads(), None)
    assert rc == nat.SSM_ERR_INVALID and "state" in _message()


def test_group_norm_refusals():
    lib, n = nat.lib(), ctypes.c_size_t(0)
    size = lambda *a: lib.ssm_group_norm_workspace_size(*a, ctypes.byref(n))
    assert size(10, 1, 64, 4, 0) == nat.SSM_OK and n.value == 0           # head norms need none forward
    assert size(10, 5, 64, 4, 0) == nat.SSM_OK and n.value > 0
    assert size(10, 1, 64, 4, 1) == nat.SSM_OK and n.value > 0
    assert size(10, 1, 64, 5, 0) == nat.SSM_ERR_INVALID and "split" in _message()
    assert size(0, 1, 64, 4, 0) == nat.SSM_ERR_INVALID
    x, none = V(P, nat.SSM_F32, 0, 64, 64), nat.NULL_VIEW

    def fwd(x, z=none, y=x, positions=1, ws=None):
        return lib.ssm_group_norm_fwd(10, positions, 64, 4, x, None, None, 1e-5, 0, 0, z, y, None, ws, 0, None)

    assert fwd(none) == nat.SSM_ERR_INVALID and "x is required" in _message()
    assert fwd(x, z=V(P, nat.SSM_BF16, 0, 64, 64)) == nat.SSM_ERR_DTYPE and "z must" in _message()
    assert fwd(x, y=none) == nat.SSM_ERR_INVALID and "y is required" in _message()
    assert fwd(x, positions=5) == nat.SSM_ERR_WORKSPACE


def test_group_norm_shapes_out_of_range():
    """More elements than a GPU holds are refused before a grid is cut off; 2^32 (sample, group) pairs are not."""
    n = ctypes.c_size_t(0)
    size = lambda *a: nat.lib().ssm_group_norm_workspace_size(*a, ctypes.byref(n))
    assert size(2 ** 30, 2 ** 30, 2 ** 20, 1, 0) == nat.SSM_ERR_INVALID and "range" in _message()
    assert size(2 ** 30, 2 ** 10, 2, 1, 0) == nat.SSM_ERR_INVALID and "range" in _message()
    assert size(2 ** 30, 1, 2 ** 11, 1, 0) == nat.SSM_ERR_INVALID and "range" in _message()
    assert size(2 ** 22, 2, 1024, 1024, 1) == nat.SSM_OK

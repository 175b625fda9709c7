"""CPU checks of the operators around the mixers: refusals of the Python functions and of the C entry points, workspace
sizes.  None of these calls launches a kernel."""

import ctypes

import pytest
import torch

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import embedding, linear_fp8, quantize_fp8, rms_norm, rms_norm_fp8, sample_tokens

P = ctypes.c_void_p(4096)
V = lambda dtype=nat.SSM_F32, stride=64: nat.SsmView(P, dtype, 0, stride, 0)
E8 = torch.float8_e4m3fn


def _message():
    return nat.lib().ssm_last_error_message().decode()


def _size(name, *dims):
    n = ctypes.c_size_t(0)
    return getattr(nat.lib(), name)(*dims, ctypes.byref(n)), n.value


def test_embedding_entry_points():
    rc, n = _size("ssm_embedding_bwd_workspace_size", 1000, 50, 64)
    assert rc == nat.SSM_OK and n >= 1000 * 16
    for dims in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1 << 31, 1, 1), (1, 1 << 31, 1)):
        assert _size("ssm_embedding_bwd_workspace_size", *dims)[0] == nat.SSM_ERR_INVALID
    lib = nat.lib()
    fwd = lambda idx=P, size=8, w=V(), y=V(): lib.ssm_embedding_fwd(10, 20, 64, idx, size, w, 1.0, y, None)
    assert fwd(idx=None) == nat.SSM_ERR_INVALID and fwd(size=2) == nat.SSM_ERR_DTYPE
    assert fwd(w=nat.NULL_VIEW) == nat.SSM_ERR_INVALID and "weight" in _message()
    assert fwd(y=V(nat.SSM_BF16)) == nat.SSM_ERR_DTYPE and fwd(w=V(5)) == nat.SSM_ERR_DTYPE
    bwd = lambda ws=P, n=1 << 30, dw=V(): lib.ssm_embedding_bwd(10, 20, 64, P, 8, 1.0, V(), dw, ws, n, None)
    assert bwd(ws=None) == nat.SSM_ERR_WORKSPACE and bwd(n=100) == nat.SSM_ERR_WORKSPACE
    assert bwd(dw=nat.NULL_VIEW) == nat.SSM_ERR_INVALID and bwd(dw=V(nat.SSM_BF16)) == nat.SSM_ERR_DTYPE


def test_rms_norm_entry_points():
    rc, n = _size("ssm_rms_norm_bwd_workspace_size", 100000, 64)
    assert rc == nat.SSM_OK and n >= 100000 // 256 * 64 * 4
    for dims in ((0, 1), (1, 0), (1, 1 << 25), (1 << 30, 1 << 20)):
        assert _size("ssm_rms_norm_bwd_workspace_size", *dims)[0] == nat.SSM_ERR_INVALID
    lib, none = nat.lib(), nat.NULL_VIEW
    fwd = lambda x=V(), r=none, y=V(), t=none, wd=0: lib.ssm_rms_norm_fwd(10, 64, x, r, P, wd, 1e-5, y, t, None)
    assert fwd(x=none) == nat.SSM_ERR_INVALID and fwd(y=none) == nat.SSM_ERR_INVALID
    assert fwd(x=V(9)) == nat.SSM_ERR_DTYPE and fwd(y=V(nat.SSM_BF16)) == nat.SSM_ERR_DTYPE and fwd(wd=9) == nat.SSM_ERR_DTYPE
    assert fwd(r=V()) == nat.SSM_ERR_INVALID and fwd(r=V(), t=V(nat.SSM_BF16)) == nat.SSM_ERR_DTYPE
    assert fwd(r=V(nat.SSM_BF16), t=V(nat.SSM_BF16)) == nat.SSM_ERR_DTYPE and "residual" in _message()
    fp8 = lambda y=P, s=P: lib.ssm_rms_norm_fp8(10, 64, V(), none, None, 0, 1e-5, 1, y, 64, s, none, None)
    assert fp8(y=None) == nat.SSM_ERR_INVALID and fp8(s=None) == nat.SSM_ERR_INVALID
    bwd = lambda t=V(), dx=V(), dr=none, ws=P, n=1 << 30: lib.ssm_rms_norm_bwd(10, 64, t, None, 0, 1e-5, V(), none, dx, dr, None, ws, n, None)
    assert bwd(t=none) == nat.SSM_ERR_INVALID and bwd(dx=none) == nat.SSM_ERR_INVALID and bwd(dr=V(1)) == nat.SSM_ERR_DTYPE
    assert bwd(ws=None) == nat.SSM_ERR_WORKSPACE and bwd(n=64) == nat.SSM_ERR_WORKSPACE


def test_linear_and_sampling_entry_points():
    lib, none = nat.lib(), nat.NULL_VIEW

    def lin(M=4, N=8, K=64, x=P, xst=64, w=P, y=V(), r=none):
        return lib.ssm_linear_fp8(M, N, K, x, xst, P, w, 64, P, None, 0, r, y, None)

    for kw in (dict(M=0), dict(N=0), dict(K=0), dict(M=1 << 30), dict(x=None), dict(w=None), dict(y=none), dict(xst=72), dict(xst=48),
               dict(x=ctypes.c_void_p(4097))):
        assert lin(**kw) == nat.SSM_ERR_INVALID, kw
    assert lin(y=V(7)) == nat.SSM_ERR_DTYPE and lin(r=V(1)) == nat.SSM_ERR_DTYPE

    def smp(B=2, n=64, l=V(), u=P, t=P):
        return lib.ssm_sample_tokens(B, n, l, u, None, 1.0, None, 0, None, 1.0, None, 0.0, t, None)

    for kw in (dict(B=0), dict(n=0), dict(n=(1 << 20) + 1), dict(l=none), dict(u=None), dict(t=None)):
        assert smp(**kw) == nat.SSM_ERR_INVALID, kw
    assert smp(l=V(3)) == nat.SSM_ERR_DTYPE


def test_embedding_refusals():
    W, idx = torch.zeros(5, 4), torch.zeros(3, dtype=torch.long)
    for args, kind, text in (((idx, W[0]), ValueError, "weight must be"), ((idx, W[:0]), ValueError, "empty"), ((idx[:0], W), ValueError, "empty"),
                             ((idx.float(), W), TypeError, "int64"), ((idx, W.double()), TypeError, "float32 or bfloat16"),
                             ((idx, W.half()), TypeError, "float32 or bfloat16"), ((idx, W), RuntimeError, "CUDA")):
        with pytest.raises(kind, match=text):
            embedding(*args)


def test_rms_norm_refusals():
    x, w = torch.zeros(3, 8), torch.ones(8)
    for fn in (rms_norm, rms_norm_fp8):
        for kw, kind, text in ((dict(x=x[:0]), ValueError, "empty"), (dict(x=x, weight=w[:4]), ValueError, "weight must be"),
                               (dict(x=x, residual=x[:1]), ValueError, "residual must be"), (dict(x=x, eps=-1.0), ValueError, "eps"),
                               (dict(x=x, eps=float("nan")), ValueError, "eps"), (dict(x=x.double()), TypeError, "float64"),
                               (dict(x=x.long()), TypeError, "not supported"), (dict(x=x, residual=x.double()), TypeError, "float64"),
                               (dict(x=x), RuntimeError, "CUDA"), (dict(x=torch.zeros(())), ValueError, "empty|must be")):
            with pytest.raises(kind, match=text):
                fn(**kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_fp8(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize_fp8(x.requires_grad_())


def test_linear_refusals():
    x8, w8 = torch.zeros(3, 32).to(E8), torch.zeros(5, 32).to(E8)
    xs, ws = torch.ones(3), torch.ones(5)
    good = dict(x8=x8, x_scale=xs, weight8=w8, weight_scale=ws)
    for kw, kind, text in ((dict(x8=x8.float()), TypeError, "float8_e4m3fn"), (dict(weight8=w8[0]), ValueError, "must be"),
                           (dict(x8=x8[:, :16]), ValueError, "columns"), (dict(x8=x8[:0], x_scale=xs[:0]), ValueError, "empty"),
                           (dict(x_scale=xs[:2]), ValueError, "scales"), (dict(weight_scale=ws[:2]), ValueError, "scales"),
                           (dict(x_scale=xs.double()), TypeError, "scales"), (dict(activation="relu"), ValueError, "activation"),
                           (dict(bias=xs), ValueError, "bias"), (dict(dtype=torch.float16), TypeError, "dtype"),
                           (dict(residual=torch.zeros(3, 4)), ValueError, "residual"),
                           (dict(residual=torch.zeros(3, 5), dtype=torch.bfloat16), ValueError, "residual"),
                           (dict(bias=torch.ones(5, requires_grad=True)), RuntimeError, "no gradient"), (dict(), RuntimeError, "CUDA")):
        with pytest.raises(kind, match=text):
            linear_fp8(**{**good, **kw})


def test_sampling_refusals():
    l, u = torch.zeros(2, 9), torch.zeros(2)
    for kw, kind, text in ((dict(logits=l[0]), ValueError, "logits must be"), (dict(logits=l[:0], uniforms=u[:0]), ValueError, "empty"),
                           (dict(uniforms=u[:1]), ValueError, "uniforms must be"), (dict(logits=l.double()), TypeError, "float32"),
                           (dict(uniforms=u.double()), TypeError, "float32"), (dict(temperature=-1.0), ValueError, "temperature"),
                           (dict(temperature=float("nan")), ValueError, "temperature"), (dict(top_k=-1), ValueError, "top_k"),
                           (dict(top_p=1.5), ValueError, "top_p"), (dict(min_p=-0.1), ValueError, "min_p"),
                           (dict(top_p=torch.ones(3)), ValueError, "number or a"), (dict(), RuntimeError, "CUDA")):
        with pytest.raises(kind, match=text):
            sample_tokens(**{**dict(logits=l, uniforms=u), **kw})
